// Matrix product of 8-bit (e4m3) operands with fp32 scales per block of 128, for one matrix or for one per expert over
// rows sorted by expert:
//   out[m, f] = sum_kb  xs[m, kb] * ws[f / 128, kb] * ( sum_{k in block kb} x[m, k] * w[f, k] )
// and, TRANS, the same stored weight contracted over its rows (the gradient of the input): out[m, f] = sum over n of
// x[m, n] * w[n, f] with the scale of block (n / 128, f / 128).
//
// The scales differ from one 128-block of the contraction to the next, so the tensor core cannot run the whole sum:
// each block's product (K 128 = four MMAs) goes to an accumulator of its own in tensor memory, and the epilogue warps
// add it, times its two scales, to sums that stay in fp32 registers for the whole tile. Tensor memory holds a ring of
// accumulators, so the MMAs of the next blocks run meanwhile.
//
// Up to 128 tokens per tile (fp8_gemm_kernel): 128 output features (weight rows, or columns under TRANS) are the MMA's M
// side and the tokens its N side. The weight's scale is one number per tile and block, ragged token counts only narrow the
// MMA, and a decode batch of a few tokens costs a narrow MMA instead of a mostly empty one. Such calls are bound by the
// weight's bytes (128 experts of 1536 x 2048, 16 tokens, 181 MB from HBM: 35 us = 5.2 TB/s) or, with few tiles, by latency
// (4096 x 7168, 1 token: 9.4 us on the device, 14 blocks of ~400 cycles behind launch, set-up and exchange). In between
// (4096 x 7168: 64 tokens 17 us, 100 20, 200 31) neither bytes nor arithmetic bound it: a CTA has 14 to 28 blocks, and
// every value added fetches its own token scale from shared memory.
// Larger ones run on CTA pairs with the roles exchanged (fp8_gemm_pair_kernel, below): 4096 x 4096 x 7168 in 134 us, 1.79
// PFLOP/s, when the GPU was idle before, and 148 us, 1.63 PFLOP/s, back to back, where the power cap holds the clock at
// 1680 MHz.
//
// TRANS reads the same 128 x 128 weight box from shared memory with the operand's transpose bit (features contiguous), so
// one copy of the weight serves both directions, at nearly the same speed (the same sums from a transposed weight: 141
// against 134 us, 152 against 147 back to back).
//
// Roles: warp 0 TMA producer, warp 1 tensor-memory owner, warps 1 and 3 MMA issuers, warp 2 the tile list, warps 4..
// epilogue (two per lane quadrant for 128 tokens). Every wait is bounded; a wait that gives up is reported by
// xmoe_fp8_status. An epilogue warp stays whole when some of its lanes give up, so that none is missing in a shuffle or an
// aligned tensor-memory read: up to 128 tokens the lanes walk on to the end of the tile (their waits return at once then),
// where the warp decides (a vote at every block costs 1 token 4 %); the pair kernel votes at every block (147 -> 148 us;
// walking on costs it 3 %).
#include "cluster.cuh"
#include "elem.cuh"
#include "kernels.h"
#include "tile_sched.cuh"

namespace xmoe {

// First error any product of this process has met on the device since the last xmoe_fp8_status (0: none).
static __device__ uint32_t g_fp8_status;

namespace {

constexpr int kMaxMats = 1032;
constexpr int kBoxBytes = 128 * 128;  // weight box of one block
constexpr uint32_t kBadSegment = 0x700u;

template <bool PAIR>
__device__ __forceinline__ void mma_fp8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
#define XMOE_MMA_FP8(GROUP)                                                                                            \
    asm volatile(                                                                                                      \
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"                                                                    \
        "mov.b64 da, {%1, %5};\n\t"                                                                                    \
        "mov.b64 db, {%2, %5};\n\t"                                                                                    \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                                    \
        "tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),                        \
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128)                                           \
        : "memory")
    if (PAIR) XMOE_MMA_FP8("2");
    else XMOE_MMA_FP8("1");
#undef XMOE_MMA_FP8
}
// kind::f8f6f4: accumulator fp32 [4,6) = 1, a/b format e4m3 = 0, transposed A [15] / B [16], N>>3 [17,23), M>>4 [24,29)
__host__ __device__ constexpr uint32_t idesc_fp8(uint32_t m, uint32_t n, bool a_trans, bool b_trans) {
    return (1u << 4) | ((a_trans ? 1u : 0u) << 15) | ((b_trans ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// A transposed operand (features contiguous): a K step of 32 is 32 rows of 128 bytes, 1024 bytes between 8-row groups, one
// box (16 KB) between swizzle atoms of 128 features.
__device__ __forceinline__ uint32_t desc_lo_trans(uint32_t smem_addr) { return ((smem_addr & 0x3ffffu) >> 4) | (((uint32_t)kBoxBytes >> 4) << 16); }
constexpr uint32_t kTransStep = (32u * 128u) >> 4;
// a * b + c on two fp32 at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// The number of tiles, by all threads; none (and reported) if segments that overlap make more than 31 bits can count.
__device__ __forceinline__ int count_tiles(const int* prefix, int mats, int threads) {
    int bad = 0;
    for (int e = threadIdx.x; e < mats; e += threads) bad |= prefix[e + 1] < prefix[e];
    if (!__syncthreads_or(bad)) return prefix[mats];
    if (threadIdx.x == 0) atomicCAS(&g_fp8_status, 0u, kBadSegment);
    return 0;
}

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// The same outcome for all lanes of a warp.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status,
                                               uint32_t code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code));
}

template <int TN>
struct Cfg {
    static constexpr int kEpiWarps = TN >= 128 ? 8 : 4;
    static constexpr int kThreads = 128 + 32 * kEpiWarps;
    static constexpr int kCols = TN / (kEpiWarps / 4);            // token columns per epilogue warp
    static constexpr int kChunk = kCols < 32 ? 16 : 32;           // columns per tensor-memory read
    static constexpr int kAcc = 4;                                // accumulators in tensor memory
    static constexpr int kTmemCols = kAcc * TN;
    static constexpr int kStageBytes = kBoxBytes + TN * 128;
    static constexpr int kStages = TN >= 128 ? 6 : (TN >= 64 ? 8 : 10);
    static constexpr int kGroup = 4, kSlots = 4;                  // blocks whose token scales come together; such groups in flight
    static_assert(kStages % 2 == 0 && kAcc % 2 == 0, "two issuing threads take the blocks in turn");
    static constexpr size_t kTail = (size_t)kSlots * kGroup * TN * 4 + 1024;
    static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kTail + (size_t)(3 * kMaxMats + 4) * 4;
    static_assert(kSmem <= 232448, "shared memory");
    static_assert(kTmemCols >= 32 && kTmemCols <= 512, "tensor memory");
};

// The experts' segments, kept inside the buffers: a segment that does not start at a multiple of 16 rows inside them
// counts as empty (and is reported), one that runs past the end is cut.
__device__ __forceinline__ void load_segments(const Fp8GemmArgs& a, int* counts, int* offsets, int threads) {
    for (int e = threadIdx.x; e < a.mats; e += threads) {
        int c = a.counts ? a.counts[e] : a.rows, o = a.counts ? a.offsets[e] : 0;
        if (c > 0 && (o < 0 || o >= a.rows || (o & 15))) {
            atomicCAS(&g_fp8_status, 0u, kBadSegment);
            c = 0;
        }
        counts[e] = c <= 0 ? 0 : min(c, a.rows - o);
        offsets[e] = o;
    }
}

// Completes the tensor-memory reads issued so far; naming the registers keeps their uses behind the wait.
template <int N>
__device__ __forceinline__ void tmem_wait_for(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
template <int N>
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t* r) {
    if (N == 32) tmem_ld32(taddr, r);
    else tmem_ld16(taddr, r);
}
// sums += v * (token scale * weight scale) over N columns; the token scales come from shared memory, the same for all lanes
template <int N>
__device__ __forceinline__ void add_scaled(float2* sum, const uint32_t* v, const float4* scale, float sw) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        const float4 x = scale[j], s = make_float4(x.x * sw, x.y * sw, x.z * sw, x.w * sw);
        sum[2 * j] = fma2(make_float2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), make_float2(s.x, s.y), sum[2 * j]);
        sum[2 * j + 1] = fma2(make_float2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), make_float2(s.z, s.w), sum[2 * j + 1]);
    }
}

template <int TN, bool TRANS, typename OT>
__global__ __launch_bounds__(Cfg<TN>::kThreads, 1) void fp8_gemm_kernel(const __grid_constant__ Fp8GemmArgs a) {
    using C = Cfg<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* scales = reinterpret_cast<float*>(smem + (size_t)C::kStages * C::kStageBytes);  // [kSlots][kGroup][TN] the tokens'
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(scales + C::kSlots * C::kGroup * TN);
    uint64_t* empty_bar = full_bar + 16;
    uint64_t* sc_full = empty_bar + 16;  // [kSlots]
    uint64_t* sc_empty = sc_full + 4;
    uint64_t* acc_full = sc_empty + 4;
    uint64_t* acc_empty = acc_full + 4;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 4);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    int* counts = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full_bar) + 1024);
    int* offsets = counts + kMaxMats;
    int* prefix = offsets + kMaxMats;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w_tiles = (a.out_features + 127) / 128;
    const int kb_total = (a.contraction + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < C::kSlots; ++s) {
            mbar_init(&sc_full[s], 1);
            mbar_init(&sc_empty[s], C::kEpiWarps);
        }
        for (int s = 0; s < C::kAcc; ++s) {
            mbar_init(&acc_full[s], 1);
            mbar_init(&acc_empty[s], C::kEpiWarps);
        }
        *abort_flag = 0u;
        mbar_fence_init();
        prefetch_tmap(&a.tm_w);
        prefetch_tmap(&a.tm_x);
        prefetch_tmap(&a.tm_s);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    load_segments(a, counts, offsets, C::kThreads);
    tc_fence_before();
    __syncthreads();
    if (warp == 2) tile_prefix_build(prefix, counts, a.mats, w_tiles, TN);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = count_tiles(prefix, a.mats, C::kThreads);
    // a.split > 1: the CTAs of a cluster share one tile, each takes a part of the contraction. The host launches a cluster for
    // every tile that segments can make which do not overlap; where they overlap and make more, each CTA takes whole tiles.
    const int split = total_tiles > (int)gridDim.x / a.split ? 1 : a.split, rank = split > 1 ? (int)cluster_ctarank() : 0;
    const int kb_lo = kb_total * rank / split, kb_hi = kb_total * (rank + 1) / split;
    const int units = (int)gridDim.x / split, unit = (int)blockIdx.x / split;
    const int stride = split > 1 ? units : balanced_stride(total_tiles, units);
    const int first = unit < stride ? unit : total_tiles;

    if (warp < 4) {
        if (warp == 0) {
            if (lane == 0) {
                uint32_t s = 0, ph = 0, slot = 0, slot_ph = 0;
                bool ok = true;
                for (int item = first; item < total_tiles && ok; item += stride) {
                    const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, TN);
                    for (int kb = kb_lo; kb < kb_hi; ++kb) {
                        if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_MMA)) {
                            ok = false;
                            break;
                        }
                        if ((kb - kb_lo) % C::kGroup == 0) {
                            if (!mbar_wait(&sc_empty[slot], slot_ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_EPI)) {
                                ok = false;
                                break;
                            }
                            mbar_expect_tx(&sc_full[slot], C::kGroup * TN * 4);
                            tma_load_2d(scales + slot * C::kGroup * TN, &a.tm_s, t.row0, kb, &sc_full[slot]);
                            if (++slot == (uint32_t)C::kSlots) { slot = 0; slot_ph ^= 1u; }
                        }
                        uint8_t* st = smem + (size_t)s * C::kStageBytes;
                        mbar_expect_tx(&full_bar[s], C::kStageBytes);
                        if (TRANS) tma_load_3d(st, &a.tm_w, t.wt * 128, kb * 128, t.e, &full_bar[s]);
                        else tma_load_3d(st, &a.tm_w, kb * 128, t.wt * 128, t.e, &full_bar[s]);
                        tma_load_2d(st + kBoxBytes, &a.tm_x, kb * 128, t.row0, &full_bar[s]);
                        if (++s == (uint32_t)C::kStages) { s = 0; ph ^= 1u; }
                    }
                }
            }
        } else if (warp == 1 || warp == 3) {
            // two issuing threads take the blocks in turn: one alone spends ~375 cycles on a block's six tcgen05 instructions
            // and as long on its waits
            if (lane == 0) {
                const uint32_t mine = warp == 1 ? 0u : 1u;
                constexpr uint32_t kStage16 = C::kStageBytes >> 4;
                const uint32_t w_lo0 = TRANS ? desc_lo_trans(smem_u32(smem)) : umma_desc_lo_sw128(smem_u32(smem));
                const uint32_t x_lo0 = umma_desc_lo_sw128(smem_u32(smem + kBoxBytes));
                constexpr uint32_t kWStep = TRANS ? kTransStep : 2u;  // K-major: 32 bytes inside the swizzle row
                uint32_t s = 0, ph = 0, acc = 0, acc_ph = 0;
                bool ok = true;
                for (int item = first; item < total_tiles && ok; item += stride) {
                    const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, TN);
                    const int n_tok = min(TN, t.count - t.nt_idx * TN);
                    const uint32_t idesc = idesc_fp8(128, (uint32_t)((n_tok + 15) & ~15), TRANS, false);
                    for (int kb = kb_lo; kb < kb_hi; ++kb) {
                        if ((s & 1u) == mine) {
                            if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_EPI) ||
                                !mbar_wait(&full_bar[s], ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            const uint32_t w_lo = w_lo0 + s * kStage16, x_lo = x_lo0 + s * kStage16;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_fp8<false>(tmem_base + acc * TN, w_lo + kk * kWStep, x_lo + kk * 2, idesc, kk ? 1u : 0u);
                            tc_commit(&empty_bar[s]);
                            tc_commit(&acc_full[acc]);
                        }
                        if (++s == (uint32_t)C::kStages) { s = 0; ph ^= 1u; }
                        if (++acc == (uint32_t)C::kAcc) { acc = 0; acc_ph ^= 1u; }
                    }
                }
            }
        }
        if (split > 1 && first < total_tiles) {  // the two barriers of the exchange below
            __syncwarp();
            cluster_sync_all();
            cluster_sync_all();
        }
    } else {
        const int q = warp & 3, part = (warp - 4) >> 2;
        const int col0 = part * C::kCols;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16) + col0;
        uint32_t acc = 0, acc_ph = 0, slot = 0, slot_ph = 0;
        bool ok = true;
        for (int item = first; item < total_tiles && ok; item += stride) {
            const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, TN);
            const int n_tok = min(TN, t.count - t.nt_idx * TN) - col0;  // this warp's live columns (may be <= 0)
            const float* ws = a.w_scale + (size_t)t.e * w_tiles * kb_total + (TRANS ? (size_t)t.wt : (size_t)t.wt * kb_total);
            float2 sum[C::kCols / 2];
#pragma unroll
            for (int j = 0; j < C::kCols / 2; ++j) sum[j] = make_float2(0.f, 0.f);
            float ws_lane = 0.f;  // the weight's scales of 32 blocks, one per lane
            for (int kb = kb_lo; kb < kb_hi; ++kb) {
                if (((kb - kb_lo) & 31) == 0) ws_lane = kb + lane < kb_hi ? ws[(size_t)(kb + lane) * (TRANS ? w_tiles : 1)] : 0.f;
                const float sw = __shfl_sync(0xffffffffu, ws_lane, (kb - kb_lo) & 31);
                const int g = (kb - kb_lo) % C::kGroup;
                if (g == 0) ok &= mbar_wait(&sc_full[slot], slot_ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA);
                ok &= mbar_wait(&acc_full[acc], acc_ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_ACC);
                tc_fence_after();
                const float4* xs = reinterpret_cast<const float4*>(scales + (slot * C::kGroup + g) * TN + col0);
                const uint32_t src = lane_addr + acc * TN;
                constexpr int kN = C::kCols / C::kChunk;
                if (n_tok > C::kCols - C::kChunk) {  // all chunks hold tokens: the next read is in flight while one is added
                    uint32_t v[2][C::kChunk];
                    tmem_read<C::kChunk>(src, v[0]);
#pragma unroll
                    for (int c = 0; c < kN; ++c) {
                        tmem_wait_for<C::kChunk>(v[c & 1]);
                        if (c + 1 < kN) tmem_read<C::kChunk>(src + (c + 1) * C::kChunk, v[(c + 1) & 1]);
                        add_scaled<C::kChunk>(sum + c * C::kChunk / 2, v[c & 1], xs + c * C::kChunk / 4, sw);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kN; ++c) {
                        if (c * C::kChunk < n_tok) {
                            uint32_t v[C::kChunk];
                            tmem_read<C::kChunk>(src + c * C::kChunk, v);
                            tmem_wait_for<C::kChunk>(v);
                            add_scaled<C::kChunk>(sum + c * C::kChunk / 2, v, xs + c * C::kChunk / 4, sw);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[acc]);
                if (++acc == (uint32_t)C::kAcc) { acc = 0; acc_ph ^= 1u; }
                if (g == C::kGroup - 1 || kb + 1 == kb_hi) {  // done with the group's scales
                    if (lane == 0) mbar_arrive(&sc_empty[slot]);
                    if (++slot == (uint32_t)C::kSlots) { slot = 0; slot_ph ^= 1u; }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (split > 1) {
                // Partial sums to the CTA that stores the column: rank r stores columns [r * TN / split, ..). Once every
                // CTA of the cluster is past its last MMA (first barrier) the pipeline's stages are free to receive them,
                // one slab per source; after the second barrier they are added in the order of the contraction.
                const int per = TN / split, shift = __ffs(per) - 1;  // both are powers of two
                float* slab = reinterpret_cast<float*>(smem);  // [split][per][128]
                __syncwarp();
                cluster_sync_all();
                const uint32_t mine = smem_u32(slab + (size_t)rank * per * 128 + q * 32 + lane);
#pragma unroll
                for (int j = 0; j < C::kCols; ++j)
                    if (j < n_tok) {
                        const int col = col0 + j;
                        st_cluster_f32(map_to_cta(mine + (uint32_t)(col & (per - 1)) * 512u, (uint32_t)(col >> shift)), j & 1 ? sum[j / 2].y : sum[j / 2].x);
                    }
                cluster_sync_all();
                if (!ok) break;
                const int lf = (threadIdx.x - 128) & 127, f = t.wt * 128 + lf;
                const int n_all = n_tok + col0 - rank * per;  // live columns of this rank
                for (int c = part; c < per && c < n_all; c += C::kEpiWarps / 4) {
                    float total = 0.f;
                    for (int r = 0; r < split; ++r) total += slab[((size_t)r * per + c) * 128 + lf];
                    if (f < a.out_features)
                        reinterpret_cast<OT*>(a.out)[(size_t)(t.row0 + rank * per + c) * a.ldo + f] = from_f32<OT>(total);
                }
                break;
            }
            if (!ok) break;
            const int f = t.wt * 128 + q * 32 + lane;
            if (f < a.out_features) {
                OT* dst = reinterpret_cast<OT*>(a.out) + (size_t)(t.row0 + col0) * a.ldo + f;
#pragma unroll
                for (int j = 0; j < C::kCols; ++j)
                    if (j < n_tok) dst[(size_t)j * a.ldo] = from_f32<OT>(j & 1 ? sum[j / 2].y : sum[j / 2].x);
            }
        }
    }

    __syncthreads();
    if (*abort_flag) {  // let copies in flight land before the shared memory is given back
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
}

// ---- 256 tokens x 256 features on CTA pairs --------------------------------------------------------------------------
// From 128 tokens per expert on the product is bound by arithmetic, and what decides is the epilogue: per block and SM
// 128 x 256 values are read from tensor memory, scaled and added. Here tokens are the MMA's M side (a lane = a token) and
// the features its N side, so a thread's token scale is one register and the weight's scale one number per warp (an
// epilogue warp owns 128 features, one scale block): one multiplication per thread and block, then one packed FMA per two
// values. With the tokens on the N side every value needs its own scale from shared memory, which the MMA's operand reads
// keep busy: 4096 x 4096 x 7168 took 210 us that way, 159 with the scale reads left out.
// Each CTA of the pair stages its 128 tokens and 128 of the 256 features: 32 KB per 128 columns of K instead of 48, which one
// CTA alone would take in and read (128 x 256 tiles on single CTAs: 165 us).
//
// What bounds it: a block takes ~1000 cycles where its MMAs take 512 (ncu: tensor pipe active 51 %, DRAM 6 %). An
// accumulator comes round again only after its MMAs, a wake-up of the epilogue, its reads and additions (430) and a wake-up
// of the issuing thread across the pair: 1000 cycles is about that round trip, as if there were one accumulator. There are
// two, which in turn should take little over half of it, so what holds a block back is not established. Halving the
// accumulators (N 128) frees them earlier but doubles the reads of the token operand: 158 to 174 us. Global loads of the
// scales inside the loop cost 125 cycles a block, hence the ring in shared memory and the lane registers. One product of
// the same size without block scales (one accumulator for the whole contraction, library call): 8192 x 4096 x 7168 in 165
// us against 242 here.
constexpr int kPairStages = 6, kPairThreads = 384, kPairEpiWarps = 8;
constexpr int kPairStageBytes = 2 * kBoxBytes;
constexpr int kPairGroup = 2, kPairSlots = 4;  // token scales: as in Cfg
// Output goes out by way of shared memory, 64 bytes of 32 rows per warp at a time: a store instruction then writes eight
// rows' 64 bytes instead of 16 bytes of 32 rows, of which the load / store unit takes one line per cycle.
constexpr int kOutBytes = 32 * 64;
constexpr size_t kPairSmem = 1024 + (size_t)kPairStages * kPairStageBytes + kPairSlots * kPairGroup * 512 + kPairEpiWarps * kOutBytes + 512 + (size_t)(3 * kMaxMats + 4) * 4;
static_assert(kPairSmem <= 232448, "shared memory");
// 128 sums and two 32-column reads per epilogue thread: these warps take registers over from the single-purpose ones. 384
// threads are launched with 168 each; 128 * 40 + 256 * 232 = 384 * 168.
constexpr int kRegsFew = 40, kRegsEpi = 232;
static_assert(128 * kRegsFew + 256 * kRegsEpi <= 384 * 168, "register pool");

__device__ __forceinline__ void add_scaled32(float2* sum, const uint32_t* v, float2 scale) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
        sum[j] = fma2(make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), scale, sum[j]);
}

template <bool TRANS, typename OT>
__global__ __launch_bounds__(kPairThreads, 1) void fp8_gemm_pair_kernel(const __grid_constant__ Fp8GemmArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* scales = reinterpret_cast<float*>(smem + (size_t)kPairStages * kPairStageBytes);  // [kPairSlots][kPairGroup][128] this CTA's tokens'
    uint8_t* out_tiles = reinterpret_cast<uint8_t*>(scales + kPairSlots * kPairGroup * 128);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(out_tiles + kPairEpiWarps * kOutBytes);
    uint64_t* empty_bar = full_bar + 8;
    uint64_t* sc_full = empty_bar + 8;
    uint64_t* sc_empty = sc_full + 4;
    uint64_t* acc_full = sc_empty + 4;   // [2] in each CTA
    uint64_t* acc_empty = acc_full + 2;  // [2] leader: both CTAs' epilogue warps
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    int* counts = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full_bar) + 512);
    int* offsets = counts + kMaxMats;
    int* prefix = offsets + kMaxMats;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const int w_blocks = (a.out_features + 127) / 128, w_tiles = (w_blocks + 1) / 2;
    const int kb_total = (a.contraction + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&full_bar[s], rank == 0 ? 2 : 1);  // leader: + the peer's report that its stage landed
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < kPairSlots; ++s) {
            mbar_init(&sc_full[s], 1);
            mbar_init(&sc_empty[s], kPairEpiWarps);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&acc_full[s], 1);
            mbar_init(&acc_empty[s], 2 * kPairEpiWarps);
        }
        *abort_flag = 0u;
        mbar_fence_init();
        prefetch_tmap(&a.tm_w);
        prefetch_tmap(&a.tm_x);
        prefetch_tmap(&a.tm_s);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    load_segments(a, counts, offsets, kPairThreads);
    tc_fence_before();
    __syncthreads();
    if (warp == 2) tile_prefix_build(prefix, counts, a.mats, w_tiles, 256);
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = count_tiles(prefix, a.mats, kPairThreads);
    const int stride = balanced_stride(total_tiles, (int)gridDim.x >> 1);
    const int first = ((int)blockIdx.x >> 1) < stride ? (int)blockIdx.x >> 1 : total_tiles;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
        if (warp == 0 && lane == 0) {
            uint32_t s = 0, ph = 0, slot = 0, slot_ph = 0;
            bool ok = true;
            for (int item = first; item < total_tiles && ok; item += stride) {
                const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, 256);
                const int f0 = t.wt * 256 + rank * 128, row = t.row0 + rank * 128;
                for (int kb = 0; kb < kb_total; ++kb) {
                    if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_MMA)) {
                        ok = false;
                        break;
                    }
                    if (kb % kPairGroup == 0) {
                        if (!mbar_wait(&sc_empty[slot], slot_ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_EPI)) {
                            ok = false;
                            break;
                        }
                        mbar_expect_tx(&sc_full[slot], kPairGroup * 512);
                        tma_load_2d(scales + slot * kPairGroup * 128, &a.tm_s, row, kb, &sc_full[slot]);
                        if (++slot == (uint32_t)kPairSlots) { slot = 0; slot_ph ^= 1u; }
                    }
                    uint8_t* st = smem + (size_t)s * kPairStageBytes;
                    mbar_expect_tx(&full_bar[s], kPairStageBytes);
                    tma_load_2d(st, &a.tm_x, kb * 128, row, &full_bar[s]);
                    if (TRANS) tma_load_3d(st + kBoxBytes, &a.tm_w, f0, kb * 128, t.e, &full_bar[s]);
                    else tma_load_3d(st + kBoxBytes, &a.tm_w, kb * 128, f0, t.e, &full_bar[s]);
                    if (++s == (uint32_t)kPairStages) { s = 0; ph ^= 1u; }
                }
            }
        } else if ((warp == 1 || warp == 3) && lane == 0 && rank == 0) {
            const uint32_t mine = warp == 1 ? 0u : 1u;  // two issuing threads take the blocks, and so the accumulators, in turn
            constexpr uint32_t kStage16 = kPairStageBytes >> 4;
            constexpr uint32_t idesc = idesc_fp8(256, 256, false, TRANS);
            constexpr uint32_t kWStep = TRANS ? kTransStep : 2u;
            const uint32_t x_lo0 = umma_desc_lo_sw128(smem_u32(smem));
            const uint32_t w_lo0 = TRANS ? desc_lo_trans(smem_u32(smem + kBoxBytes)) : umma_desc_lo_sw128(smem_u32(smem + kBoxBytes));
            uint32_t s = 0, ph = 0, acc = 0, acc_ph = 0;
            bool ok = true;
            for (int item = first; item < total_tiles && ok; item += stride) {
                for (int kb = 0; kb < kb_total; ++kb) {
                    if (acc == mine) {
                        if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_EPI) ||
                            !mbar_wait(&full_bar[s], ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t w_lo = w_lo0 + s * kStage16, x_lo = x_lo0 + s * kStage16;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_fp8<true>(tmem_base + acc * 256, x_lo + kk * 2, w_lo + kk * kWStep, idesc, kk ? 1u : 0u);
                        tc_commit_pair_mask(smem_u32(&empty_bar[s]), 3);
                        tc_commit_pair_mask(smem_u32(&acc_full[acc]), 3);
                    }
                    if (++s == (uint32_t)kPairStages) { s = 0; ph ^= 1u; }
                    acc ^= 1u;
                    acc_ph ^= acc ^ 1u;
                }
            }
        } else if (warp == 1 && lane == 0) {
            // the peer reports its landed stages to the leader
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (int item = first; item < total_tiles && ok; item += stride) {
                for (int kb = 0; kb < kb_total; ++kb) {
                    if (!mbar_wait(&full_bar[s], ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_cluster(map_to_cta(smem_u32(&full_bar[s]), 0));
                    if (++s == (uint32_t)kPairStages) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
        const int q = warp & 3, part = (warp - 4) >> 2;
        const uint32_t src0 = tmem_base + ((uint32_t)(q * 32) << 16) + part * 128;
        const uint32_t leader_empty = map_to_cta(smem_u32(acc_empty), 0);
        uint32_t acc = 0, acc_ph = 0, slot = 0, slot_ph = 0;
        const size_t ws_step = TRANS ? w_blocks : 1;
        bool ok = true;
        for (int item = first; item < total_tiles && ok; item += stride) {
            const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, 256);
            const int m = rank * 128 + q * 32 + lane;  // token of the tile
            const bool live = m < t.count - t.nt_idx * 256;
            const int fb = min(t.wt * 2 + part, w_blocks - 1);  // a block past the end: its values are not stored
            const float* ws = a.w_scale + (size_t)t.e * w_blocks * kb_total + (TRANS ? (size_t)fb : (size_t)fb * kb_total);
            float2 sum[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j] = make_float2(0.f, 0.f);
            float ws_lane = 0.f;  // the weight's scales of 32 blocks, one per lane: no global load inside the loop
            for (int kb = 0; kb < kb_total; ++kb) {
                if ((kb & 31) == 0) ws_lane = kb + lane < kb_total ? ws[(size_t)(kb + lane) * ws_step] : 0.f;
                const int g = kb % kPairGroup;
                if (g == 0 && !mbar_wait_warp(&sc_full[slot], slot_ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA)) {
                    ok = false;
                    break;
                }
                const float s = scales[(slot * kPairGroup + g) * 128 + q * 32 + lane] * __shfl_sync(0xffffffffu, ws_lane, kb & 31);
                const float2 s2 = make_float2(s, s);
                if (!mbar_wait_warp(&acc_full[acc], acc_ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_ACC)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t src = src0 + acc * 256;
                uint32_t v0[32], v1[32];
                tmem_ld32(src, v0);
                tmem_wait_for<32>(v0);
                tmem_ld32(src + 32, v1);
                add_scaled32(sum, v0, s2);
                tmem_wait_for<32>(v1);
                tmem_ld32(src + 64, v0);
                add_scaled32(sum + 16, v1, s2);
                tmem_wait_for<32>(v0);
                tmem_ld32(src + 96, v1);
                add_scaled32(sum + 32, v0, s2);
                tmem_wait_for<32>(v1);
                // everything is in registers: hand the accumulator back before the last columns are added
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(leader_empty + acc * 8u);
                acc ^= 1u;
                acc_ph ^= acc ^ 1u;
                if (g == kPairGroup - 1 || kb + 1 == kb_total) {  // done with the group's scales
                    if (lane == 0) mbar_arrive(&sc_empty[slot]);
                    if (++slot == (uint32_t)kPairSlots) { slot = 0; slot_ph ^= 1u; }
                }
                add_scaled32(sum + 48, v1, s2);
            }
            if (!ok) break;
            const int f = t.wt * 256 + part * 128;
            const int rows = min(32, t.count - t.nt_idx * 256 - (m - lane));  // this warp's live rows (may be <= 0)
            if (rows > 0 && f < a.out_features) {
                OT* dst = reinterpret_cast<OT*>(a.out) + (size_t)(t.row0 + m - lane) * a.ldo + f;
                constexpr int kVec = 16 / sizeof(OT), kChunk = 4 * kVec;
                // 16-byte piece p of row r sits at piece p ^ (r / 2) & 3: neither side meets a bank conflict
                uint8_t* tile = out_tiles + (warp - 4) * kOutBytes;
#pragma unroll
                for (int c = 0; c < 128; c += kChunk) {
                    if (a.out_vec && f + c + kChunk <= a.out_features) {
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            Pack<OT, kVec> o;
#pragma unroll
                            for (int i = 0; i < kVec; ++i) {
                                const int j = c + p * kVec + i;
                                o.v[i] = from_f32<OT>(j & 1 ? sum[j / 2].y : sum[j / 2].x);
                            }
                            *reinterpret_cast<uint4*>(tile + lane * 64 + ((p ^ (lane >> 1)) & 3) * 16) = *reinterpret_cast<const uint4*>(&o);
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = i * 8 + (lane >> 2), p = lane & 3;
                            const uint4 o = *reinterpret_cast<const uint4*>(tile + r * 64 + ((p ^ (r >> 1)) & 3) * 16);
                            if (r < rows) *reinterpret_cast<uint4*>(dst + (size_t)r * a.ldo + c + p * kVec) = o;
                        }
                        __syncwarp();
                    } else if (live) {
#pragma unroll
                        for (int j = c; j < c + kChunk; ++j)
                            if (f + j < a.out_features) dst[(size_t)lane * a.ldo + j] = from_f32<OT>(j & 1 ? sum[j / 2].y : sum[j / 2].x);
                    }
                }
            }
        }
    }

    __syncthreads();
    if (*abort_flag) {  // let copies in flight land before the shared memory is given back
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the peer's barriers and tensor memory are in use until both are here
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// Shared memory beyond the default limit has to be asked for once per kernel and device.
template <typename K>
bool allow_smem(K kernel, size_t bytes, bool* done) {
    const int dev = device_slot();
    if (dev < 0) return false;
    if (!done[dev]) done[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess;
    return done[dev];
}
// No more tiles than this can exist (the experts' rows are on the device).
size_t most_tiles(const Fp8GemmArgs& a, int tokens, int features) {
    const size_t row_tiles = (size_t)(a.rows + tokens - 1) / tokens + (a.counts ? a.mats : 0);
    return row_tiles * (size_t)((a.out_features + features - 1) / features);
}

int launch_cluster(void (*kernel)(Fp8GemmArgs), const Fp8GemmArgs& a, unsigned grid, unsigned threads, size_t smem, unsigned cluster,
                   cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess) return XMOE_OK;
    cudaGetLastError();  // reported here: the next call does not find it again
    return XMOE_ERR_CUDA;
}

template <bool TRANS, typename OT>
int launch_pair(const Fp8GemmArgs& a, cudaStream_t stream) {
    static bool smem_ok[kMaxDevices] = {};
    if (!allow_smem(fp8_gemm_pair_kernel<TRANS, OT>, kPairSmem, smem_ok)) return XMOE_ERR_CUDA;
    const size_t tiles = most_tiles(a, 256, 256), pairs = a.num_sms / 2;
    return launch_cluster(fp8_gemm_pair_kernel<TRANS, OT>, a, (unsigned)(tiles < pairs ? tiles : pairs) * 2, kPairThreads,
                          kPairSmem, 2, stream);
}
template <int TN, bool TRANS, typename OT>
int launch_t(const Fp8GemmArgs& a, cudaStream_t stream) {
    if constexpr (TN == 256) {
        return launch_pair<TRANS, OT>(a, stream);
    } else {
        static bool smem_ok[kMaxDevices] = {};
        if (!allow_smem(fp8_gemm_kernel<TN, TRANS, OT>, Cfg<TN>::kSmem, smem_ok)) return XMOE_ERR_CUDA;
        const size_t tiles = most_tiles(a, TN, 128), sms = a.num_sms;
        Fp8GemmArgs b = a;
        // fewer tiles than half the SMs: the contraction of a tile is shared by a cluster of 2, 4 or 8 CTAs
        b.split = 1;
        while (b.split < 8 && tiles * b.split * 2 <= sms && b.split * 2 * 2 <= (a.contraction + 127) / 128) b.split *= 2;
        return launch_cluster(fp8_gemm_kernel<TN, TRANS, OT>, b, (unsigned)(tiles < sms ? tiles : sms) * b.split, Cfg<TN>::kThreads, Cfg<TN>::kSmem,
                              b.split, stream);
    }
}
template <int TN>
int launch_tile(const Fp8GemmArgs& a, bool transpose, cudaStream_t stream) {
    switch (a.out_dtype) {
        case XMOE_BF16: return transpose ? launch_t<TN, true, __nv_bfloat16>(a, stream) : launch_t<TN, false, __nv_bfloat16>(a, stream);
        case XMOE_FP16: return transpose ? launch_t<TN, true, __half>(a, stream) : launch_t<TN, false, __half>(a, stream);
        case XMOE_FP32: return transpose ? launch_t<TN, true, float>(a, stream) : launch_t<TN, false, float>(a, stream);
        default: return XMOE_ERR_SHAPE;
    }
}

}  // namespace

int launch_fp8_gemm(const Fp8GemmArgs& a, int token_tile, bool transpose, cudaStream_t stream) {
    if (a.mats > kMaxMats) return XMOE_ERR_LIMIT;
    switch (token_tile) {
        case 16: return launch_tile<16>(a, transpose, stream);
        case 32: return launch_tile<32>(a, transpose, stream);
        case 64: return launch_tile<64>(a, transpose, stream);
        case 128: return launch_tile<128>(a, transpose, stream);
        case 256: return launch_tile<256>(a, transpose, stream);
        default: return XMOE_ERR_SHAPE;
    }
}

int fp8_read_status(uint32_t* host_out, cudaStream_t stream) {
    const uint32_t zero = 0u;
    if (cudaMemcpyFromSymbolAsync(host_out, g_fp8_status, 4, 0, cudaMemcpyDeviceToHost, stream) != cudaSuccess ||
        cudaMemcpyToSymbolAsync(g_fp8_status, &zero, 4, 0, cudaMemcpyHostToDevice, stream) != cudaSuccess ||
        cudaStreamSynchronize(stream) != cudaSuccess)
        return XMOE_ERR_CUDA;
    return *host_out ? XMOE_ERR_TIMEOUT : XMOE_OK;
}

}  // namespace xmoe
