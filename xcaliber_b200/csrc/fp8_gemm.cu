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
// 128 output features (weight rows, or columns under TRANS) are the MMA's M side and the tokens its N side: the
// weight's scale is one number per tile and block, ragged token counts only narrow the MMA, and a decode batch of a few
// tokens costs a narrow MMA instead of a mostly empty one. TRANS reads the same 128 x 128 weight box from shared memory
// with the operand's transpose bit (features contiguous), so one copy of the weight serves both directions.
//
// Roles: warp 0 TMA producer, warp 1 tensor-memory owner and MMA issuer, warps 4.. epilogue (two per lane quadrant from
// 128 tokens on). Every wait is bounded; a wait that gives up is reported by xmoe_fp8_status.
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

__device__ __forceinline__ void mma_fp8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128)
        : "memory");
}
// kind::f8f6f4: accumulator fp32 [4,6) = 1, a/b format e4m3 = 0, transposed A [15], N>>3 [17,23), M>>4 [24,29)
__host__ __device__ constexpr uint32_t idesc_fp8(uint32_t m, uint32_t n, bool a_trans) {
    return (1u << 4) | ((a_trans ? 1u : 0u) << 15) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
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
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

template <int TN>
struct Cfg {
    static constexpr int kEpiWarps = TN >= 128 ? 8 : 4;
    static constexpr int kThreads = 128 + 32 * kEpiWarps;
    static constexpr int kCols = TN / (kEpiWarps / 4);            // token columns per epilogue warp
    static constexpr int kChunk = kCols < 32 ? 16 : 32;           // columns per tensor-memory read
    static constexpr int kAcc = TN >= 256 ? 2 : 4;                // accumulators in tensor memory
    static constexpr int kTmemCols = kAcc * TN < 64 ? 64 : kAcc * TN;
    static constexpr int kStageBytes = kBoxBytes + TN * 128;
    static constexpr int kStages = TN >= 256 ? 4 : (TN >= 128 ? 6 : (TN >= 64 ? 8 : 10));
    // a scale slot is written again kStages + kAcc blocks later: by then the MMA of the block that used the stage
    // kStages blocks ago has been issued, so the epilogue has drained the block kAcc before that one
    static constexpr int kScaleSlots = kStages + kAcc;
    static constexpr size_t kTail = (size_t)kScaleSlots * TN * 4 + 1024;
    static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kTail + (size_t)(3 * kMaxMats + 4) * 4;
    static_assert(kSmem <= 232448, "shared memory");
    static_assert(kTmemCols <= 512, "tensor memory");
};

template <int TN, bool TRANS, typename OT>
__global__ __launch_bounds__(Cfg<TN>::kThreads, 1) void fp8_gemm_kernel(const __grid_constant__ Fp8GemmArgs a) {
    using C = Cfg<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* scales = reinterpret_cast<float*>(smem + (size_t)C::kStages * C::kStageBytes);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(scales + C::kScaleSlots * TN);
    uint64_t* empty_bar = full_bar + 16;
    uint64_t* sc_full = empty_bar + 16;  // [kScaleSlots]
    uint64_t* acc_full = sc_full + 16;
    uint64_t* acc_empty = acc_full + 4;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 4);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    int* counts = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full_bar) + 1024);
    int* offsets = counts + kMaxMats;
    int* prefix = offsets + kMaxMats;
    static_assert(C::kScaleSlots <= 16, "barrier block");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w_tiles = (a.out_features + 127) / 128;
    const int kb_total = (a.contraction + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < C::kScaleSlots; ++s) mbar_init(&sc_full[s], 1);
        for (int s = 0; s < C::kAcc; ++s) {
            mbar_init(&acc_full[s], 1);
            mbar_init(&acc_empty[s], C::kEpiWarps);
        }
        *abort_flag = 0u;
        mbar_fence_init();
        prefetch_tmap(&a.tm_w);
        prefetch_tmap(&a.tm_x);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    // the experts' segments, kept inside the buffers: a segment that does not start at a multiple of 16 rows inside
    // them counts as empty (and is reported), one that runs past the end is cut
    for (int e = threadIdx.x; e < a.mats; e += C::kThreads) {
        int c = a.counts ? a.counts[e] : a.rows, o = a.counts ? a.offsets[e] : 0;
        if (c > 0 && (o < 0 || o >= a.rows || (o & 15))) {
            atomicCAS(&g_fp8_status, 0u, kBadSegment);
            c = 0;
        }
        counts[e] = c <= 0 ? 0 : min(c, a.rows - o);
        offsets[e] = o;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) tile_prefix_build(prefix, counts, a.mats, w_tiles, TN);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = prefix[a.mats];
    const int stride = balanced_stride(total_tiles, gridDim.x);
    const int first = (int)blockIdx.x < stride ? (int)blockIdx.x : total_tiles;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0, slot = 0;
            bool ok = true;
            for (int item = first; item < total_tiles && ok; item += stride) {
                const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, TN);
                // scales of this tile's tokens: a multiple of 16 bytes, inside the block's row (lds >= rows, both ends
                // multiples of 4)
                const uint32_t sc_bytes = (uint32_t)min(TN, ((a.rows + 3) & ~3) - t.row0) * 4u;
                const float* sc = a.x_scale + t.row0;
                for (int kb = 0; kb < kb_total; ++kb) {
                    if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_MMA)) {
                        ok = false;
                        break;
                    }
                    uint8_t* st = smem + (size_t)s * C::kStageBytes;
                    mbar_expect_tx(&full_bar[s], C::kStageBytes);
                    if (TRANS) tma_load_3d(st, &a.tm_w, t.wt * 128, kb * 128, t.e, &full_bar[s]);
                    else tma_load_3d(st, &a.tm_w, kb * 128, t.wt * 128, t.e, &full_bar[s]);
                    tma_load_2d(st + kBoxBytes, &a.tm_x, kb * 128, t.row0, &full_bar[s]);
                    mbar_expect_tx(&sc_full[slot], sc_bytes);
                    tma_load_1d(scales + slot * TN, sc + (size_t)kb * a.lds, sc_bytes, &sc_full[slot]);
                    if (++s == (uint32_t)C::kStages) { s = 0; ph ^= 1u; }
                    if (++slot == (uint32_t)C::kScaleSlots) slot = 0;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t kStage16 = C::kStageBytes >> 4;
            // K-major: 32 values further along K are 32 bytes inside the swizzle row. TRANS: features are contiguous,
            // a K step of 32 is 32 rows of 128 bytes; both stride fields are the 1024 bytes between 8-row groups (the
            // tile is one swizzle atom wide, so only one of them is used).
            const uint32_t w_lo0 = TRANS ? ((smem_u32(smem) & 0x3ffffu) >> 4) | ((1024u >> 4) << 16) : umma_desc_lo_sw128(smem_u32(smem));
            const uint32_t x_lo0 = umma_desc_lo_sw128(smem_u32(smem + kBoxBytes));
            constexpr uint32_t kWStep = TRANS ? (32u * 128u) >> 4 : 2u;
            uint32_t s = 0, ph = 0, acc = 0, acc_ph = 0;
            bool ok = true;
            for (int item = first; item < total_tiles && ok; item += stride) {
                const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, TN);
                const int n_mma = (min(TN, t.count - t.nt_idx * TN) + 15) & ~15;
                const uint32_t idesc = idesc_fp8(128, (uint32_t)n_mma, TRANS);
                for (int kb = 0; kb < kb_total; ++kb) {
                    if (!mbar_wait(&acc_empty[acc], acc_ph ^ 1u, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_EPI) ||
                        !mbar_wait(&full_bar[s], ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t w_lo = w_lo0 + s * kStage16, x_lo = x_lo0 + s * kStage16;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        mma_fp8(tmem_base + acc * TN, w_lo + kk * kWStep, x_lo + kk * 2, idesc, kk ? 1u : 0u);
                    tc_commit(&empty_bar[s]);
                    tc_commit(&acc_full[acc]);
                    if (++s == (uint32_t)C::kStages) { s = 0; ph ^= 1u; }
                    if (++acc == (uint32_t)C::kAcc) { acc = 0; acc_ph ^= 1u; }
                }
            }
        }
    } else if (warp >= 4) {
        const int q = warp & 3, part = (warp - 4) >> 2;
        const int col0 = part * C::kCols;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16) + col0;
        const int ws_ld = TRANS ? w_tiles : kb_total;  // row length of a matrix's scale table
        uint32_t acc = 0, acc_ph = 0, slot = 0, slot_ph = 0;
        bool ok = true;
        for (int item = first; item < total_tiles && ok; item += stride) {
            const TileInfo t = tile_decode(item, prefix, counts, offsets, a.mats, TN);
            const int n_tok = min(TN, t.count - t.nt_idx * TN) - col0;  // this warp's live columns (may be <= 0)
            const float* ws = a.w_scale + (size_t)t.e * w_tiles * kb_total + (TRANS ? t.wt : t.wt * ws_ld);
            float2 sum[C::kCols / 2];
#pragma unroll
            for (int j = 0; j < C::kCols / 2; ++j) sum[j] = make_float2(0.f, 0.f);
            float ws_lane = 0.f;
            for (int kb = 0; kb < kb_total; ++kb) {
                if ((kb & 31) == 0) ws_lane = kb + lane < kb_total ? ws[(size_t)(kb + lane) * (TRANS ? ws_ld : 1)] : 0.f;
                const float sw = __shfl_sync(0xffffffffu, ws_lane, kb & 31);
                if (!mbar_wait(&sc_full[slot], slot_ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_TMA) ||
                    !mbar_wait(&acc_full[acc], acc_ph, abort_flag, &g_fp8_status, XMOE_DEV_TIMEOUT_ACC)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float4* xs = reinterpret_cast<const float4*>(scales + slot * TN + col0);
#pragma unroll
                for (int c = 0; c < C::kCols / C::kChunk; ++c) {
                    if (c * C::kChunk < n_tok) {
                        uint32_t v[C::kChunk];
                        if (C::kChunk == 32) tmem_ld32(lane_addr + acc * TN + c * C::kChunk, v);
                        else tmem_ld16(lane_addr + acc * TN + c * C::kChunk, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < C::kChunk / 4; ++j) {
                            const float4 x4 = xs[c * (C::kChunk / 4) + j];
                            float2* d = &sum[(c * C::kChunk + 4 * j) / 2];
                            const float2 sw2 = make_float2(sw, sw);
                            d[0] = fma2(make_float2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])),
                                        mul2(make_float2(x4.x, x4.y), sw2), d[0]);
                            d[1] = fma2(make_float2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])),
                                        mul2(make_float2(x4.z, x4.w), sw2), d[1]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[acc]);
                if (++acc == (uint32_t)C::kAcc) { acc = 0; acc_ph ^= 1u; }
                if (++slot == (uint32_t)C::kScaleSlots) { slot = 0; slot_ph ^= 1u; }
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

template <int TN, bool TRANS, typename OT>
int launch_t(const Fp8GemmArgs& a, cudaStream_t stream) {
    static bool attr_set_dev[kMaxDevices] = {};
    const int dev = device_slot();
    if (dev < 0) return XMOE_ERR_CUDA;
    if (!attr_set_dev[dev]) {
        if (cudaFuncSetAttribute(fp8_gemm_kernel<TN, TRANS, OT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Cfg<TN>::kSmem) != cudaSuccess)
            return XMOE_ERR_CUDA;
        attr_set_dev[dev] = true;
    }
    // no more CTAs than there can be tiles
    const size_t row_tiles = (size_t)(a.rows + TN - 1) / TN + (a.counts ? a.mats : 0);
    const size_t tiles = row_tiles * (size_t)((a.out_features + 127) / 128);
    const int grid = tiles < (size_t)a.num_sms ? (int)tiles : a.num_sms;
    fp8_gemm_kernel<TN, TRANS, OT><<<grid, Cfg<TN>::kThreads, Cfg<TN>::kSmem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}
template <int TN, bool TRANS>
int launch_out(const Fp8GemmArgs& a, cudaStream_t stream) {
    switch (a.out_dtype) {
        case XMOE_BF16: return launch_t<TN, TRANS, __nv_bfloat16>(a, stream);
        case XMOE_FP16: return launch_t<TN, TRANS, __half>(a, stream);
        case XMOE_FP32: return launch_t<TN, TRANS, float>(a, stream);
        default: return XMOE_ERR_SHAPE;
    }
}
template <int TN>
int launch_dir(const Fp8GemmArgs& a, bool transpose, cudaStream_t stream) {
    return transpose ? launch_out<TN, true>(a, stream) : launch_out<TN, false>(a, stream);
}

}  // namespace

int launch_fp8_gemm(const Fp8GemmArgs& a, int token_tile, bool transpose, cudaStream_t stream) {
    if (a.mats > kMaxMats) return XMOE_ERR_LIMIT;
    switch (token_tile) {
        case 16: return launch_dir<16>(a, transpose, stream);
        case 32: return launch_dir<32>(a, transpose, stream);
        case 64: return launch_dir<64>(a, transpose, stream);
        case 128: return launch_dir<128>(a, transpose, stream);
        case 256: return launch_dir<256>(a, transpose, stream);
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
