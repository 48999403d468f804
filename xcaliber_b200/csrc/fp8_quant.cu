// Quantisation to 8 bits (e4m3) with one fp32 scale per 128 values: rows of activations (optionally straight into rows
// sorted by expert), the gated activation between two expert products (and its gradient), and 128 x 128 blocks of a
// weight.
//   scale = max|v| / 448 (fp32, correctly rounded),  code = e4m3(v / scale), nearest, ties to even, at most 448
// A block of zeros (or one whose scale underflows) has scale 0 and zero codes; a block that holds an infinity or a NaN
// has the scale max|v| / 448 = inf or NaN and NaN codes, so that whatever is computed from it shows it.
//
// One block of 128 is handled by 8 lanes with twice 8 values each: two coalesced 16-byte loads per lane (bf16, fp16), three
// shuffles for the maximum, two 8-byte stores. Scales are stored block-major, [ceil(cols / 128), lds], the order in which the product
// reads them: the scales of consecutive rows for one block are contiguous.
//
// Measured: fp32 8192 x 4096 31 us = 5.4 TB/s; bf16 8192 x 7168 55 us = 3.2 TB/s, fp16 45 us = 3.9 TB/s; gated activation
// of 16384 rows of 2 x 2880 58 (silu) to 69 us (clamped) = 3.4 to 4.1 TB/s, its gradient 98 to 119 us = 4.0 to 4.8 TB/s;
// weights 32 x 4096 x 7168 1.74 ms = 1.6 TB/s (load time). Rows that are not 16-byte aligned are read element by element:
// 49024 rows of 2050 bf16 in 99 us against 92 for 2048 aligned ones.
// fp32 rows are bound by bytes. With 16-bit inputs neither bytes nor instructions are at their limit: about 15 instructions
// per value (8 of them on the half-rate integer pipe) are 24 of the 55 us, the bytes 27; a warp loads, waits, computes and
// stores in turn with no load of its next step in flight, so latency is the likely rest. Ties of two codes cost a branch,
// which bf16 values with a bf16 maximum meet in one block of 14. The gated activation and its gradient are alike: issue 63
// to 67 %, DRAM 32 to 44 %.
#include "elem.cuh"
#include "kernels.h"
#include "tile_sched.cuh"

namespace xmoe {

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                  // per block of 128 values
constexpr int kUnits = kThreads / kLanes;  // blocks a CTA handles at once
constexpr int kMaxMats = 1032;
constexpr float kE4m3Max = 448.f;

__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// x / s to within half an fp32 step and 2^-44 of it (s > 0, r an approximation of 1 / s, off by 2^-22 of it at most): the
// product with r, corrected once by its residual.
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float y0 = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-y0, s, x), r, y0);
}
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN on either side is the result
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The scale of a block from its largest magnitude, and what its lanes divide with. The usual range (all but zeros,
// blocks below 2^-60 or above 2^120, infinities and NaN) takes the quotient by 448 as above: a / 448 is never nearer than
// 2^-28 of itself to the middle of two fp32 numbers, so the correction rounds it correctly.
struct BlockScale {
    float scale, r;
    bool usual;
};
__device__ __forceinline__ BlockScale block_scale(float amax) {
    BlockScale b;
    b.usual = amax == 0.f || (amax > 8.6736174e-19f && amax < 1.3292280e36f);
    if (b.usual) {
        b.scale = quotient(amax, kE4m3Max, 1.f / kE4m3Max);
        b.r = amax == 0.f ? 0.f : rcp_approx(b.scale);
    } else {
        b.scale = __fdiv_rn(amax, kE4m3Max);
        b.r = 0.f;
    }
    return b;
}
// Two neighbouring codes of which the exact x / s rounds to one, in byte j of lo and hi: the sign of x - T s, with T the
// border between them (the middle of two code values is an fp32 number, and an fma gives the sign exactly), says on
// which side it lies; on the border itself the even code is the one.
__device__ __forceinline__ uint32_t decide(uint32_t lo, uint32_t hi, float x, float s) {
    uint32_t both;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(both) : "h"((uint16_t)(lo | (hi << 8))));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&both));
    const float side = copysignf(1.f, x) * __fmaf_rn(-0.5f * (v.x + v.y), s, x);
    return side > 0.f || (side == 0.f && (lo & 1u)) ? hi : lo;
}

// Codes of N values x / s, r approximating 1 / s to 2^-23 of it. Two products bracket every quotient (the factors move
// r by 2^-21, each product adds 2^-24): where both round to the same code, so does the quotient. They differ only next to
// a border: rarely for fp32 values, more often where values and scale have few bits (bf16), so that is cheap too.
template <int N>
__device__ __forceinline__ void bracket(const float* v, float s, float r, uint32_t* code) {
    const float r_lo = r * (1.f - 4.7683716e-7f), r_hi = r * (1.f + 4.7683716e-7f);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        const float* x = v + 4 * j;
        code[j] = cvt_e4m3x2(x[0] * r_lo, x[1] * r_lo) | (cvt_e4m3x2(x[2] * r_lo, x[3] * r_lo) << 16);
        const uint32_t hi = cvt_e4m3x2(x[0] * r_hi, x[1] * r_hi) | (cvt_e4m3x2(x[2] * r_hi, x[3] * r_hi) << 16);
        if (code[j] != hi) {
            const uint32_t lo = code[j];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t l = (lo >> (8 * i)) & 0xffu, h = (hi >> (8 * i)) & 0xffu;
                if (l != h) code[j] ^= (l ^ decide(l, h, x[i], s)) << (8 * i);
            }
        }
    }
}
// An unusual block: NaN codes where the scale is not finite, 0 where it is 0; else divisor and values are first brought to
// where no product is subnormal.
__device__ __noinline__ uint32_t unusual4(float4 a, float scale) {
    if (!(scale <= 3.4028235e38f)) return 0x7f7f7f7fu;
    if (scale == 0.f) return 0u;
    const float f = scale < 1.f ? 18446744073709551616.f : 5.4210109e-20f;  // 2^64, 2^-64
    const float v[4] = {a.x * f, a.y * f, a.z * f, a.w * f}, s = scale * f;
    uint32_t code;
    bracket<4>(v, s, __frcp_rn(s), &code);
    return code;
}
// N is 8 times the pieces a lane holds
template <int N>
__device__ __forceinline__ void codes_of(const float* v, const BlockScale& b, uint32_t* code) {
    if (b.usual) {
        bracket<N>(v, b.scale, b.r, code);
    } else {
#pragma unroll
        for (int j = 0; j < N / 4; ++j) code[j] = unusual4(make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]), b.scale);
    }
}
// Sixteen values of a block, this lane's share, `m` their largest magnitude; all lanes of the block take part.
__device__ __forceinline__ void quantise16(const float* v, float m, uint32_t* code, float& scale) {
#pragma unroll
    for (int d = kLanes / 2; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    const BlockScale b = block_scale(m);
    scale = b.scale;
    codes_of<16>(v, b, code);
}
template <int N>
__device__ __forceinline__ float largest(const float* v) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) m = max_nan(m, fabsf(v[j]));
    return m;
}

// The largest magnitude of the eight values of a 16-byte piece of 16-bit values, two at a time (a NaN is the result).
__device__ __forceinline__ float largest8(const Pack<__nv_bfloat16, 8>& k) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&k);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
    return max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float largest8(const Pack<__half, 8>& k) {
    const __half2* p = reinterpret_cast<const __half2*>(&k);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
    return max_nan(__low2float(m), __high2float(m));
}
// Eight consecutive values of a row from column `col`, zero beyond `cols`, and their largest magnitude. VEC: the row is
// 16-byte aligned at col.
template <typename T, bool VEC>
__device__ __forceinline__ float load8(const T* row, int col, int cols, float* v) {
    if (VEC && col + 8 <= cols) {
        constexpr int P = 16 / sizeof(T);
        float m = 0.f;
#pragma unroll
        for (int p = 0; p < 8 / P; ++p) {
            const Pack<T, P> k = load_pack_once<T, P>(row + col + p * P);
#pragma unroll
            for (int j = 0; j < P; ++j) v[p * P + j] = to_f32<T>(k.v[j]);
            if constexpr (P == 8) m = largest8(k);
            else m = max_nan(m, largest<P>(v + p * P));
        }
        return m;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? to_f32<T>(row[col + j]) : 0.f;
    return largest<8>(v);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int col, int cols, const float* v) {
    if (VEC && col + 8 <= cols) {
        constexpr int P = 16 / sizeof(T);
#pragma unroll
        for (int p = 0; p < 8 / P; ++p) {
            Pack<T, P> k;
#pragma unroll
            for (int j = 0; j < P; ++j) k.v[j] = from_f32<T>(v[p * P + j]);
            store_pack<T, P>(row + col + p * P, k);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < cols) row[col + j] = from_f32<T>(v[j]);
    }
}
// code rows start at multiples of 16 bytes, so eight codes from a multiple of 8 are one aligned store
__device__ __forceinline__ void store_codes(uint8_t* row, int col, int cols, const uint32_t* c) {
    if (col + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + col) = make_uint2(c[0], c[1]);
    } else {
        const unsigned long long w = ((unsigned long long)c[1] << 32) | c[0];
        for (int j = 0; col + j < cols; ++j) row[col + j] = (uint8_t)(w >> (8 * j));
    }
}

// The blocks of a matrix row by row, handed out to the CTA's kUnits groups of lanes in turn: group u takes blocks u, u +
// kUnits, .. of the CTA's share. Steps of kUnits blocks are a fixed number of rows and blocks: no division follows the first.
struct Walk {
    int row, kb;
    __device__ __forceinline__ void step(int rows, int blocks, int kb_total) {
        row += rows;
        kb += blocks;
        if (kb >= kb_total) {
            kb -= kb_total;
            ++row;
        }
    }
};

template <typename T, bool VEC, bool SORTED>
__global__ __launch_bounds__(kThreads) void fp8_quant_kernel(const Fp8QuantArgs a, int kb_total, int share) {
    const int unit = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const T* x = reinterpret_cast<const T*>(a.x);
    const uint32_t first = blockIdx.x * (uint32_t)share + unit;  // 2^32 blocks of 128 values would not fit the memory
    Walk w{(int)(first / (uint32_t)kb_total), (int)(first % (uint32_t)kb_total)};
    const int d_row = kUnits / kb_total, d_kb = kUnits % kb_total;
    // every group takes the same number of steps (the shuffles need all lanes of a warp): a block past the last row loads
    // and stores nothing
    for (int i = 0; i < share; i += kUnits, w.step(d_row, d_kb, kb_total)) {
        const int t = w.row, kb = w.kb, col = kb * 128 + lane * 8;
        const bool on = t < a.rows;
        const T* row = x + (size_t)(on ? t : 0) * a.ldx;
        const int cols = on ? a.cols : 0;
        float v[16];
        const float m = max_nan(load8<T, VEC>(row, col, cols, v), load8<T, VEC>(row, col + 64, cols, v + 8));
        // a sorted row's slots, one per lane, on their way while the block is quantised
        const int32_t* idx = a.topk_row + (size_t)(on ? t : 0) * a.idx_stride;
        int mine = SORTED && lane < a.k ? idx[lane] : -1;
        uint32_t code[4];
        float scale;
        quantise16(v, m, code, scale);
        auto store = [&](int r) {
            uint8_t* q = a.q + (size_t)r * a.ldq;
            store_codes(q, col, a.cols, code);
            store_codes(q, col + 64, a.cols, code + 2);
            if (lane == 0) a.scale[(size_t)kb * a.lds + r] = scale;
        };
        if (!SORTED) {
            if (on) store(t);
            continue;
        }
#pragma unroll 1
        for (int s = 0; s < a.k; ++s) {
            if (s && s % kLanes == 0) mine = s + lane < a.k ? idx[s + lane] : -1;
            const int r = __shfl_sync(0xffffffffu, mine, s % kLanes, kLanes);
            if (on && r >= 0 && r < a.num_rows) store(r);
        }
    }
}

// ---- gated activations: v = act(g) * u ------------------------------------------------------------------------------
// ACT 0: silu(g) * u;  1: min(g, limit) * sigmoid(alpha * min(g, limit)) * (clamp(u, -limit, limit) + 1);
// 2: gelu_tanh(g) * u, written as g * sigmoid(2 z) (z the tanh's argument): no cancellation for negative g. NaN passes.
// The sigmoid is 1 / (1 + 2^(-z log2 e)) with the exponential and reciprocal units (2^-22 and 2^-23 relative); the rounded
// exponent adds |z| 2^-23.
__device__ __forceinline__ float sigmoid(float z) { return rcp_approx(1.f + ex2_approx(z * -1.4426950408889634f)); }
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f;

template <int ACT>
__device__ __forceinline__ float glu_value(float g, float u, float alpha, float limit) {
    if (ACT == 1) {
        g = g > limit ? limit : g;
        u = u > limit ? limit : (u < -limit ? -limit : u);
        return g * sigmoid(alpha * g) * (u + 1.f);
    }
    if (ACT == 2) return g * sigmoid(2.f * kGeluC * (g + kGeluA * g * g * g)) * u;
    return g * sigmoid(g) * u;
}
// The derivative has a factor z' (1 - s) or z (1 - s) that goes to zero as z grows; z is kept inside where s is still neither
// 0 nor 1 or has just become it, so that the factor is that zero instead of infinity times zero (NaN) for huge gates.
template <int ACT>
__device__ __forceinline__ void glu_gradient(float g, float u, float da, float alpha, float limit, float& dg, float& du) {
    if (ACT == 1) {
        const bool in_g = g <= limit, in_u = fabsf(u) <= limit;
        const float gc = g > limit ? limit : g, uc = u > limit ? limit : (u < -limit ? -limit : u);
        const float z = alpha * gc, s = sigmoid(z);
        dg = in_g ? da * (uc + 1.f) * s * (1.f + fminf(fmaxf(z, -256.f), 256.f) * (1.f - s)) : 0.f;
        du = in_u ? da * gc * s : 0.f;
    } else if (ACT == 2) {
        const float s = sigmoid(2.f * kGeluC * (g + kGeluA * g * g * g));
        const float gc = fminf(fmaxf(g, -64.f), 64.f);
        dg = da * u * s * (1.f + 2.f * kGeluC * gc * (1.f + 3.f * kGeluA * gc * gc) * (1.f - s));
        du = da * g * s;
    } else {
        const float s = sigmoid(g);
        dg = da * u * s * (1.f + g * (1.f - s));
        du = da * g * s;
    }
}

// Live rows only: with expert segments the rows between an expert's last and the next multiple of 128 hold nothing and are
// neither read nor written. The live rows are numbered through; every CTA takes an equal, contiguous share of their blocks
// and finds its first expert once.
template <typename T, bool VEC, int ACT, bool BACKWARD>
__global__ __launch_bounds__(kThreads, BACKWARD ? 5 : 4) void glu_kernel(const Fp8QuantArgs a, int kb_total) {
    // the gradient has no block to share a scale: 16 lanes with 8 values, for more warps in flight
    constexpr int kP = BACKWARD ? 1 : 2, kLanes = 16 / kP, kUnits = kThreads / kLanes;
    __shared__ int before[kMaxMats + 1];  // live rows of the experts before e
    __shared__ int shift[kMaxMats];       // the experts' counts, then: buffer row - live row, within expert e
    const int mats = a.counts ? a.e_tot : 1;
    // segments are kept inside the rows: one that starts outside counts as empty, one that runs past the end is cut
    for (int e = threadIdx.x; e < mats; e += kThreads) {
        const int c = a.counts ? a.counts[e] : a.rows, o = a.counts ? a.offsets[e] : 0;
        shift[e] = o < 0 || o >= a.rows ? 0 : max(min(c, a.rows - o), 0);
    }
    __syncthreads();
    if (threadIdx.x < 32) tile_prefix_build(before, shift, mats, 1, 1);
    __syncthreads();
    for (int e = threadIdx.x; e < mats; e += kThreads) shift[e] = (a.counts ? a.offsets[e] : 0) - before[e];
    __syncthreads();
    const int live = max(before[mats], 0);
    const size_t blocks = (size_t)live * kb_total;
    const size_t share = ((blocks + gridDim.x - 1) / gridDim.x + kUnits - 1) / kUnits * kUnits;
    const size_t begin = blockIdx.x * share;
    if (begin >= blocks) return;
    const int steps = (int)(((begin + share < blocks ? share : blocks - begin) + kUnits - 1) / kUnits);
    const int unit = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    Walk w{(int)((begin + unit) / kb_total), (int)((begin + unit) % kb_total)};
    const int d_row = kUnits / kb_total, d_kb = kUnits % kb_total;
    int e = 0;
    for (int hi = mats; hi - e > 1;) {  // largest e with before[e] <= row
        const int mid = (e + hi) >> 1;
        if (before[mid] <= w.row) e = mid; else hi = mid;
    }
    const T* h = reinterpret_cast<const T*>(a.x);
    for (int i = 0; i < steps; ++i, w.step(d_row, d_kb, kb_total)) {
        while (e + 1 < mats && before[e + 1] <= w.row) ++e;
        const int r = w.row + shift[e], kb = w.kb, col = kb * 128 + lane * 8;
        const bool on = w.row < live && r >= 0 && r < a.rows;
        const size_t at = on ? r : 0;
        const int cols = on ? a.cols : 0;
        const T* row = h + at * a.ldx;
        float g[8 * kP], u[8 * kP];
#pragma unroll
        for (int p = 0; p < kP; ++p) {
            load8<T, VEC>(row, col + p * 64, cols, g + 8 * p);
            load8<T, VEC>(row + a.cols, col + p * 64, cols, u + 8 * p);
        }
        if constexpr (BACKWARD) {
            float d[8];
            load8<T, VEC>(reinterpret_cast<const T*>(a.da) + at * a.cols, col, cols, d);
#pragma unroll
            for (int j = 0; j < 8; ++j) glu_gradient<ACT>(g[j], u[j], d[j], a.alpha, a.limit, g[j], u[j]);
            T* out = reinterpret_cast<T*>(a.dh) + at * 2 * a.cols;
            store8<T, VEC>(out, col, cols, g);
            store8<T, VEC>(out + a.cols, col, cols, u);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) g[j] = glu_value<ACT>(g[j], u[j], a.alpha, a.limit);
            if (col + 72 > cols) {  // columns past the last take no part in the block's maximum
#pragma unroll
                for (int j = 0; j < 16; ++j) g[j] = col + (j < 8 ? j : j + 56) < cols ? g[j] : 0.f;
            }
            uint32_t code[4];
            float scale;
            quantise16(g, largest<16>(g), code, scale);
            if (on) {
                uint8_t* q = a.q + at * a.ldq;
                store_codes(q, col, cols, code);
                store_codes(q, col + 64, cols, code + 2);
                if (lane == 0) a.scale[(size_t)kb * a.lds + r] = scale;
            }
        }
    }
}

// One CTA per 128 x 128 block of a weight (load time): every thread keeps eight pieces of eight values in registers.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void fp8_quant_weight_kernel(const T* __restrict__ w, int n, int k, int nb, int kb,
                                                                    uint8_t* __restrict__ q, int ldq,
                                                                    float* __restrict__ scale) {
    __shared__ float warp_max[kThreads / 32];
    const size_t block = blockIdx.x;
    const int bk = (int)(block % kb), bn = (int)(block / kb % nb);
    const size_t mat = block / kb / nb;
    const int rows = min(128, n - bn * 128), col = bk * 128 + (threadIdx.x & 15) * 8, row = threadIdx.x >> 4;
    const T* src = w + (mat * n + (size_t)bn * 128) * k;
    float v[8][8], m = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int r = p * 16 + row;
        m = max_nan(m, load8<T, VEC>(src + (size_t)(r < rows ? r : 0) * k, r < rows ? col : 0, r < rows ? k : 0, v[p]));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) m = max_nan(m, warp_max[i]);
    const BlockScale b = block_scale(m);
    if (threadIdx.x == 0) scale[block] = b.scale;
    uint8_t* dst = q + (mat * n + (size_t)bn * 128) * ldq;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int r = p * 16 + row;
        uint32_t code[2];
        codes_of<8>(v[p], b, code);
        if (r < rows) store_codes(dst + (size_t)r * ldq, col, k, code);
    }
}

template <typename T>
bool rows_aligned(const void* p, size_t ld) { return ((uintptr_t)p & 15u) == 0 && ld * sizeof(T) % 16 == 0; }

template <typename T, bool VEC>
int quant_v(const Fp8QuantArgs& a, cudaStream_t stream) {
    const int kb = (a.cols + 127) / 128;
    const size_t blocks = (size_t)a.rows * kb;
    // four blocks per group of lanes; small calls one, so that every SM has some
    const int share = blocks >= (size_t)148 * 8 * kUnits ? 4 * kUnits : kUnits;
    const size_t grid = (blocks + share - 1) / share;
    if (grid > 0x7fffffffu) return XMOE_ERR_LIMIT;
    if (a.topk_row) fp8_quant_kernel<T, VEC, true><<<(unsigned)grid, kThreads, 0, stream>>>(a, kb, share);
    else fp8_quant_kernel<T, VEC, false><<<(unsigned)grid, kThreads, 0, stream>>>(a, kb, share);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}
template <typename T>
int quant_t(const Fp8QuantArgs& a, cudaStream_t stream) {
    return rows_aligned<T>(a.x, a.ldx) ? quant_v<T, true>(a, stream) : quant_v<T, false>(a, stream);
}

template <typename T, int ACT, bool BACKWARD>
int glu_act(const Fp8QuantArgs& a, cudaStream_t stream) {
    const int kb = (a.cols + 127) / 128;
    const size_t ctas = ((size_t)a.rows * kb + kUnits - 1) / kUnits, most = 148 * (BACKWARD ? 5 : 4);
    const unsigned grid = (unsigned)(ctas < most ? ctas : most);
    const bool vec = rows_aligned<T>(a.x, a.ldx) && a.cols * sizeof(T) % 16 == 0 &&
                     (!BACKWARD || (((uintptr_t)a.da | (uintptr_t)a.dh) & 15u) == 0);
    if (vec) glu_kernel<T, true, ACT, BACKWARD><<<grid, kThreads, 0, stream>>>(a, kb);
    else glu_kernel<T, false, ACT, BACKWARD><<<grid, kThreads, 0, stream>>>(a, kb);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}
template <typename T, bool BACKWARD>
int glu_t(const Fp8QuantArgs& a, cudaStream_t stream) {
    switch (a.activation) {
        case 0: return glu_act<T, 0, BACKWARD>(a, stream);
        case 1: return glu_act<T, 1, BACKWARD>(a, stream);
        case 2: return glu_act<T, 2, BACKWARD>(a, stream);
        default: return XMOE_ERR_SHAPE;
    }
}
template <typename T>
int quant_weight_t(const void* w, int mats, int n, int k, uint8_t* q, int ldq, float* scale, cudaStream_t stream) {
    const int nb = (n + 127) / 128, kb = (k + 127) / 128;
    const size_t blocks = (size_t)mats * nb * kb;
    if (blocks > 0x7fffffffu) return XMOE_ERR_LIMIT;
    if (rows_aligned<T>(w, k)) fp8_quant_weight_kernel<T, true><<<(unsigned)blocks, kThreads, 0, stream>>>((const T*)w, n, k, nb, kb, q, ldq, scale);
    else fp8_quant_weight_kernel<T, false><<<(unsigned)blocks, kThreads, 0, stream>>>((const T*)w, n, k, nb, kb, q, ldq, scale);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}

#define XMOE_BY_TYPE(dt, call)                       \
    switch (dt) {                                    \
        case XMOE_BF16: return call(__nv_bfloat16);  \
        case XMOE_FP16: return call(__half);         \
        case XMOE_FP32: return call(float);          \
        default: return XMOE_ERR_SHAPE;              \
    }

}  // namespace

int launch_fp8_quant(const Fp8QuantArgs& a, cudaStream_t stream) {
#define XMOE_CALL(T) quant_t<T>(a, stream)
    XMOE_BY_TYPE(a.dtype, XMOE_CALL)
#undef XMOE_CALL
}
int launch_glu_fp8_quant(const Fp8QuantArgs& a, cudaStream_t stream) {
#define XMOE_CALL(T) glu_t<T, false>(a, stream)
    XMOE_BY_TYPE(a.dtype, XMOE_CALL)
#undef XMOE_CALL
}
int launch_glu_backward(const Fp8QuantArgs& a, cudaStream_t stream) {
#define XMOE_CALL(T) glu_t<T, true>(a, stream)
    XMOE_BY_TYPE(a.dtype, XMOE_CALL)
#undef XMOE_CALL
}
int launch_fp8_quant_weight(const void* w, int dtype, int mats, int n, int k, uint8_t* q, int ldq, float* scale,
                            cudaStream_t stream) {
#define XMOE_CALL(T) quant_weight_t<T>(w, mats, n, k, q, ldq, scale, stream)
    XMOE_BY_TYPE(dtype, XMOE_CALL)
#undef XMOE_CALL
}

}  // namespace xmoe
