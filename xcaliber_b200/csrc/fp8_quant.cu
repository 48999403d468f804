// Quantisation to 8 bits (e4m3) with one fp32 scale per 128 values: rows of activations (optionally straight into rows
// sorted by expert), the gated activation between two expert products (and its gradient), and 128 x 128 blocks of a
// weight.
//   scale = max|v| / 448 (fp32, correctly rounded),  code = e4m3(v / scale), nearest, ties to even, at most 448
// A block of zeros (or one whose scale underflows) has scale 0 and zero codes; a block that holds an infinity or a NaN
// has the scale max|v| / 448 = inf or NaN and NaN codes, so that whatever is computed from it shows it.
//
// One block of 128 is handled by 16 lanes with 8 values each: a 16-byte load per lane (bf16, fp16), four shuffles for
// the maximum, an 8-byte store. Scales are stored block-major, [ceil(cols / 128), lds], the order in which the product
// reads them: the scales of consecutive rows for one block are contiguous.
#include "elem.cuh"
#include "kernels.h"
#include "tile_sched.cuh"

namespace xmoe {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = kThreads / 16;  // 128-value blocks a CTA handles at once
constexpr int kMaxMats = 1032;
constexpr float kE4m3Max = 448.f;

__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// A value that rounds to e4m3 the way the exact quotient a / s does (a >= 0, s > 0, r = 1 / s rounded to nearest).
// y = a * r with one correction by its residual is a / s to within half an fp32 step (plus 2^-47 of it), so it lies on
// the same side of every border between two codes as a / s, or exactly on the border: borders have five significant
// bits and are fp32 numbers. On a border (low mantissa bits as tested) the sign of the residual a - y * s, which an fma
// gives exactly, says on which side a / s lies; y then moves one fp32 step that way.
__device__ __forceinline__ float quotient_for_e4m3(float a, float s, float r) {
    const float y0 = __fmul_rn(a, r);
    const float y = __fmaf_rn(__fmaf_rn(-y0, s, a), r, y0);
    uint32_t bits = __float_as_uint(y);
    // normal codes: a 1 followed by 19 zeros below the three mantissa bits; subnormal codes: odd multiples of 2^-10
    if ((bits & 0xfffffu) == (y >= 0.015625f ? 0x80000u : 0u) && bits != 0u) {
        const float e = __fmaf_rn(-y, s, a);
        bits = e > 0.f ? bits + 1u : (e < 0.f ? bits - 1u : bits);
    }
    return __uint_as_float(bits);
}

// The block's scale from the bits of its largest magnitude, and what the lanes need to quantise with it.
struct BlockScale {
    float scale;        // stored
    float s, r, shift;  // divisor, its reciprocal, power of two that keeps small blocks away from subnormal products
    bool finite;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits) {
    BlockScale b;
    b.finite = amax_bits < 0x7f800000u;
    b.scale = __fdiv_rn(__uint_as_float(amax_bits), kE4m3Max);
    b.shift = b.scale < 8.6736174e-19f ? 18446744073709551616.f : 1.f;  // below 2^-60: times 2^64
    b.s = __fmul_rn(b.scale, b.shift);
    b.r = b.scale > 0.f ? __frcp_rn(b.s) : 0.f;
    return b;
}

// Eight values of a block, this lane's share; all 16 lanes of the block take part. Returns eight codes.
__device__ __forceinline__ uint2 quantise8(const float* v, float& scale) {
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);  // NaN > inf > every finite value
#pragma unroll
    for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    const BlockScale b = block_scale(m);
    scale = b.scale;
    if (!b.finite) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = v[2 * j + i];
            y[i] = copysignf(quotient_for_e4m3(fabsf(x) * b.shift, b.s, b.r), x);
        }
        c[j] = cvt_e4m3x2(y[0], y[1]);
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// Eight consecutive values of a row from column `col`, zero beyond `cols`. VEC: the row is 16-byte aligned at col.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int col, int cols, float* v) {
    if (VEC && col + 8 <= cols) {
        constexpr int P = 16 / sizeof(T);
#pragma unroll
        for (int p = 0; p < 8 / P; ++p) {
            const Pack<T, P> k = load_pack_once<T, P>(row + col + p * P);
#pragma unroll
            for (int j = 0; j < P; ++j) v[p * P + j] = to_f32<T>(k.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? to_f32<T>(row[col + j]) : 0.f;
    }
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
__device__ __forceinline__ void store_codes(uint8_t* row, int col, int cols, uint2 c) {
    if (col + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + col) = c;
    } else {
        const unsigned long long w = ((unsigned long long)c.y << 32) | c.x;
        for (int j = 0; col + j < cols; ++j) row[col + j] = (uint8_t)(w >> (8 * j));
    }
}

// How the 16 units of a CTA are laid over a row: `across` blocks of one row side by side, 16 / across rows.
int units_across(int blocks) {
    int a = 1;
    while (a < kUnits && a < blocks) a *= 2;
    return a;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void fp8_quant_kernel(const Fp8QuantArgs a, int across, int kb_total) {
    const int unit = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const int rows_at_once = kUnits / across;
    const int kb_first = blockIdx.y * across + unit % across;
    const T* x = reinterpret_cast<const T*>(a.x);
    // every thread of a warp runs the same trip count (the shuffles need all lanes): rows and blocks past the end load
    // nothing and store nothing
    for (int row0 = blockIdx.x * rows_at_once; row0 < a.rows; row0 += gridDim.x * rows_at_once) {
        const int t = row0 + unit / across;
        for (int kb0 = 0; kb0 < kb_total; kb0 += gridDim.y * across) {
            const int kb = kb0 + kb_first, col = kb * 128 + l16 * 8;
            const bool on = t < a.rows && kb < kb_total;
            float v[8];
            load8<T, VEC>(x + (size_t)(on ? t : 0) * a.ldx, on ? col : 0, on ? a.cols : 0, v);
            float scale;
            const uint2 codes = quantise8(v, scale);
            if (!on) continue;
            if (!a.topk_row) {
                store_codes(a.q + (size_t)t * a.ldq, col, a.cols, codes);
                if (l16 == 0) a.scale[(size_t)kb * a.lds + t] = scale;
            } else {
                for (int s = 0; s < a.k; ++s) {
                    const int r = a.topk_row[(size_t)t * a.idx_stride + s];
                    if (r < 0 || r >= a.num_rows) continue;
                    store_codes(a.q + (size_t)r * a.ldq, col, a.cols, codes);
                    if (l16 == 0) a.scale[(size_t)kb * a.lds + r] = scale;
                }
            }
        }
    }
}

// ---- gated activations: v = act(g) * u, sigmoid by expf and one reciprocal --------------------------------------------
// ACT 0: silu(g) * u;  1: min(g, limit) * sigmoid(alpha * min(g, limit)) * (clamp(u, -limit, limit) + 1);
// 2: gelu_tanh(g) * u, written as g * sigmoid(2 z) (z the tanh's argument): no cancellation for negative g. NaN passes.
__device__ __forceinline__ float sigmoid(float z) { return rcp_approx(1.f + expf(-z)); }
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
template <int ACT>
__device__ __forceinline__ void glu_gradient(float g, float u, float da, float alpha, float limit, float& dg, float& du) {
    if (ACT == 1) {
        const bool in_g = g <= limit, in_u = fabsf(u) <= limit;
        const float gc = g > limit ? limit : g, uc = u > limit ? limit : (u < -limit ? -limit : u);
        const float s = sigmoid(alpha * gc);
        dg = in_g ? da * (uc + 1.f) * s * (1.f + alpha * gc * (1.f - s)) : 0.f;
        du = in_u ? da * gc * s : 0.f;
    } else if (ACT == 2) {
        const float s = sigmoid(2.f * kGeluC * (g + kGeluA * g * g * g));
        dg = da * u * s * (1.f + 2.f * kGeluC * g * (1.f + 3.f * kGeluA * g * g) * (1.f - s));
        du = da * g * s;
    } else {
        const float s = sigmoid(g);
        dg = da * u * s * (1.f + g * (1.f - s));
        du = da * g * s;
    }
}

// Row tiles of the live rows only: with expert segments the rows between an expert's last and the next multiple of 128
// hold nothing and are neither read nor written.
template <typename T, bool VEC, int ACT, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void glu_kernel(const Fp8QuantArgs a, int across, int kb_total, int tile_rows) {
    __shared__ int prefix[kMaxMats + 1];
    if (a.counts) {
        if (threadIdx.x < 32) tile_prefix_build(prefix, a.counts, a.e_tot, 1, tile_rows);
        __syncthreads();
    }
    const int total = a.counts ? prefix[a.e_tot] : (a.rows + tile_rows - 1) / tile_rows;
    const int unit = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const int rows_at_once = kUnits / across;
    const T* h = reinterpret_cast<const T*>(a.x);
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        int row0 = item * tile_rows, row_end = min(row0 + tile_rows, a.rows);
        if (a.counts) {
            const TileInfo t = tile_decode(item, prefix, a.counts, a.offsets, a.e_tot, tile_rows);
            row0 = t.row0;
            row_end = min(row0 + min(tile_rows, t.count - t.nt_idx * tile_rows), a.rows);
            if (row0 < 0) continue;
        }
        for (int r0 = row0; r0 < row_end; r0 += rows_at_once) {
            const int r = r0 + unit / across;
            for (int kb0 = blockIdx.y * across; kb0 < kb_total; kb0 += gridDim.y * across) {
                const int kb = kb0 + unit % across, col = kb * 128 + l16 * 8;
                const bool on = r < row_end && kb < kb_total;
                const T* row = h + (size_t)(on ? r : row0) * a.ldx;
                const int c = on ? col : 0, cols = on ? a.cols : 0;
                float g[8], u[8];
                load8<T, VEC>(row, c, cols, g);
                load8<T, VEC>(row + a.cols, c, cols, u);
                if (BACKWARD) {
                    float d[8];
                    load8<T, VEC>(reinterpret_cast<const T*>(a.da) + (size_t)(on ? r : row0) * a.cols, c, cols, d);
#pragma unroll
                    for (int j = 0; j < 8; ++j) glu_gradient<ACT>(g[j], u[j], d[j], a.alpha, a.limit, g[j], u[j]);
                    if (on) {
                        T* out = reinterpret_cast<T*>(a.dh) + (size_t)r * 2 * a.cols;
                        store8<T, VEC>(out, c, cols, g);
                        store8<T, VEC>(out + a.cols, c, cols, u);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] = col + j < cols ? glu_value<ACT>(g[j], u[j], a.alpha, a.limit) : 0.f;
                    float scale;
                    const uint2 codes = quantise8(g, scale);
                    if (on) {
                        store_codes(a.q + (size_t)r * a.ldq, col, a.cols, codes);
                        if (l16 == 0) a.scale[(size_t)kb * a.lds + r] = scale;
                    }
                }
            }
        }
    }
}

// One CTA per 128 x 128 block of a weight (load time): 64 values per thread, read twice (the second time from L2).
template <typename T>
__global__ __launch_bounds__(kThreads) void fp8_quant_weight_kernel(const T* __restrict__ w, int n, int k, int nb, int kb,
                                                                    uint8_t* __restrict__ q, int ldq,
                                                                    float* __restrict__ scale) {
    __shared__ uint32_t warp_max[kThreads / 32];
    const size_t block = blockIdx.x;
    const int bk = (int)(block % kb), bn = (int)(block / kb % nb);
    const size_t mat = block / kb / nb;
    const int rows = min(128, n - bn * 128), cols = min(128, k - bk * 128);
    const T* src = w + mat * n * k + (size_t)bn * 128 * k + (size_t)bk * 128;
    uint32_t m = 0u;
    for (int i = threadIdx.x; i < rows * 128; i += kThreads)
        if ((i & 127) < cols) m = max(m, __float_as_uint(to_f32<T>(src[(size_t)(i >> 7) * k + (i & 127)])) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) m = max(m, warp_max[i]);
    const BlockScale b = block_scale(m);
    if (threadIdx.x == 0) scale[block] = b.scale;
    uint8_t* dst = q + mat * n * ldq + (size_t)bn * 128 * ldq + (size_t)bk * 128;
    for (int i = threadIdx.x; i < rows * 128; i += kThreads) {
        if ((i & 127) >= cols) continue;
        const float x = to_f32<T>(src[(size_t)(i >> 7) * k + (i & 127)]);
        const float y = copysignf(quotient_for_e4m3(fabsf(x) * b.shift, b.s, b.r), x);
        dst[(size_t)(i >> 7) * ldq + (i & 127)] = b.finite ? (uint8_t)cvt_e4m3x2(y, 0.f) : (uint8_t)0x7fu;
    }
}

template <typename T>
bool rows_aligned(const void* p, size_t ld) { return ((uintptr_t)p & 15u) == 0 && ld * sizeof(T) % 16 == 0; }

template <typename T>
int quant_t(const Fp8QuantArgs& a, cudaStream_t stream) {
    const int kb = (a.cols + 127) / 128, across = units_across(kb);
    const int row_groups = (a.rows + kUnits / across - 1) / (kUnits / across);
    const int k_groups = (kb + across - 1) / across;
    // few rows: the blocks of a row go to different CTAs; many rows: one CTA walks a row
    dim3 grid(row_groups < 148 * 16 ? row_groups : 148 * 16, row_groups < 148 * 8 ? k_groups : 1);
    if (rows_aligned<T>(a.x, a.ldx)) fp8_quant_kernel<T, true><<<grid, kThreads, 0, stream>>>(a, across, kb);
    else fp8_quant_kernel<T, false><<<grid, kThreads, 0, stream>>>(a, across, kb);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}

template <typename T, int ACT, bool BACKWARD>
int glu_act(const Fp8QuantArgs& a, cudaStream_t stream) {
    const int kb = (a.cols + 127) / 128, across = units_across(kb);
    const int rows_at_once = kUnits / across;
    const int tile_rows = rows_at_once < 4 ? 4 : rows_at_once;
    const int tiles = (a.rows + tile_rows - 1) / tile_rows;
    const dim3 grid(tiles < 148 * 8 ? tiles : 148 * 8, 1);
    const bool vec = rows_aligned<T>(a.x, a.ldx) && a.cols * sizeof(T) % 16 == 0 &&
                     (!BACKWARD || (((uintptr_t)a.da | (uintptr_t)a.dh) & 15u) == 0);
    if (vec) glu_kernel<T, true, ACT, BACKWARD><<<grid, kThreads, 0, stream>>>(a, across, kb, tile_rows);
    else glu_kernel<T, false, ACT, BACKWARD><<<grid, kThreads, 0, stream>>>(a, across, kb, tile_rows);
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
    fp8_quant_weight_kernel<T><<<(unsigned)blocks, kThreads, 0, stream>>>((const T*)w, n, k, nb, kb, q, ldq, scale);
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
