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

// A value that rounds to e4m3 the way the exact quotient x / s does (s > 0, r an approximation of 1 / s, off by 2^-22 of it
// at most). y0 = x * r with one correction by its residual is x / s to within half an fp32 step and 2^-44 of it, so it
// lies on the same side of every border between two codes as x / s, or exactly on the border: borders have at most five
// significant bits and are fp32 numbers.
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float y0 = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-y0, s, x), r, y0);
}
// y can only be a border if its low 19 bits are zero (normal codes: a 1 and 19 zeros below the three mantissa bits;
// subnormal codes: odd multiples of 2^-10). Then the sign of the residual, which an fma gives exactly, says on which side
// of the border x / s lies, and y moves one fp32 step that way.
__device__ __forceinline__ float off_border(float y, float x, float s) {
    uint32_t bits = __float_as_uint(y);
    const float size = fabsf(y);
    if ((bits & 0xfffffu) == (size >= 0.015625f ? 0x80000u : 0u) && size > 0.f) {
        const float e = __fmaf_rn(-y, s, x);
        if (e != 0.f) bits += (e > 0.f) == (y > 0.f) ? 1u : ~0u;
    }
    return __uint_as_float(bits);
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
// The code of one value of an unusual block: NaN where the scale is not finite, 0 where it is 0; else divisor and value are
// first brought to where no product is subnormal.
__device__ __noinline__ uint32_t unusual_code(float x, float scale) {
    if (!(scale <= 3.4028235e38f)) return 0x7fu;
    if (scale == 0.f) return 0u;
    const float f = scale < 1.f ? 18446744073709551616.f : 5.4210109e-20f;  // 2^64, 2^-64
    const float s = __fmul_rn(scale, f), v = __fmul_rn(x, f);
    return cvt_e4m3x2(off_border(quotient(v, s, __frcp_rn(s)), v, s), 0.f) & 0xffu;
}

__device__ __forceinline__ uint2 codes8(const float* v, const BlockScale& b) {
    uint32_t c[4];
    if (b.usual) {
        float y[8];
        uint32_t low = ~0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[j] = quotient(v[j], b.scale, b.r);
            low = min(low, __float_as_uint(y[j]) << 13);
        }
        if (low == 0u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = off_border(y[j], v[j], b.scale);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = cvt_e4m3x2(y[2 * j], y[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = unusual_code(v[2 * j], b.scale) | (unusual_code(v[2 * j + 1], b.scale) << 8);
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
// Eight values of a block, this lane's share; all 16 lanes of the block take part. Returns eight codes.
__device__ __forceinline__ uint2 quantise8(const float* v, float& scale) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
#pragma unroll
    for (int d = 8; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    const BlockScale b = block_scale(m);
    scale = b.scale;
    return codes8(v, b);
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

// The blocks of a matrix row by row, handed out to the CTA's 16 half-warps in turn: half-warp u takes blocks u, u + 16, ..
// of the CTA's share. Steps of 16 blocks are a fixed number of rows and blocks, so no division follows the first.
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

constexpr int kUnroll = 2;   // blocks per half-warp with their loads in flight together
constexpr int kShare = 128;  // blocks per CTA of the row quantiser

template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void fp8_quant_kernel(const Fp8QuantArgs a, int kb_total, int share) {
    const int unit = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const T* x = reinterpret_cast<const T*>(a.x);
    const size_t first = (size_t)blockIdx.x * share + unit;
    Walk w{(int)(first / kb_total), (int)(first % kb_total)};
    const int d_row = kUnits / kb_total, d_kb = kUnits % kb_total;
    // every half-warp takes the same number of steps (the shuffles need all lanes of a warp): a block past the last row
    // loads and stores nothing
    for (int i = 0; i < share; i += kUnits * kUnroll) {
        float v[kUnroll][8];
        Walk at[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            at[u] = w;
            if (i + u * kUnits >= share) at[u].row = a.rows;
            const bool on = at[u].row < a.rows;
            load8<T, VEC>(x + (size_t)(on ? at[u].row : 0) * a.ldx, on ? at[u].kb * 128 + l16 * 8 : 0, on ? a.cols : 0, v[u]);
            w.step(d_row, d_kb, kb_total);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float scale;
            const uint2 codes = quantise8(v[u], scale);
            const int t = at[u].row, kb = at[u].kb, col = kb * 128 + l16 * 8;
            if (t >= a.rows) continue;
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
__global__ __launch_bounds__(kThreads) void glu_kernel(const Fp8QuantArgs a, int kb_total, int tile_rows) {
    __shared__ int prefix[kMaxMats + 1];
    if (a.counts) {
        if (threadIdx.x < 32) tile_prefix_build(prefix, a.counts, a.e_tot, 1, tile_rows);
        __syncthreads();
    }
    const int total = a.counts ? prefix[a.e_tot] : (a.rows + tile_rows - 1) / tile_rows;
    const int unit = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    const int d_row = kUnits / kb_total, d_kb = kUnits % kb_total;
    const Walk start{unit / kb_total, unit % kb_total};
    const T* h = reinterpret_cast<const T*>(a.x);
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        int row0 = item * tile_rows, row_end = min(row0 + tile_rows, a.rows);
        if (a.counts) {
            const TileInfo t = tile_decode(item, prefix, a.counts, a.offsets, a.e_tot, tile_rows);
            row0 = t.row0;
            row_end = min(row0 + min(tile_rows, t.count - t.nt_idx * tile_rows), a.rows);
            if (row0 < 0) continue;
        }
        const int n_units = (row_end - row0) * kb_total;
        Walk w = start;
        for (int i = 0; i < n_units; i += kUnits) {
            const int r = row0 + w.row, kb = w.kb, col = kb * 128 + l16 * 8;
            const bool on = r < row_end;
            w.step(d_row, d_kb, kb_total);
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
                for (int j = 0; j < 8; ++j) g[j] = glu_value<ACT>(g[j], u[j], a.alpha, a.limit);
                if (c + 8 > cols) {  // columns past the last take no part in the block's maximum
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] = c + j < cols ? g[j] : 0.f;
                }
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
        load8<T, VEC>(src + (size_t)(r < rows ? r : 0) * k, r < rows ? col : 0, r < rows ? k : 0, v[p]);
    }
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[p][j]));
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
        if (r < rows) store_codes(dst + (size_t)r * ldq, col, k, codes8(v[p], b));
    }
}

template <typename T>
bool rows_aligned(const void* p, size_t ld) { return ((uintptr_t)p & 15u) == 0 && ld * sizeof(T) % 16 == 0; }

template <typename T>
int quant_t(const Fp8QuantArgs& a, cudaStream_t stream) {
    const int kb = (a.cols + 127) / 128;
    const size_t blocks = (size_t)a.rows * kb;
    // small calls: one block per half-warp, so that every SM has some
    const int share = blocks >= (size_t)148 * 4 * kShare ? kShare : kUnits;
    const size_t grid = (blocks + share - 1) / share;
    if (grid > 0x7fffffffu) return XMOE_ERR_LIMIT;
    if (rows_aligned<T>(a.x, a.ldx)) fp8_quant_kernel<T, true><<<(unsigned)grid, kThreads, 0, stream>>>(a, kb, share);
    else fp8_quant_kernel<T, false><<<(unsigned)grid, kThreads, 0, stream>>>(a, kb, share);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}

template <typename T, int ACT, bool BACKWARD>
int glu_act(const Fp8QuantArgs& a, cudaStream_t stream) {
    const int kb = (a.cols + 127) / 128;
    const int tile_rows = kb >= 4 ? 4 : 16;
    const int tiles = (a.rows + tile_rows - 1) / tile_rows;
    const dim3 grid(tiles < 148 * 8 ? tiles : 148 * 8);
    const bool vec = rows_aligned<T>(a.x, a.ldx) && a.cols * sizeof(T) % 16 == 0 &&
                     (!BACKWARD || (((uintptr_t)a.da | (uintptr_t)a.dh) & 15u) == 0);
    if (vec) glu_kernel<T, true, ACT, BACKWARD><<<grid, kThreads, 0, stream>>>(a, kb, tile_rows);
    else glu_kernel<T, false, ACT, BACKWARD><<<grid, kThreads, 0, stream>>>(a, kb, tile_rows);
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
