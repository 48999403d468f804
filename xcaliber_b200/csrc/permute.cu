// Tokens to rows sorted by expert and back, with routing weights, and the gradients of both. The plan is
// topk_row [N, k] (xmoe_route_pack): slot s of token t lives in row topk_row[t, s]; a negative or out-of-range entry is
// a slot without a row.
//   permute             rows[topk_row[t, s]] = x[t]
//   unpermute           y[t] = sum_s w[t, s] * rows[topk_row[t, s]]     (w absent: 1; also the gradient of permute)
//   unpermute_backward  drows[topk_row[t, s]] = w[t, s] * dy[t],  dw[t, s] = <dy[t], rows[topk_row[t, s]]>
// Sums run in fp32, slot 0 first, with one rounding at the store: the same bits on every run (no atomics). Rows that no
// slot names are left as they were.
//
// All three move bytes and do next to no arithmetic: each token's data is read once and all its slots are served from
// registers, so HBM traffic is the floor (one read of every input, one write of every output). Measured, 8191 tokens, 8
// slots, 2048 bf16: unpermute 47.5 us = 6.4 TB/s, its gradient 95 us = 6.0 TB/s; 4095 tokens, 4 slots, 2880 fp16: permute
// 21 us = 5.4 TB/s and its gradient 21 us = 5.6 TB/s. Rows of 16-bit values that are not 16-byte aligned take narrower
// accesses (4096 tokens, 8 slots; permute, unpermute, its gradient): width 2048 26, 25, 48 us; 2050, 4 bytes each, 41, 41,
// 72; 2049, 2 bytes each, 50, 92, 214.
#include "elem.cuh"
#include "kernels.h"

namespace xmoe {

namespace {

constexpr int kThreads = 256;

// A CTA covers 256 >> shift tokens with 1 << shift threads side by side on each; blockIdx.y walks a wider row. So every
// thread moves one vector of one token without a division, and few tokens still spread over many CTAs.
// Where an access is narrow (rows that are not 16-byte aligned) a thread takes REP of them, 1 << shift apart.
struct Place {
    size_t t;
    int c;
};
template <int REP>
__device__ __forceinline__ Place place(int shift) {
    return {(size_t)blockIdx.x * (kThreads >> shift) + (threadIdx.x >> shift),
            (int)(((size_t)blockIdx.y * REP << shift) + (threadIdx.x & ((1 << shift) - 1)))};
}
template <typename T, int VEC> constexpr int kPermuteRep = VEC * sizeof(T) == 16 ? 1 : 4;
template <typename T, int VEC> constexpr int kUnpermuteRep = VEC * sizeof(T) == 16 ? 1 : 2;

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void permute_kernel(const T* __restrict__ x, const int32_t* __restrict__ topk_row,
                                                           T* __restrict__ rows, int n, int hv, int k, int idx_stride,
                                                           int num_rows, int shift) {
    constexpr int R = kPermuteRep<T, VEC>;
    const Place p = place<R>(shift);
    if (p.t >= (size_t)n || p.c >= hv) return;
    const size_t h = (size_t)hv * VEC;
    Pack<T, VEC> v[R];
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (u == 0 || p.c + (u << shift) < hv) v[u] = load_pack_once<T, VEC>(x + p.t * h + (size_t)(p.c + (u << shift)) * VEC);
    const int32_t* idx = topk_row + p.t * idx_stride;
#pragma unroll 8
    for (int s = 0; s < k; ++s) {
        const int r = idx[s];
        if (r < 0 || r >= num_rows) continue;
#pragma unroll
        for (int u = 0; u < R; ++u)
            if (u == 0 || p.c + (u << shift) < hv) store_pack<T, VEC>(rows + (size_t)r * h + (size_t)(p.c + (u << shift)) * VEC, v[u]);
    }
}

// WT 0: no weights, 1: bf16, 2: fp32
template <int WT>
__device__ __forceinline__ float slot_weight(const void* w, size_t i) {
    if constexpr (WT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
    else if constexpr (WT == 2) return static_cast<const float*>(w)[i];
    else return 1.f;
}

// SLOTS rows are in flight per thread. A slot without a row reads row 0 instead (so that the loads do not wait for a
// branch each) and adds nothing.
template <typename T, int VEC, int WT, int SLOTS>
__global__ __launch_bounds__(kThreads) void unpermute_kernel(const T* __restrict__ rows, const int32_t* __restrict__ topk_row,
                                                             const void* __restrict__ w, T* __restrict__ y, int n, int hv,
                                                             int k, int idx_stride, int w_stride, int num_rows, int shift) {
    constexpr int R = kUnpermuteRep<T, VEC>;
    const Place p = place<R>(shift);
    if (p.t >= (size_t)n || p.c >= hv) return;
    const size_t h = (size_t)hv * VEC;
    const int32_t* idx = topk_row + p.t * idx_stride;
    float acc[R][VEC];
#pragma unroll
    for (int u = 0; u < R; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
    for (int s0 = 0; s0 < k; s0 += SLOTS) {
        int r[SLOTS];
        Pack<T, VEC> v[R][SLOTS];
        float ws[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            r[s] = s0 + s < k ? idx[s0 + s] : -1;
            if (r[s] >= num_rows) r[s] = -1;
            ws[s] = slot_weight<WT>(w, p.t * w_stride + min(s0 + s, k - 1));
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int c = u == 0 || p.c + (u << shift) < hv ? p.c + (u << shift) : p.c;  // past the row: read, not stored
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) v[u][s] = load_pack_once<T, VEC>(rows + (size_t)max(r[s], 0) * h + (size_t)c * VEC);
        }
#pragma unroll
        for (int u = 0; u < R; ++u)
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float x = to_f32<T>(v[u][s].v[j]);
                    acc[u][j] = r[s] < 0 ? acc[u][j] : (WT ? fmaf(ws[s], x, acc[u][j]) : acc[u][j] + x);
                }
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(acc[u][j]);
        if (u == 0 || p.c + (u << shift) < hv) store_pack<T, VEC>(y + p.t * h + (size_t)(p.c + (u << shift)) * VEC, o);
    }
}

// One CTA per token: dy[t] is read once per batch of slots, every thread keeps one partial dot product per slot, and
// the partials are added over the warp and then over the warps in a fixed order.
template <typename T, int VEC, int WT, int SLOTS>
__global__ __launch_bounds__(kThreads, 3) void unpermute_backward_kernel(const T* __restrict__ dy, const T* __restrict__ rows,
                                                                      const int32_t* __restrict__ topk_row,
                                                                      const void* __restrict__ w, T* __restrict__ drows,
                                                                      float* __restrict__ dw, int n, int hv, int k,
                                                                      int idx_stride, int w_stride, int num_rows) {
    __shared__ float part[kThreads / 32][SLOTS];
    const size_t h = (size_t)hv * VEC;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (size_t t = blockIdx.x; t < (size_t)n; t += gridDim.x) {
        for (int s0 = 0; s0 < k; s0 += SLOTS) {
            int r[SLOTS];
            float ws[SLOTS], dot[SLOTS];
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                r[s] = s0 + s < k ? topk_row[t * idx_stride + s0 + s] : -1;
                if (r[s] >= num_rows) r[s] = -1;
                ws[s] = slot_weight<WT>(w, t * w_stride + min(s0 + s, k - 1));
                dot[s] = 0.f;
            }
            for (int c = threadIdx.x; c < hv; c += kThreads) {
                const Pack<T, VEC> g = load_pack<T, VEC>(dy + t * h + (size_t)c * VEC);
                Pack<T, VEC> v[SLOTS];
#pragma unroll
                for (int s = 0; s < SLOTS; ++s) v[s] = load_pack_once<T, VEC>(rows + (size_t)max(r[s], 0) * h + (size_t)c * VEC);
                float gf[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) gf[j] = to_f32<T>(g.v[j]);
#pragma unroll
                for (int s = 0; s < SLOTS; ++s) {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        dot[s] = fmaf(gf[j], to_f32<T>(v[s].v[j]), dot[s]);
                        o.v[j] = from_f32<T>(ws[s] * gf[j]);
                    }
                    if (r[s] >= 0) store_pack<T, VEC>(drows + (size_t)r[s] * h + (size_t)c * VEC, o);
                }
            }
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
#pragma unroll
                for (int d = 16; d; d >>= 1) dot[s] += __shfl_xor_sync(0xffffffffu, dot[s], d);
                if (lane == 0) part[warp][s] = r[s] < 0 ? 0.f : dot[s];
            }
            __syncthreads();
            if (threadIdx.x < SLOTS && s0 + (int)threadIdx.x < k) {
                float sum = 0.f;
#pragma unroll
                for (int q = 0; q < kThreads / 32; ++q) sum += part[q][threadIdx.x];
                dw[t * k + s0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
}

// Threads side by side on a row: the power of two that covers it, 32 to 256.
int row_shift(int hv) {
    int shift = 5;
    while (shift < 8 && (1 << shift) < hv) ++shift;
    return shift;
}
dim3 grid_for(int n, int hv, int shift, int rep) {
    const int tokens = kThreads >> shift;
    const size_t across = (size_t)rep << shift;
    return dim3((unsigned)((n + (size_t)tokens - 1) / tokens), (unsigned)((hv + across - 1) / across));
}
constexpr int kMaxGridY = 65535;

// bytes = 16 or 4: whether every row of the buffers starts at a multiple of it
template <typename T>
bool vectors_ok(int h, const void* a, const void* b, const void* c, unsigned bytes = 16) {
    return (size_t)h * sizeof(T) % bytes == 0 &&
           (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & (bytes - 1)) == 0;
}

template <typename T, int V>
int permute_v(const PermuteArgs& a, cudaStream_t stream) {
    const int hv = a.H / V, shift = row_shift(hv);
    const dim3 grid = grid_for(a.N, hv, shift, kPermuteRep<T, V>);
    if (grid.y > kMaxGridY) return XMOE_ERR_LIMIT;
    permute_kernel<T, V><<<grid, kThreads, 0, stream>>>((const T*)a.x, a.topk_row, (T*)a.rows, a.N, hv, a.k, a.idx_stride,
                                                        a.num_rows, shift);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}
template <typename T>
int permute_t(const PermuteArgs& a, cudaStream_t stream) {
    if (vectors_ok<T>(a.H, a.x, a.rows, nullptr)) return permute_v<T, 16 / sizeof(T)>(a, stream);
    if constexpr (sizeof(T) == 2)
        if (vectors_ok<T>(a.H, a.x, a.rows, nullptr, 4)) return permute_v<T, 2>(a, stream);
    return permute_v<T, 1>(a, stream);
}

template <typename T, int V, int WT, int SLOTS>
int unpermute_s(const PermuteArgs& a, cudaStream_t stream) {
    const int hv = a.H / V, shift = row_shift(hv);
    const dim3 grid = grid_for(a.N, hv, shift, kUnpermuteRep<T, V>);
    if (grid.y > kMaxGridY) return XMOE_ERR_LIMIT;
    unpermute_kernel<T, V, WT, SLOTS><<<grid, kThreads, 0, stream>>>((const T*)a.rows, a.topk_row, a.w, (T*)a.x, a.N, hv, a.k,
                                                                     a.idx_stride, a.w_stride, a.num_rows, shift);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}
template <typename T, int V, int WT, int SLOTS>
int unpermute_backward_s(const PermuteArgs& a, cudaStream_t stream) {
    const int grid = a.N < 148 * 64 ? a.N : 148 * 64;
    unpermute_backward_kernel<T, V, WT, SLOTS><<<grid, kThreads, 0, stream>>>((const T*)a.x, (const T*)a.rows, a.topk_row, a.w,
                                                                              (T*)a.drows, a.dw, a.N, a.H / V, a.k,
                                                                              a.idx_stride, a.w_stride, a.num_rows);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}
// rows in flight per thread: the smallest of 2, 4, 8 that holds a token's slots
#define XMOE_BY_SLOTS(fn, T, V, WT) \
    (a.k <= 2 ? fn<T, V, WT, 2>(a, stream) : a.k <= 4 ? fn<T, V, WT, 4>(a, stream) : fn<T, V, WT, 8>(a, stream))
template <typename T, int WT>
int unpermute_t(const PermuteArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (vectors_ok<T>(a.H, a.x, a.rows, nullptr)) return XMOE_BY_SLOTS(unpermute_s, T, V, WT);
    if constexpr (sizeof(T) == 2)
        if (vectors_ok<T>(a.H, a.x, a.rows, nullptr, 4)) return XMOE_BY_SLOTS(unpermute_s, T, 2, WT);
    return XMOE_BY_SLOTS(unpermute_s, T, 1, WT);
}
template <typename T, int WT>
int unpermute_backward_t(const PermuteArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (vectors_ok<T>(a.H, a.x, a.rows, a.drows)) return XMOE_BY_SLOTS(unpermute_backward_s, T, V, WT);
    if constexpr (sizeof(T) == 2)
        if (vectors_ok<T>(a.H, a.x, a.rows, a.drows, 4)) return XMOE_BY_SLOTS(unpermute_backward_s, T, 2, WT);
    return XMOE_BY_SLOTS(unpermute_backward_s, T, 1, WT);
}

#define XMOE_BY_WEIGHT(fn, T)                     \
    (a.w == nullptr          ? fn<T, 0>(a, stream) \
     : a.w_dtype == XMOE_BF16 ? fn<T, 1>(a, stream) \
                              : fn<T, 2>(a, stream))
#define XMOE_BY_TYPE(fn)                                            \
    switch (a.dtype) {                                              \
        case XMOE_BF16: return XMOE_BY_WEIGHT(fn, __nv_bfloat16);   \
        case XMOE_FP16: return XMOE_BY_WEIGHT(fn, __half);          \
        case XMOE_FP32: return XMOE_BY_WEIGHT(fn, float);           \
        default: return XMOE_ERR_SHAPE;                             \
    }

}  // namespace

int launch_permute(const PermuteArgs& a, cudaStream_t stream) {
    switch (a.dtype) {
        case XMOE_BF16: return permute_t<__nv_bfloat16>(a, stream);
        case XMOE_FP16: return permute_t<__half>(a, stream);
        case XMOE_FP32: return permute_t<float>(a, stream);
        default: return XMOE_ERR_SHAPE;
    }
}
int launch_unpermute(const PermuteArgs& a, cudaStream_t stream) { XMOE_BY_TYPE(unpermute_t) }
int launch_unpermute_backward(const PermuteArgs& a, cudaStream_t stream) { XMOE_BY_TYPE(unpermute_backward_t) }

}  // namespace xmoe
