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
// registers, so HBM traffic is the floor (one read of every input, one write of every output).
#include "elem.cuh"
#include "kernels.h"

namespace xmoe {

namespace {

constexpr int kThreads = 256;
constexpr int kSlotBatch = 8;  // rows in flight per thread

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void permute_kernel(const T* __restrict__ x, const int32_t* __restrict__ topk_row,
                                                           T* __restrict__ rows, int n, int hv, int k, int idx_stride,
                                                           int num_rows) {
    const size_t h = (size_t)hv * VEC, total = (size_t)n * hv;
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
        const size_t t = i / hv, c = i % hv;
        const Pack<T, VEC> v = load_pack_once<T, VEC>(x + t * h + c * VEC);
        const int32_t* idx = topk_row + t * idx_stride;
        for (int s = 0; s < k; ++s) {
            const int r = idx[s];
            if (r >= 0 && r < num_rows) store_pack<T, VEC>(rows + (size_t)r * h + c * VEC, v);
        }
    }
}

// WT 0: no weights, 1: bf16, 2: fp32
template <int WT>
__device__ __forceinline__ float slot_weight(const void* w, size_t i) {
    if constexpr (WT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
    else if constexpr (WT == 2) return static_cast<const float*>(w)[i];
    else return 1.f;
}

template <typename T, int VEC, int WT>
__global__ __launch_bounds__(kThreads) void unpermute_kernel(const T* __restrict__ rows, const int32_t* __restrict__ topk_row,
                                                             const void* __restrict__ w, T* __restrict__ y, int n, int hv,
                                                             int k, int idx_stride, int w_stride, int num_rows) {
    const size_t h = (size_t)hv * VEC, total = (size_t)n * hv;
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
        const size_t t = i / hv, c = i % hv;
        const int32_t* idx = topk_row + t * idx_stride;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        for (int s0 = 0; s0 < k; s0 += kSlotBatch) {
            Pack<T, VEC> v[kSlotBatch];
            float ws[kSlotBatch];
            bool on[kSlotBatch];
#pragma unroll
            for (int s = 0; s < kSlotBatch; ++s) {
                const int r = s0 + s < k ? idx[s0 + s] : -1;
                on[s] = r >= 0 && r < num_rows;
                if (on[s]) {
                    v[s] = load_pack_once<T, VEC>(rows + (size_t)r * h + c * VEC);
                    ws[s] = slot_weight<WT>(w, t * w_stride + s0 + s);
                }
            }
#pragma unroll
            for (int s = 0; s < kSlotBatch; ++s)
                if (on[s]) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        acc[j] = WT ? fmaf(ws[s], to_f32<T>(v[s].v[j]), acc[j]) : acc[j] + to_f32<T>(v[s].v[j]);
                }
        }
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(acc[j]);
        store_pack<T, VEC>(y + t * h + c * VEC, o);
    }
}

// One CTA per token: dy[t] is read once per batch of slots, every thread keeps one partial dot product per slot, and
// the partials are added over the warp and then over the warps in a fixed order.
template <typename T, int VEC, int WT>
__global__ __launch_bounds__(kThreads) void unpermute_backward_kernel(const T* __restrict__ dy, const T* __restrict__ rows,
                                                                      const int32_t* __restrict__ topk_row,
                                                                      const void* __restrict__ w, T* __restrict__ drows,
                                                                      float* __restrict__ dw, int n, int hv, int k,
                                                                      int idx_stride, int w_stride, int num_rows) {
    __shared__ float part[kThreads / 32][kSlotBatch];
    const size_t h = (size_t)hv * VEC;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (size_t t = blockIdx.x; t < (size_t)n; t += gridDim.x) {
        for (int s0 = 0; s0 < k; s0 += kSlotBatch) {
            int r[kSlotBatch];
            float ws[kSlotBatch], dot[kSlotBatch];
#pragma unroll
            for (int s = 0; s < kSlotBatch; ++s) {
                r[s] = s0 + s < k ? topk_row[t * idx_stride + s0 + s] : -1;
                if (r[s] >= num_rows) r[s] = -1;
                ws[s] = r[s] >= 0 ? slot_weight<WT>(w, t * w_stride + s0 + s) : 0.f;
                dot[s] = 0.f;
            }
            for (int c = threadIdx.x; c < hv; c += kThreads) {
                const Pack<T, VEC> g = load_pack<T, VEC>(dy + t * h + (size_t)c * VEC);
                float gf[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) gf[j] = to_f32<T>(g.v[j]);
                Pack<T, VEC> v[kSlotBatch];
#pragma unroll
                for (int s = 0; s < kSlotBatch; ++s)
                    if (r[s] >= 0) v[s] = load_pack_once<T, VEC>(rows + (size_t)r[s] * h + (size_t)c * VEC);
#pragma unroll
                for (int s = 0; s < kSlotBatch; ++s)
                    if (r[s] >= 0) {
                        Pack<T, VEC> o;
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            dot[s] = fmaf(gf[j], to_f32<T>(v[s].v[j]), dot[s]);
                            o.v[j] = from_f32<T>(ws[s] * gf[j]);
                        }
                        store_pack<T, VEC>(drows + (size_t)r[s] * h + (size_t)c * VEC, o);
                    }
            }
#pragma unroll
            for (int s = 0; s < kSlotBatch; ++s) {
#pragma unroll
                for (int d = 16; d; d >>= 1) dot[s] += __shfl_xor_sync(0xffffffffu, dot[s], d);
                if (lane == 0) part[warp][s] = dot[s];
            }
            __syncthreads();
            if (threadIdx.x < kSlotBatch && s0 + (int)threadIdx.x < k) {
                float sum = 0.f;
#pragma unroll
                for (int q = 0; q < kThreads / 32; ++q) sum += part[q][threadIdx.x];
                dw[t * k + s0 + threadIdx.x] = sum;  // a slot without a row: its partials are all zero
            }
            __syncthreads();
        }
    }
}

int grid_for(size_t threads) {
    const size_t blocks = (threads + kThreads - 1) / kThreads;
    return (int)(blocks < 148 * 32 ? blocks : 148 * 32);
}

template <typename T>
bool vectors_ok(int h, const void* a, const void* b, const void* c) {
    return (size_t)h * sizeof(T) % 16 == 0 &&
           (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15u) == 0;
}

template <typename T>
int permute_t(const PermuteArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (vectors_ok<T>(a.H, a.x, a.rows, nullptr))
        permute_kernel<T, V><<<grid_for((size_t)a.N * (a.H / V)), kThreads, 0, stream>>>(
            (const T*)a.x, a.topk_row, (T*)a.rows, a.N, a.H / V, a.k, a.idx_stride, a.num_rows);
    else
        permute_kernel<T, 1><<<grid_for((size_t)a.N * a.H), kThreads, 0, stream>>>((const T*)a.x, a.topk_row, (T*)a.rows, a.N,
                                                                                   a.H, a.k, a.idx_stride, a.num_rows);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}

template <typename T, int WT>
int unpermute_t(const PermuteArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (vectors_ok<T>(a.H, a.x, a.rows, nullptr))
        unpermute_kernel<T, V, WT><<<grid_for((size_t)a.N * (a.H / V)), kThreads, 0, stream>>>(
            (const T*)a.rows, a.topk_row, a.w, (T*)a.x, a.N, a.H / V, a.k, a.idx_stride, a.w_stride, a.num_rows);
    else
        unpermute_kernel<T, 1, WT><<<grid_for((size_t)a.N * a.H), kThreads, 0, stream>>>(
            (const T*)a.rows, a.topk_row, a.w, (T*)a.x, a.N, a.H, a.k, a.idx_stride, a.w_stride, a.num_rows);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
}

template <typename T, int WT>
int unpermute_backward_t(const PermuteArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const int grid = a.N < 148 * 64 ? a.N : 148 * 64;
    if (vectors_ok<T>(a.H, a.x, a.rows, a.drows))
        unpermute_backward_kernel<T, V, WT><<<grid, kThreads, 0, stream>>>((const T*)a.x, (const T*)a.rows, a.topk_row, a.w,
                                                                           (T*)a.drows, a.dw, a.N, a.H / V, a.k, a.idx_stride,
                                                                           a.w_stride, a.num_rows);
    else
        unpermute_backward_kernel<T, 1, WT><<<grid, kThreads, 0, stream>>>((const T*)a.x, (const T*)a.rows, a.topk_row, a.w,
                                                                           (T*)a.drows, a.dw, a.N, a.H, a.k, a.idx_stride,
                                                                           a.w_stride, a.num_rows);
    return cudaGetLastError() == cudaSuccess ? XMOE_OK : XMOE_ERR_CUDA;
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
