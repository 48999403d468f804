// Element types of the memory-bound operators (bf16, fp16, fp32): widening loads, one rounding at the store, and
// 16-byte vectors of them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace xmoe {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// VEC elements that move as one access: 16 bytes, or 4 bytes or a single element where rows are not 16-byte aligned.
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    static_assert(VEC == 1 || VEC * sizeof(T) == 16 || (VEC == 2 && sizeof(T) == 2), "access width");
    Pack<T, VEC> r;
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(&r) = *reinterpret_cast<const uint32_t*>(p);
    else r.v[0] = *p;
    return r;
}
// the same for data that is read once: it need not displace what L1 holds
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack_once(const T* p) {
    Pack<T, VEC> r;
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
    else return load_pack<T, VEC>(p);
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& r) {
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
    else if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(&r);
    else *p = r.v[0];
}

}  // namespace xmoe
