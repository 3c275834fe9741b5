// Vectors of V elements of one of the three storage types, held as FP32 in registers; fixed-order CTA sums.
#pragma once
#include "common.cuh"

namespace nvfp4 {

template <typename T> struct Code;
template <> struct Code<float> { static constexpr int value = NVFP4_F32; };
template <> struct Code<__nv_bfloat16> { static constexpr int value = NVFP4_BF16; };
template <> struct Code<__half> { static constexpr int value = NVFP4_F16; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// V elements as one register block; loads and stores are as wide as the block (at most 16 bytes each, a block of 32 bytes
// is two of them).
template <typename T, int V> struct __align__(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack { T e[V]; };

template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }
// The same through the read-only path, for tensors that the kernel does not write: such loads may be moved ahead of stores,
// which a plain load behind a store to an unknown address may not.
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_const(const T* p) {
    Pack<T, V> v;
    if constexpr (sizeof(v) == 32) {
        reinterpret_cast<uint4*>(&v)[0] = __ldg(reinterpret_cast<const uint4*>(p));
        reinterpret_cast<uint4*>(&v)[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    } else if constexpr (sizeof(v) == 16) *reinterpret_cast<uint4*>(&v) = __ldg(reinterpret_cast<const uint4*>(p));
    else if constexpr (sizeof(v) == 8) *reinterpret_cast<uint2*>(&v) = __ldg(reinterpret_cast<const uint2*>(p));
    else if constexpr (sizeof(v) == 4) *reinterpret_cast<uint32_t*>(&v) = __ldg(reinterpret_cast<const uint32_t*>(p));
    else *reinterpret_cast<uint16_t*>(&v) = __ldg(reinterpret_cast<const uint16_t*>(p));
    return v;
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) { *reinterpret_cast<Pack<T, V>*>(p) = v; }
template <typename T, int V> __device__ __forceinline__ void unpack(const Pack<T, V>& v, float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = to_float(v.e[j]);
}
template <typename T, int V> __device__ __forceinline__ Pack<T, V> pack(const float (&f)[V]) {
    Pack<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.e[j] = from_float<T>(f[j]);
    return v;
}
template <typename T, int V> __device__ __forceinline__ float abs_max(const Pack<T, V>& v) {
    float best = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) best = fmaxf(best, fabsf(to_float(v.e[j])));
    return best;
}
// V parameters (weight, bias) of a type known at run time; the branch is the same for the whole grid
template <int V> __device__ __forceinline__ void load_param(const void* p, int dtype, int64_t i, float (&f)[V]) {
    if (dtype == NVFP4_F32) unpack(load_const<float, V>(static_cast<const float*>(p) + i), f);
    else if (dtype == NVFP4_BF16) unpack(load_const<__nv_bfloat16, V>(static_cast<const __nv_bfloat16*>(p) + i), f);
    else unpack(load_const<__half, V>(static_cast<const __half*>(p) + i), f);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
    if (dtype == NVFP4_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == NVFP4_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

inline int dtype_size(int dtype) { return dtype == NVFP4_F32 ? 4 : 2; }
inline bool is_float_dtype(int dtype) { return dtype == NVFP4_F32 || dtype == NVFP4_BF16 || dtype == NVFP4_F16; }
inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace nvfp4
