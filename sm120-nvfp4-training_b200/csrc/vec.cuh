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

// V elements as they lie in memory, in 32-bit registers (two 16-bit elements to one; a single one in the low half).  Held as
// words, not as elements: a copy element by element and conversions one at a time were 50 instructions per element of the
// layer norm where 15 do.
template <typename T, int V> struct Pack {
    static constexpr int BYTES = sizeof(T) * V, WORDS = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t w[WORDS];
};
// At most 16 bytes per load and store; 32 bytes are two of them.  CONST: through the read-only path.
template <typename T, int V, bool CONST = false> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    constexpr int B = Pack<T, V>::BYTES;
    Pack<T, V> v;
    auto get = [](const auto* q) { if constexpr (CONST) return __ldg(q); else return *q; };
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) {
            const uint4 q = get(reinterpret_cast<const uint4*>(p) + i);
            v.w[4 * i] = q.x; v.w[4 * i + 1] = q.y; v.w[4 * i + 2] = q.z; v.w[4 * i + 3] = q.w;
        }
    } else if constexpr (B == 8) {
        const uint2 q = get(reinterpret_cast<const uint2*>(p));
        v.w[0] = q.x; v.w[1] = q.y;
    } else if constexpr (B == 4) {
        v.w[0] = get(reinterpret_cast<const uint32_t*>(p));
    } else {
        v.w[0] = get(reinterpret_cast<const uint16_t*>(p));
    }
    return v;
}
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_const(const T* p) { return load_pack<T, V, true>(p); }
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    constexpr int B = Pack<T, V>::BYTES;
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(v.w[4 * i], v.w[4 * i + 1], v.w[4 * i + 2], v.w[4 * i + 3]);
    } else if constexpr (B == 8) *reinterpret_cast<uint2*>(p) = make_uint2(v.w[0], v.w[1]);
    else if constexpr (B == 4) *reinterpret_cast<uint32_t*>(p) = v.w[0];
    else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(v.w[0]);
}
template <typename T, int V> __device__ __forceinline__ float element(const Pack<T, V>& v, int j) {      // j known at compile time
    if constexpr (sizeof(T) == 4) return __uint_as_float(v.w[j]);
    else if constexpr (Code<T>::value == NVFP4_BF16) return __uint_as_float((j & 1) ? v.w[j / 2] & 0xffff0000u : v.w[j / 2] << 16);
    else {
        const __half2 h = *reinterpret_cast<const __half2*>(&v.w[j / 2]);
        return (j & 1) ? __high2float(h) : __low2float(h);
    }
}
template <typename T, int V> __device__ __forceinline__ void set_element(Pack<T, V>& v, int j, T value) {
    if constexpr (sizeof(T) == 4) v.w[j] = __float_as_uint(to_float(value));
    else {
        const uint32_t bits = *reinterpret_cast<const uint16_t*>(&value);
        v.w[j / 2] = (j & 1) ? (v.w[j / 2] & 0xffffu) | bits << 16 : (v.w[j / 2] & 0xffff0000u) | bits;
    }
}
template <typename T, int V> __device__ __forceinline__ void unpack(const Pack<T, V>& v, float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = element(v, j);
}
template <typename T, int V> __device__ __forceinline__ Pack<T, V> pack(const float (&f)[V]) {
    Pack<T, V> v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < V; ++j) v.w[j] = __float_as_uint(f[j]);
    } else if constexpr (V == 1) {
        const T one = from_float<T>(f[0]);
        v.w[0] = *reinterpret_cast<const uint16_t*>(&one);
    } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            if constexpr (Code<T>::value == NVFP4_BF16) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                v.w[j] = *reinterpret_cast<const uint32_t*>(&two);
            } else {
                const __half2 two = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
                v.w[j] = *reinterpret_cast<const uint32_t*>(&two);
            }
        }
    }
    return v;
}
template <typename T, int V> __device__ __forceinline__ float abs_max(const Pack<T, V>& v) {
    float best = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) best = fmaxf(best, fabsf(element(v, j)));
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
