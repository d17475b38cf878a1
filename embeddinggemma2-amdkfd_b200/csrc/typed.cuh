// Typed rows: loads and stores of fp32, fp16 and bf16 elements as fp32, one at a
// time or in 16-byte vectors, for the operators that take more than one type.
// Each store rounds once, to nearest even.
#pragma once
#include "common.cuh"

namespace eg2 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements, held in their own type: V * sizeof(T) bytes, moved in
// 16-byte accesses where they are that long (the address is then a multiple of
// 16), element by element otherwise.
template <typename T, int V>
struct Pack {
    static constexpr int BYTES = V * int(sizeof(T)), WORDS = BYTES / 16;
    static constexpr bool WIDE = BYTES % 16 == 0;
    static_assert(WIDE || V == 1, "a vector is whole 16-byte words or one element");
    uint4 w[WIDE ? WORDS : 1];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
        } else {
            *reinterpret_cast<T *>(w) = *p;
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
        } else {
            *p = *reinterpret_cast<const T *>(w);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (auto &x : w) x = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f32(e[i]);
    }
    __device__ __forceinline__ void set(const float (&f)[V]) {
        T *e = reinterpret_cast<T *>(w);
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = from_f32<T>(f[i]);
    }
};

}  // namespace eg2
