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

// V consecutive elements, held in their own type and moved in the widest accesses
// of 2 to 16 bytes that divide them; the address is a multiple of that width.
template <int BYTES>
struct Word;
template <>
struct Word<2> {
    using type = uint16_t;
};
template <>
struct Word<4> {
    using type = uint32_t;
};
template <>
struct Word<8> {
    using type = uint2;
};
template <>
struct Word<16> {
    using type = uint4;
};
template <typename T, int V>
struct Pack {
    static constexpr int BYTES = V * int(sizeof(T)), WIDTH = BYTES < 16 ? BYTES : 16, WORDS = BYTES / WIDTH;
    using W = typename Word<WIDTH>::type;
    union {
        W w[WORDS];
        T e[V];
    };
    __device__ __forceinline__ Pack() {}
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const W *>(p)[i];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) reinterpret_cast<W *>(p)[i] = w[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = W{};
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f32(e[i]);
    }
    __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = from_f32<T>(f[i]);
    }
};

// ---------------------------------------------------------------- pairs
// Two fp32 operations in one instruction (FFMA2 and its kin), each rounded as
// its scalar form: half the issue slots of a row kernel's arithmetic.
__device__ __forceinline__ uint64_t bits2(float2 a) {
    return uint64_t(__float_as_uint(a.x)) | uint64_t(__float_as_uint(a.y)) << 32;
}
__device__ __forceinline__ float2 pair2(uint64_t b) {
    return make_float2(__uint_as_float(uint32_t(b)), __uint_as_float(uint32_t(b >> 32)));
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
    return pair2(d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
    return pair2(d);
}
// A 16-byte vector of T as pairs, and back (each element rounded once).
__device__ __forceinline__ void unpack2(const uint4 &w, float2 (&f)[2], float) {
    f[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    f[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ void unpack2(const uint4 &w, float2 (&f)[4], __half) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(h[i]);
}
__device__ __forceinline__ void unpack2(const uint4 &w, float2 (&f)[4], __nv_bfloat16) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint4 packed(const float2 (&f)[2], float) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}
template <typename T>
__device__ __forceinline__ uint4 packed(const float2 (&f)[4], T) {
    return make_uint4(pack2<T>(f[0].x, f[0].y), pack2<T>(f[1].x, f[1].y), pack2<T>(f[2].x, f[2].y),
                      pack2<T>(f[3].x, f[3].y));
}

// ---------------------------------------------------------------- copies to shared memory
// 16 bytes from global to shared memory, or 16 zero bytes (nothing is read) when
// `on` is false; complete after copies_wait<K>() leaves at most K committed
// groups of this thread outstanding.
__device__ __forceinline__ void copy16(uint4 *dst, const void *src, bool on) {
    asm volatile(
        "{\n\t.reg .pred off;\n\t"
        "setp.eq.u32 off, %2, 0;\n\t"
        "cp.async.cg.shared.global [%0], [%1], 16, off;\n\t}" ::"r"(smem_u32(dst)),
        "l"(src), "r"(uint32_t(on))
        : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int K>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(K) : "memory");
}

}  // namespace eg2
