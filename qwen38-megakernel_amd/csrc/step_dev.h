// Device-side building blocks of the step operators (step_*.hip): rows of fp32 / fp16 / bf16 values at any alignment, and
// reductions over a wave.
#pragma once
#include "kv_dev.h"
#include "step_launch.h"

namespace qkv {

// 8 consecutive values as loads of 16 bytes that need no more than the type's own alignment (the rows of a strided or
// odd-sized tensor; the hardware splits a load that crosses a cache line)
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t u16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 f16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// the largest of 8 16-bit floats by their bits without the sign
__device__ __forceinline__ uint16_t top16(u16x8 v) {
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    v &= (uint16_t) 0x7fff;
    const u16x4 a = __builtin_elementwise_max(v.lo, v.hi);
    const u16x2 b = __builtin_elementwise_max(a.lo, a.hi);
    return b[0] > b[1] ? b[0] : b[1];
}

// Raw8: 8 values as they are in memory; open8: as floats; top8: the bits of the largest one's absolute value as fp32 (an
// infinity or a NaN where there is one)
template <int DT> struct Elem;
template <> struct Elem<DT_F32> {
    typedef float T;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ T down(float v) { return v; }
    struct Raw8 {
        f32x4 a, b;
    };
    static __device__ __forceinline__ Raw8 raw8(const T * p) {
        return Raw8{*reinterpret_cast<const f32x4_u *>(p), *reinterpret_cast<const f32x4_u *>(p + 4)};
    }
    static __device__ __forceinline__ void open8(const Raw8 & r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = r.a[i], v[4 + i] = r.b[i];
    }
    static __device__ __forceinline__ unsigned top8(const Raw8 & r) {
        unsigned t = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = r.a[i], y = r.b[i]; // (a bit cast of a vector's element itself takes the first one)
            t = max(max(t, __builtin_bit_cast(unsigned, x) & 0x7fffffffu), __builtin_bit_cast(unsigned, y) & 0x7fffffffu);
        }
        return t;
    }
    static __device__ __forceinline__ void load4(const T * p, float (&v)[4]) {
        const f32x4_u a = *reinterpret_cast<const f32x4_u *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = a[i];
    }
    static __device__ __forceinline__ void store8(T * p, const float (&v)[8]) {
        *reinterpret_cast<f32x4_u *>(p) = f32x4_u{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_u *>(p + 4) = f32x4_u{v[4], v[5], v[6], v[7]};
    }
};
template <> struct Elem<DT_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float up(T v) { return (float) v; }
    static __device__ __forceinline__ T down(float v) { return (T) v; }
    typedef half8 Raw8;
    static __device__ __forceinline__ Raw8 raw8(const T * p) { return *reinterpret_cast<const f16x8_u *>(p); }
    static __device__ __forceinline__ void open8(const Raw8 & r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float) r[i];
    }
    static __device__ __forceinline__ unsigned top8(const Raw8 & r) {
        return __builtin_bit_cast(unsigned, (float) __builtin_bit_cast(_Float16, top16(__builtin_bit_cast(u16x8, r))));
    }
    static __device__ __forceinline__ void load4(const T * p, float (&v)[4]) {
        const f16x4_u a = *reinterpret_cast<const f16x4_u *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (float) a[i];
    }
    static __device__ __forceinline__ void store8(T * p, const float (&v)[8]) {
        f16x8_u a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (T) v[i];
        *reinterpret_cast<f16x8_u *>(p) = a;
    }
};
template <> struct Elem<DT_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float up(T v) { return __builtin_bit_cast(float, (unsigned) __builtin_bit_cast(uint16_t, v) << 16); }
    static __device__ __forceinline__ T down(float v) { return (T) v; }
    typedef u16x8 Raw8;
    static __device__ __forceinline__ Raw8 raw8(const T * p) { return *reinterpret_cast<const u16x8_u *>(p); }
    static __device__ __forceinline__ void open8(const Raw8 & r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __builtin_bit_cast(float, (unsigned) r[i] << 16);
    }
    static __device__ __forceinline__ unsigned top8(const Raw8 & r) { return (unsigned) top16(r) << 16; }
    static __device__ __forceinline__ void load4(const T * p, float (&v)[4]) {
        const u16x4_u a = *reinterpret_cast<const u16x4_u *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __builtin_bit_cast(float, (unsigned) a[i] << 16);
    }
    static __device__ __forceinline__ void store8(T * p, const float (&v)[8]) {
        bf16x8_u a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (T) v[i];
        *reinterpret_cast<bf16x8_u *>(p) = a;
    }
};

template <int DT> __device__ __forceinline__ void load8(const typename Elem<DT>::T * p, float (&v)[8]) { Elem<DT>::open8(Elem<DT>::raw8(p), v); }

// a launch and its own status (hipGetLastError would also give what an earlier call of the thread left)
template <class A> inline hipError_t launch(void (*k)(A), dim3 grid, dim3 block, size_t lds, hipStream_t st, A a) {
    void * args[] = {&a};
    return hipLaunchKernel(reinterpret_cast<const void *>(k), grid, block, args, lds, st);
}

// the first n (1..8) of 8 values, the rest zero
template <int DT> __device__ __forceinline__ void load_n(const typename Elem<DT>::T * p, int n, float (&v)[8]) {
    if (n >= 8) return load8<DT>(p, v);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < n ? Elem<DT>::up(p[i]) : 0.f;
}
template <int DT> __device__ __forceinline__ void store_n(typename Elem<DT>::T * p, int n, const float (&v)[8]) {
    if (n >= 8) return Elem<DT>::store8(p, v);
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) p[i] = Elem<DT>::down(v[i]);
}

// a workgroup barrier for LDS data only: __syncthreads() also waits for the wave's loads and stores in flight
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ double shfl_xor_d(double v, int m) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = shfl_xor_u((unsigned) b, m), hi = shfl_xor_u((unsigned) (b >> 32), m);
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
// sum over the wave, the same bits in every lane
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += shfl_xor_d(v, m);
    return v;
}

} // namespace qkv
