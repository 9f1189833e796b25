// Device helpers of the block operators (gated_norm.hip, linear_i8.hip, prefix_attention.hip): element types, 16-byte
// accesses, wave sums on the vector ALU.  All arithmetic is fp32; a type is converted where it is loaded or stored.
#pragma once
#include <float.h>

#include "common.hpp"

namespace cmdi {

typedef unsigned short bf16_bits;
struct Bf16 { bf16_bits v; };

template <class T> struct Elem;
template <> struct Elem<float> {
    static constexpr int W = 4;                                   // elements of a 16-byte access
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<_Float16> {
    static constexpr int W = 8;
    static __device__ __forceinline__ float up(_Float16 x) { return (float)x; }
    static __device__ __forceinline__ _Float16 down(float x) { return (_Float16)x; }
};
template <> struct Elem<Bf16> {
    static constexpr int W = 8;
    static __device__ __forceinline__ float up(Bf16 x) { return __uint_as_float((unsigned)x.v << 16); }
    // nearest, ties to even, NaN stays NaN (v_cvt_pk_bf16_f32)
    static __device__ __forceinline__ Bf16 down(float x) { return Bf16{__builtin_bit_cast(bf16_bits, (__bf16)x)}; }
};

// W consecutive elements <-> fp32 registers, one access of up to 16 bytes at any element's address (the hardware takes vector
// accesses that straddle their alignment; the compiler is told that an element's alignment is all there is).
template <class T, int W>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[W]) {
    struct __attribute__((packed, aligned(sizeof(T)))) Pack { T e[W]; };
    const Pack k = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = Elem<T>::up(k.e[i]);
}
template <class T, int W>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[W]) {
    struct __attribute__((packed, aligned(sizeof(T)))) Pack { T e[W]; };
    Pack k;
#pragma unroll
    for (int i = 0; i < W; ++i) k.e[i] = Elem<T>::down(v[i]);
    *reinterpret_cast<Pack*>(p) = k;
}
// the same of the first `n` of them (the end of a row); the others read as 0
template <class T, int W>
__device__ __forceinline__ void load_part(const T* p, float (&v)[W], int n) {
    if (n >= W) {
        load_vec<T, W>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = i < n ? Elem<T>::up(p[i]) : 0.f;
    }
}
template <class T, int W>
__device__ __forceinline__ void store_part(T* p, const float (&v)[W], int n) {
    if (n >= W) {
        store_vec<T, W>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < n) p[i] = Elem<T>::down(v[i]);
    }
}

// Sum / maximum over the 64 lanes, the same value in every lane.  Rows of 16 lanes by data-parallel-primitive moves (one
// vector instruction a step instead of a round trip through LDS), then the four rows by broadcasts into the last lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_mov(float old, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_total(float v) {
    v += dpp_mov<0xB1, 0xf>(0.f, v);    // quad_perm [1,0,3,2]
    v += dpp_mov<0x4E, 0xf>(0.f, v);    // quad_perm [2,3,0,1]
    v += dpp_mov<0x141, 0xf>(0.f, v);   // row_half_mirror
    v += dpp_mov<0x140, 0xf>(0.f, v);   // row_mirror: every lane holds its row's sum
    v += dpp_mov<0x142, 0xa>(0.f, v);   // row_bcast15 into rows 1, 3
    v += dpp_mov<0x143, 0xc>(0.f, v);   // row_bcast31 into rows 2, 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_highest(float v) {
    v = fmaxf(v, dpp_mov<0xB1, 0xf>(v, v));
    v = fmaxf(v, dpp_mov<0x4E, 0xf>(v, v));
    v = fmaxf(v, dpp_mov<0x141, 0xf>(v, v));
    v = fmaxf(v, dpp_mov<0x140, 0xf>(v, v));
    v = fmaxf(v, dpp_mov<0x142, 0xa>(v, v));
    v = fmaxf(v, dpp_mov<0x143, 0xc>(v, v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// The block's barrier without the waits of __syncthreads(): those of this wave's LDS accesses and requests that the barrier stands for
// come before it, counted; no access moves over it in either direction.
__device__ __forceinline__ void meet_waves() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace cmdi
