// Element types of the encoder-layer operators (rope.hip, gated_ff.hip, bucket_attn.hip) and the "pieces" their matrix
// products are made of.
//
// Products run on v_mfma_f32_*_bf16 (but for those of float16 inputs in gated_ff.hip beyond 64 rows).  A value is held as NP
// bf16 pieces, x = x0 + x1 + x2 with x0 = bf16(x), x1 = bf16(x - x0), x2 = bf16(x - x0 - x1):
//   bfloat16 : NP = 1, exact                       one product
//   float16  : NP = 2, exact (11 bits = 8 + 3)     x0 y0 + x0 y1 + x1 y0: what is dropped is 2^-16 of a term
//                                                  (attention's scores: all four, exact)
//   float32  : NP = 3, exact (24 bits = 8 + 8 + 8) the six products x_i y_j with i + j <= 2: dropped 2^-24 of a term
// bf16 has the exponent range of float32, so nothing over- or underflows on the way (float16 gradients in particular),
// and six bf16 products cost 6/16 of the time of one exact fp32 product (v_mfma_f32_32x32x2_f32 runs at 1/16 of the bf16
// rate).  A value whose bf16 rounding is infinite or NaN keeps no lower pieces (inf - inf would be NaN there).
#pragma once
#include "common.h"

typedef __bf16 bf16x2p __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4p __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8p __attribute__((ext_vector_type(8)));
typedef float f32x2p __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2p __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4p __attribute__((ext_vector_type(4)));

enum { ASR_T_F32 = 0, ASR_T_BF16 = 1, ASR_T_F16 = 2 };

template <int DT> struct ElemOf;
template <> struct ElemOf<ASR_T_F32> { typedef float type; static constexpr int NP = 3; };
template <> struct ElemOf<ASR_T_BF16> { typedef __bf16 type; static constexpr int NP = 1; };
template <> struct ElemOf<ASR_T_F16> { typedef _Float16 type; static constexpr int NP = 2; };

// V consecutive elements <-> fp32, one access of V * sizeof(E) bytes (the host has checked the alignment)
template <typename E, int V> struct VecOf { typedef E type __attribute__((ext_vector_type(V))); };
template <typename E> struct VecOf<E, 1> { typedef E type; };
template <typename E, int V>
__device__ __forceinline__ void load_vec(const E *p, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = (float)*p;
    } else if constexpr (sizeof(E) * V > 16) {
        float a[V / 2], b[V / 2];
        load_vec<E, V / 2>(p, a);
        load_vec<E, V / 2>(p + V / 2, b);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { v[i] = a[i]; v[V / 2 + i] = b[i]; }
    } else {
        const typename VecOf<E, V>::type t = *reinterpret_cast<const typename VecOf<E, V>::type *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)t[i];
    }
}
template <typename E, int V>
__device__ __forceinline__ void store_vec(E *p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = (E)v[0];
    } else if constexpr (sizeof(E) * V > 16) {
        float a[V / 2], b[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { a[i] = v[i]; b[i] = v[V / 2 + i]; }
        store_vec<E, V / 2>(p, a);
        store_vec<E, V / 2>(p + V / 2, b);
    } else {
        typename VecOf<E, V>::type t;
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = (E)v[i];
        *reinterpret_cast<typename VecOf<E, V>::type *>(p) = t;
    }
}

// two values -> one word per piece (low half = a); v_cvt_pk_bf16_f32 rounds to nearest even
__device__ __forceinline__ unsigned pk_bf16(float a, float b) {
    const f32x2p f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, bf16x2p));
}
// a - bf16(a) for the bf16 in the high half of `top`; 0 where that is infinite or NaN
__device__ __forceinline__ float piece_rest(float a, unsigned top) {
    const float r = a - __uint_as_float(top);
    return (top & 0x7f800000u) == 0x7f800000u ? 0.f : r;
}
template <int NP>
__device__ __forceinline__ void split_pair(float a, float b, unsigned (&w)[NP]) {
    w[0] = pk_bf16(a, b);
    if constexpr (NP > 1) {
        a = piece_rest(a, w[0] << 16);
        b = piece_rest(b, w[0] & 0xffff0000u);
        w[1] = pk_bf16(a, b);
    }
    if constexpr (NP > 2) w[2] = pk_bf16(a - __uint_as_float(w[1] << 16), b - __uint_as_float(w[1] & 0xffff0000u));
}
// the same for values known to be finite (probabilities, score gradients of finite inputs)
template <int NP>
__device__ __forceinline__ void split_pair_finite(float a, float b, unsigned (&w)[NP]) {
    w[0] = pk_bf16(a, b);
    if constexpr (NP > 1) {
        a -= __uint_as_float(w[0] << 16);
        b -= __uint_as_float(w[0] & 0xffff0000u);
        w[1] = pk_bf16(a, b);
    }
    if constexpr (NP > 2) w[2] = pk_bf16(a - __uint_as_float(w[1] << 16), b - __uint_as_float(w[1] & 0xffff0000u));
}

// What this wave's lanes wrote to LDS is seen by its other lanes.  The barrier costs no instruction, but without it the
// fences order the accesses of one lane only: the compiler may let the lanes that skip a branch run ahead of those that
// take it, and overwrite what these have yet to read.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
