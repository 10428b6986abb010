// common.h -- scalar types, the matrix-core forms they take, activations and small helpers of the leaf-decoder kernels.
//
// The matrix cores multiply 16-bit operands and add in 32 bits.  bfloat16 and float16 go in as they are (one "plane").  A
// float32 number goes in as three bfloat16 numbers whose sum it is to within 2^-25 of itself,
//     hi = round(x),  mid = round(x - hi),  lo = round(x - hi - mid)      (8 significant bits each, signs of their own),
// and a product of two of them as the six products of planes whose weights are at least 2^-16 of the whole,
//     hi*hi' + hi*mid' + mid*hi' + hi*lo' + lo*hi' + mid*mid';
// what is left out is below 2^-24 of the product, as much as a 32-bit multiplication rounds away.  Six bfloat16 products cost
// 6/16 of what the 32-bit matrix instructions cost.  (Infinite inputs, and finite ones from 3.396e38 on, of which the first plane is
// infinite, give NaN: inf - inf in the second plane.  Numbers below 2^-109 lose bits, where bfloat16's numbers run out for the third plane.)
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "rules.h"

namespace svox_decoder {

typedef unsigned short u16;
typedef u16 u16x4 __attribute__((ext_vector_type(4)));
typedef u16 u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

typedef __bf16 Bf16;
typedef _Float16 F16;

// ---- a type's planes
template <class T>
struct Form;
template <>
struct Form<Bf16> {
    static constexpr int planes = 1;
    static __device__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ void split(f32x4 v, u16x4* out) { out[0] = __builtin_bit_cast(u16x4, __builtin_convertvector(v, bf16x4)); }
    static __device__ u16 one() { return 0x3f80; }
};
template <>
struct Form<F16> {
    static constexpr int planes = 1;
    static __device__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ void split(f32x4 v, u16x4* out) { out[0] = __builtin_bit_cast(u16x4, __builtin_convertvector(v, f16x4)); }
    static __device__ u16 one() { return 0x3c00; }
};
template <>
struct Form<float> {
    static constexpr int planes = 3;
    static __device__ f32x4 mma(u16x8 a, u16x8 b, f32x4 c) { return Form<Bf16>::mma(a, b, c); }
    static __device__ void split(f32x4 v, u16x4* out) {
        for (int p = 0; p < 3; ++p) {
            const bf16x4 part = __builtin_convertvector(v, bf16x4);
            out[p] = __builtin_bit_cast(u16x4, part);
            if (p < 2) v -= __builtin_convertvector(part, f32x4);
        }
    }
    static __device__ u16 one() { return 0x3f80; }
};

// c and the product of two fragments, all planes, the small products first.
//
// The matrix cores round a sum a little downwards whatever its sign.  float32 shows it: the planes' six products are therefore added
// up by themselves and c is added in 32 bits, rounded to nearest; and where results are summed up over many rows afterwards, as the
// gradients of the hidden numbers are for the biases', every other time the product of an operand turned around is taken away
// (multiply_turned), by steps of the reduction and by tiles of rows, so that the sums do not drift; b_down's sums, products with ones, are
// taken with minus ones every other time.  (A step of 43 345 rows of 239 -> 127 -> 239, relu, against 64 bits: gradients of x, the weights
// and b_up 3.9e-7, 6.5e-7 and 15e-7 off with all products added to c; 1.3e-7, 3.1e-7 and 2.0e-7 so, b_down's 1.4e-7.  131 072 rows of
// 80 -> 33 -> 20: b_gate, b_up and b_down 7.9e-7, 19e-7 and 2.9e-7 off where only the steps alternate and the ones do not, 2.7e-7, 2.6e-7 and
// 1.1e-7 so.)
template <class T>
__device__ __forceinline__ f32x4 product(const u16x8 (&a)[Form<T>::planes], const u16x8 (&b)[Form<T>::planes]) {
    f32x4 p = Form<T>::mma(a[1], b[1], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
    p = Form<T>::mma(a[0], b[2], p);
    p = Form<T>::mma(a[2], b[0], p);
    p = Form<T>::mma(a[0], b[1], p);
    p = Form<T>::mma(a[1], b[0], p);
    return Form<T>::mma(a[0], b[0], p);
}
template <class T>
__device__ __forceinline__ f32x4 multiply(const u16x8 (&a)[Form<T>::planes], const u16x8 (&b)[Form<T>::planes], f32x4 c) {
    if constexpr (Form<T>::planes == 3)
        return c + product<T>(a, b);
    else
        return Form<T>::mma(a[0], b[0], c);
}
template <class T>
__device__ __forceinline__ f32x4 multiply_turned(const u16x8 (&a)[Form<T>::planes], const u16x8 (&b)[Form<T>::planes], f32x4 c) {
    if constexpr (Form<T>::planes == 3) {
        u16x8 minus[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) minus[p] = b[p] ^ (u16)0x8000;
        return c - product<T>(a, minus);
    } else {
        return Form<T>::mma(a[0], b[0], c);
    }
}

// ---- a few values of a row at any alignment of the type's own
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Few {
    typedef T vector __attribute__((ext_vector_type(N)));
    vector v;
};
template <class T, int N>
__device__ __forceinline__ typename Few<T, N>::vector load_few(const T* at) {
    return reinterpret_cast<const Few<T, N>*>(at)->v;
}
template <class T, int N>
__device__ __forceinline__ void store_few(T* at, typename Few<T, N>::vector v) {
    reinterpret_cast<Few<T, N>*>(at)->v = v;
}

// N numbers from `at` on of which `room` can be read: all of them in one load, or one by one where there is no room.  What a branch
// leaves is the numbers as they lie in memory; they are converted behind it, so that the load is waited for there and not in the
// branch.
template <class T, int N>
__device__ __forceinline__ typename Few<T, N>::vector load_some(const T* at, int64_t room) {
    typename Few<T, N>::vector v;
    if (room >= N) {
        v = load_few<T, N>(at);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < room ? at[i] : (T)0.0f;
    }
    return v;
}

// 8 numbers as the matrix cores take them
template <class T>
__device__ __forceinline__ void planes_of(const typename Few<T, 8>::vector& v, u16x8 (&out)[Form<T>::planes]) {
    if constexpr (Form<T>::planes == 1) {
        out[0] = __builtin_bit_cast(u16x8, v);
    } else {
        u16x4 half[2][Form<T>::planes];
        Form<T>::split(f32x4{v[0], v[1], v[2], v[3]}, half[0]);
        Form<T>::split(f32x4{v[4], v[5], v[6], v[7]}, half[1]);
#pragma unroll
        for (int q = 0; q < Form<T>::planes; ++q) out[q] = __builtin_shufflevector(half[0][q], half[1][q], 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// ---- activations
enum Activation { kSilu = 0, kGelu = 1, kRelu = 2, kSigmoid = 3 };

// exp and the reciprocal: for results that are rounded to 16 bits the hardware's, good to 22 bits
template <bool accurate>
__device__ __forceinline__ float sigmoid(float g) {
    if constexpr (accurate) return 1.0f / (1.0f + expf(-g));
    return __builtin_amdgcn_rcpf(1.0f + __expf(-g));
}
// Phi(g), the normal distribution's, and exp(-g^2 / 2).  For results of 16 bits by 7.1.26 of Abramowitz and Stegun, Handbook of
// Mathematical Functions: erf to 1.5e-7, with the exponential that the derivative needs as well.  (That is an absolute error: g Phi(g) is
// off by 2.1e-7 at most, but by 2^-11 of itself at g = -4, 2^-8 at -6.2 and more beyond, where it is below 2e-9.)
template <bool accurate>
__device__ __forceinline__ float phi(float g, float& bell) {
    if constexpr (accurate) {
        bell = expf(-0.5f * g * g);
        return 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    } else {
        bell = __expf(-0.5f * g * g);
        const float x = __builtin_fabsf(g) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
        float poly = __builtin_fmaf(1.061405429f, t, -1.453152027f);
        poly = __builtin_fmaf(poly, t, 1.421413741f);
        poly = __builtin_fmaf(poly, t, -0.284496736f);
        poly = __builtin_fmaf(poly, t, 0.254829592f);
        const float beyond = 0.5f * poly * t * bell;   // 1 - Phi(|g|)
        return g < 0.0f ? beyond : 1.0f - beyond;
    }
}
// act(g); slope: its derivative too
template <bool accurate, int activation>
__device__ __forceinline__ float activate(float g, float* slope) {
    if constexpr (activation == kSilu) {
        const float s = sigmoid<accurate>(g), a = g * s;
        if (slope) *slope = __builtin_fmaf(a, 1.0f - s, s);
        return a;
    } else if constexpr (activation == kGelu) {
        float bell;
        const float below = phi<accurate>(g, bell);
        if (slope) *slope = __builtin_fmaf(g * 0.3989422804014327f, bell, below);
        return g * below;
    } else if constexpr (activation == kRelu) {
        // (NaN stays NaN; the derivative at 0 is 0)
        if (slope) *slope = g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
        return g < 0.0f ? 0.0f : g;
    } else {
        const float s = sigmoid<accurate>(g);
        if (slope) *slope = s * (1.0f - s);
        return s;
    }
}
// f with the activation as a constant, so that a loop over numbers asks once
template <class F>
__device__ __forceinline__ void with_activation(int activation, F f) {
    switch (activation) {
        case kSilu: return f(std::integral_constant<int, kSilu>());
        case kGelu: return f(std::integral_constant<int, kGelu>());
        case kRelu: return f(std::integral_constant<int, kRelu>());
        default: return f(std::integral_constant<int, kSigmoid>());
    }
}

__host__ __device__ inline int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

}  // namespace svox_decoder
