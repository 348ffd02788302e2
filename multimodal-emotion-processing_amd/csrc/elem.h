// Element types and 16-byte row accesses shared by the differential-attention block's kernels
// (rotary.hip, block_norm.hip, diff_attn.hip).
#pragma once
#include "common.h"

namespace mep {

// MEP_F32 / MEP_BF16 / MEP_F16 storage.  Loads widen to fp32 exactly; stores round to nearest even.
template <int TYPE> struct ElemOf;
template <> struct ElemOf<MEP_F32> { typedef float T; };
template <> struct ElemOf<MEP_BF16> { typedef __bf16 T; };
template <> struct ElemOf<MEP_F16> { typedef _Float16 T; };

// V consecutive elements (V * sizeof(T) a power of two, at most 16 bytes: one access).  `loose`: at any element's address (the
// hardware's unaligned access; rows of an odd width start at any)
template <class T, int V> struct VecOf {
    typedef T type __attribute__((ext_vector_type(V)));
    typedef type loose __attribute__((aligned(sizeof(T))));
};
template <class T> struct VecOf<T, 1> { typedef T type, loose; };

// V elements at p as fp32, in accesses of at most 16 bytes
template <class T, int V>
MEP_DEV void load_f32(const MEP_G T* p, float (&v)[V]) {
    constexpr int N = V * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
#pragma unroll
    for (int i = 0; i < V; i += N) {
        const typename VecOf<T, N>::type w = *reinterpret_cast<const MEP_G typename VecOf<T, N>::loose*>(p + i);
        if constexpr (N == 1) {
            v[i] = (float)w;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[i + j] = (float)w[j];
        }
    }
}

template <class T, int V>
MEP_DEV void store_f32(MEP_G T* p, const float (&v)[V]) {
    constexpr int N = V * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
#pragma unroll
    for (int i = 0; i < V; i += N) {
        typename VecOf<T, N>::type w;
        if constexpr (N == 1) {
            w = (T)v[i];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = (T)v[i + j];
        }
        *reinterpret_cast<MEP_G typename VecOf<T, N>::loose*>(p + i) = w;
    }
}

}  // namespace mep
