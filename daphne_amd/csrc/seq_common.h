// Rows as 16-byte vectors wherever they begin and however long they are, for the sequence-model kernels. A vector load or
// store needs no more than its values' own alignment on this hardware; what rows of odd length cost is a line more per
// wavefront. The last vector of a row that is no whole number of them moves back until it ends with the row.
#pragma once

#include "common.h"

namespace dh_seq {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef double f64x2_any __attribute__((ext_vector_type(2), aligned(8)));
template <typename T> struct any_vec;
template <> struct any_vec<float> {
    using type = f32x4_any;
};
template <> struct any_vec<double> {
    using type = f64x2_any;
};

template <typename T, int VEC> __device__ __forceinline__ void load(const T *p, T (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = *p;
    } else {
        const typename any_vec<T>::type t = *reinterpret_cast<const typename any_vec<T>::type *>(p);
#pragma unroll
        for (int i = 0; i < VEC; i++)
            v[i] = t[i];
    }
}
// For data that is read once.
template <typename T, int VEC> __device__ __forceinline__ void load_stream(const T *p, T (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = __builtin_nontemporal_load(p);
    } else {
        const typename any_vec<T>::type t = __builtin_nontemporal_load(reinterpret_cast<const typename any_vec<T>::type *>(p));
#pragma unroll
        for (int i = 0; i < VEC; i++)
            v[i] = t[i];
    }
}

// Most workgroups of one launch along x, far below where a grid's threads no longer count in 32 bits. What needs more takes several
// launches, or several turns of a workgroup.
constexpr size_t MOST_GROUPS = size_t(1) << 20;

// Vector j of n values: where it begins, and how many of its values belong to the vector before it.
struct Piece {
    size_t at;
    size_t shift; // at least VEC: there is no vector j
};
template <int VEC> __device__ __forceinline__ Piece piece(size_t j, size_t n) {
    const size_t at = j * VEC;
    return at + VEC <= n ? Piece{at, 0} : Piece{n - VEC, at + VEC - n};
}

// Stores the values that belong to the vector itself (none if there is no such vector), so that nobody writes a value that
// another thread may not have read yet.
template <typename T, int VEC, bool STREAM = false> __device__ __forceinline__ void store(T *p, const T (&v)[VEC], size_t shift) {
    if (shift == 0) {
        if constexpr (VEC == 1) {
            *p = v[0];
        } else {
            typename any_vec<T>::type t;
#pragma unroll
            for (int i = 0; i < VEC; i++)
                t[i] = v[i];
            if constexpr (STREAM)
                __builtin_nontemporal_store(t, reinterpret_cast<typename any_vec<T>::type *>(p));
            else
                *reinterpret_cast<typename any_vec<T>::type *>(p) = t;
        }
    } else {
#pragma unroll
        for (int i = 1; i < VEC; i++)
            if (static_cast<size_t>(i) >= shift)
                p[i] = v[i];
    }
}

} // namespace dh_seq
