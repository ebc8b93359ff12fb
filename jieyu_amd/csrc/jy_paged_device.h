// jy_paged_device.h — element types and slots of the paged cache, on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jieyu_amd.h"
#include "jy_paged.h"

namespace jy {

template <int T>
struct ElemOf;
template <>
struct ElemOf<JYHIP_T_F32> {
    typedef float type;
};
template <>
struct ElemOf<JYHIP_T_F16> {
    typedef _Float16 type;
};
template <>
struct ElemOf<JYHIP_T_BF16> {
    typedef __bf16 type;
};
template <>
struct ElemOf<JYHIP_T_I8> {
    typedef int8_t type;
};
template <int T>
using elem_t = typename ElemOf<T>::type;

// N elements at p as floats and back (one rounding to nearest even); VEC: p is aligned to
// min(16, N * sizeof(E)) bytes, else only to one element
template <class E, int N, bool VEC>
__device__ __forceinline__ void load_n(const E* p, float (&x)[N]) {
    if constexpr (VEC) {
        constexpr int B = (int)(N * sizeof(E)), W = B < 16 ? B : 16;
        typedef E vec __attribute__((ext_vector_type(W / sizeof(E))));
        constexpr int PER = W / (int)sizeof(E);
#pragma unroll
        for (int c = 0; c < N / PER; c++) {
            const vec v = reinterpret_cast<const vec*>(p)[c];
#pragma unroll
            for (int i = 0; i < PER; i++) x[c * PER + i] = (float)v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = (float)p[i];
    }
}

template <class E, int N, bool VEC>
__device__ __forceinline__ void store_n(E* p, const float (&x)[N]) {
    if constexpr (VEC) {
        constexpr int B = (int)(N * sizeof(E)), W = B < 16 ? B : 16;
        typedef E vec __attribute__((ext_vector_type(W / sizeof(E))));
        constexpr int PER = W / (int)sizeof(E);
#pragma unroll
        for (int c = 0; c < N / PER; c++) {
            vec v;
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = (E)x[c * PER + i];
            reinterpret_cast<vec*>(p)[c] = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = (E)x[i];
    }
}

// the slot of (sequence, position) as an index over [num_pages][page_size], -1 where there is none;
// page_size = 1 << ps_log2
__device__ __forceinline__ int64_t slot_of(const PageMap& M, int num_pages, int ps_log2, int seq, int pos) {
    const int at = pos >> ps_log2;
    if ((seq < 0) | (seq >= M.nseq) | (pos < 0) | (at >= M.stride)) return -1;  // (one branch)
    const int page = M.tables[(int64_t)seq * M.stride + at];
    if (page < 0 || page >= num_pages) return -1;
    return ((int64_t)page << ps_log2) + (pos & ((1 << ps_log2) - 1));
}

// groups of 32 elements of a 4-bit vector as it is laid out, so that its bytes and its groups' words are
// aligned to their sizes
__host__ __device__ __forceinline__ int groups4(int hd) { return hd <= 64 ? 2 : hd <= 128 ? 4 : 8; }

}  // namespace jy
