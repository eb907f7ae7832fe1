// Element types and vectors shared by the layer norm, AdamW and attention kernels.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "rwk_common.h"

// The 16-bit types travel as raw bits in vectors of the compiler's own types, so that conversions are single
// instructions (v_cvt_f16_f32, v_cvt_pk_bf16_f32) rounding to nearest even.
using rwk_f16 = _Float16;
using rwk_bf16 = __bf16;

template <typename T> struct RwkVecOf { static constexpr int n = 16 / (int)sizeof(T); };

// N elements with the alignment of one: a row of odd width begins at any element.  gfx950 serves global accesses of
// 16 bytes at any address, so rows of every width use the same wide loads.
template <typename T, int N>
struct RwkPack {
    typedef T type __attribute__((ext_vector_type(N)));
    typedef T loose __attribute__((ext_vector_type(N), aligned(alignof(T))));
};

template <typename T, int N>
__device__ static inline typename RwkPack<T, N>::type rwk_load(const T *p) {
    return *reinterpret_cast<const typename RwkPack<T, N>::loose *>(p);
}

template <typename T, int N>
__device__ static inline void rwk_store(T *p, typename RwkPack<T, N>::type v) {
    *reinterpret_cast<typename RwkPack<T, N>::loose *>(p) = v;
}

// A pointer that came out of a table in memory, as one into global memory: the compiler cannot know, and accesses that
// might be to LDS as well are slower.
template <typename T> using RwkGlobal = __attribute__((address_space(1))) T *;
template <typename T>
__device__ static inline RwkGlobal<T> rwk_global(void *p) {
    return (RwkGlobal<T>)(uintptr_t)p;
}
template <typename T, int N>
__device__ static inline typename RwkPack<T, N>::type rwk_load(RwkGlobal<T> p) {
    return *(RwkGlobal<typename RwkPack<T, N>::loose>)p;
}
template <typename T, int N>
__device__ static inline void rwk_store(RwkGlobal<T> p, typename RwkPack<T, N>::type v) {
    *(RwkGlobal<typename RwkPack<T, N>::loose>)p = v;
}

// sum over the 64 lanes, in a fixed order, to every lane
__device__ static inline float rwk_wave_sum(float v) { return rwk_group_sum(v, 64); }
