// Element types of the entry points that take fp32, bf16 or fp16 operands (DDG_F32 / DDG_BF16 / DDG_F16): dispatch, and
// loads / stores of eight consecutive elements as fp32 values.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

static inline bool ddg_type_ok(int t) { return t == DDG_F32 || t == DDG_BF16 || t == DDG_F16; }

// workgroups that a launch takes at most: it counts its threads in 32 bits
static inline int64_t ddg_max_grid(int threads) { return 0xFFFFFFFFll / threads; }

// calls f(T()) with the element type of code t, which the caller has checked with ddg_type_ok
template <class F> static inline int ddg_with_type(int t, F &&f) {
    switch (t) {
        case DDG_F32: return f(float());
        case DDG_BF16: return f(bf16_t());
        default: return f(f16_t());
    }
}

// a 16-byte store past the caches, at any alignment
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ void store16_streaming(void *p, const void *v) {
    i32x4_any w;
    __builtin_memcpy(&w, v, 16);
    __builtin_nontemporal_store(w, (i32x4_any *)p);
}

// n <= N consecutive elements -> fp32 (elements from n on read as 0).  A full vector is moved with the widest access; the
// address needs the alignment of one element only (gfx950 serves unaligned 16-byte accesses of global memory), so rows of
// odd length take the same path.  STREAM: past the caches, for what is larger than they are and touched once.
template <int N, bool STREAM = false, class T> __device__ __forceinline__ void load_n(const T *p, int n, float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (n >= N) {
        const vec t = STREAM ? __builtin_nontemporal_load((const vec *)p) : *(const vec *)p;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}
template <int N, bool STREAM = false, class T> __device__ __forceinline__ void store_n(T *p, int n, const float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (n >= N) {
        vec t;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = (T)v[i];
        if (STREAM) __builtin_nontemporal_store(t, (vec *)p);
        else *(vec *)p = t;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// eight consecutive elements, all of them in bounds: one load without a branch around it
template <class T> using vec8 = T __attribute__((ext_vector_type(8)));
template <bool STREAM = false, class T> __device__ __forceinline__ vec8<T> load_whole(const T *p) {
    typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    return STREAM ? __builtin_nontemporal_load((const vec *)p) : *(const vec *)p;
}

// maximum over the 16 lanes of a DPP row, in every lane
__device__ __forceinline__ float row16_max(float x) {
#define DDG_DPP_MAX(ctrl)                                                                                                   \
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xF, 0xF, true)))
    DDG_DPP_MAX(0xB1);       // quad_perm [1,0,3,2]
    DDG_DPP_MAX(0x4E);       // quad_perm [2,3,0,1]
    DDG_DPP_MAX(0x141);      // row_half_mirror
    DDG_DPP_MAX(0x140);      // row_mirror
#undef DDG_DPP_MAX
    return x;
}
