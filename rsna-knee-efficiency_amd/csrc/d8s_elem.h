// Element types and wave reductions shared by the context layer's and the optimizer's kernels (not part of the C ABI).
#ifndef D8S_ELEM_H
#define D8S_ELEM_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#define DEV __device__ __forceinline__

namespace d8s {

typedef __bf16 bf16;
typedef _Float16 f16;

// N elements at any element's address: one wide load or store where N * sizeof(T) is 4, 8 or 16 bytes (the
// hardware takes any alignment of at least the element's)
template <class T, int N>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T, int N>
using Vec = typename VecOf<T, N>::type;

// f[0 .. N) = p[0 .. n), zeros from n on
template <class T, int N>
DEV void load_n(const T* p, int n, float* f) {
    if (n >= N) {
        const Vec<T, N> v = *(const Vec<T, N>*)p;
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = i < n ? (float)p[i] : 0.0f;
    }
}

// p[0 .. n) = f[0 .. n), each rounded to the nearest T (ties to even)
template <class T, int N>
DEV void store_n(T* p, int n, const float* f) {
    if (n >= N) {
        Vec<T, N> v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (T)f[i];
        *(Vec<T, N>*)p = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (T)f[i];
    }
}

template <int CTRL>
DEV float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// x of the lane's own 16 lanes and of the 16 beside them, in every one of the 32
DEV void swap16(float x, float& a, float& b) {
    const unsigned u = __float_as_uint(x);
    const u32x2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
// x of the wave's lower and upper half, in every lane
DEV void swap32(float x, float& a, float& b) {
    const unsigned u = __float_as_uint(x);
    const u32x2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}

// The sum over aligned groups of L lanes (8, 16, 32 or 64), in every lane of the group; the order is fixed.
// (row_ror within 16 lanes; with L = 8 the lanes 8 apart are left out)
template <int L>
DEV float lanes_sum(float x) {
    if constexpr (L == 8) {
        x += dpp<0xb1>(x);                     // quad_perm 1,0,3,2
        x += dpp<0x4e>(x);                     // quad_perm 2,3,0,1
        x += dpp<0x141>(x);                    // mirrored within 8 lanes
        return x;
    } else {
        x += dpp<0x128>(x);
        x += dpp<0x124>(x);
        x += dpp<0x122>(x);
        x += dpp<0x121>(x);
        float a, b;
        if constexpr (L >= 32) {
            swap16(x, a, b);
            x = a + b;
        }
        if constexpr (L >= 64) {
            swap32(x, a, b);
            x = a + b;
        }
        return x;
    }
}

}  // namespace d8s

#endif
