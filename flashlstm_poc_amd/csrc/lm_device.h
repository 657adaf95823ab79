// Shared helpers of the language-model operators (lm_ops.h): element types, loads and stores of any alignment, reductions.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/flashlstm/lm_ops.h"
#include "../../include/flashlstm/lstm_core.h"
#include "common.h"

namespace flstm_hip {

typedef __bf16 bfloat_t;
typedef float float8 __attribute__((ext_vector_type(8)));

template <class T> struct Vec8;
template <> struct Vec8<half_t> { typedef half8 type; };
template <> struct Vec8<bfloat_t> { typedef __bf16 type __attribute__((ext_vector_type(8))); };
template <> struct Vec8<float> { typedef float8 type; };

// Eight consecutive elements as floats.  The hardware loads 16 bytes from any address, so callers' tensors may begin anywhere;
// only the element type's own alignment is assumed.
template <class T> __device__ __forceinline__ float8 load8(const T* p) {
    typename Vec8<T>::type v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), sizeof(v));
    return __builtin_convertvector(v, float8);
}
template <class T> __device__ __forceinline__ void store8(T* p, float8 v) {
    const typename Vec8<T>::type r = __builtin_convertvector(v, typename Vec8<T>::type);
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &r, sizeof(r));
}
// N consecutive elements, N a power of two up to 4, at places `at` .. of a vector of eight
template <class T, int N> __device__ __forceinline__ void load_part(float8& v, int at, const T* p) {
    T e[N];
    __builtin_memcpy(e, __builtin_assume_aligned(p, sizeof(T)), sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; i += N)
#pragma unroll
        for (int j = 0; j < N; ++j) v[i + j] = at == i ? float(e[j]) : v[i + j];
}
template <class T, int N> __device__ __forceinline__ void store_part(float8 v, int at, T* p) {
    T e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float x = v[j];
#pragma unroll
        for (int i = N; i < 8; i += N) x = at == i ? v[i + j] : x;
        e[j] = T(x);
    }
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), e, sizeof(e));
}
// The same for a row's last vector, of which `n` elements exist (n <= 0: none; the others read as zero): in parts of 4, 2 and 1.
template <class T> __device__ __forceinline__ float8 load8(const T* p, int n) {
    if (n >= 8) return load8(p);
    float8 v = 0.f;
    if (n > 0) {
        if (n & 4) load_part<T, 4>(v, 0, p);
        if (n & 2) load_part<T, 2>(v, n & 4, p + (n & 4));
        if (n & 1) load_part<T, 1>(v, n & 6, p + (n & 6));
    }
    return v;
}
template <class T> __device__ __forceinline__ void store8(T* p, float8 v, int n) {
    if (n >= 8) return store8(p, v);
    if (n > 0) {
        if (n & 4) store_part<T, 4>(v, 0, p);
        if (n & 2) store_part<T, 2>(v, n & 4, p + (n & 4));
        if (n & 1) store_part<T, 1>(v, n & 6, p + (n & 6));
    }
}

// A value folded over groups of `N` neighbouring lanes (a power of two up to a wave), in every lane: lanes 1 and 2 apart, mirrored
// halves of eight and of sixteen (each half holds one value by then), then rows of sixteen and of thirty-two exchanged.  Moves
// inside the vector unit, a few clocks each, where a shuffle goes through LDS.
template <int CTRL> __device__ __forceinline__ float lane_moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int N, class Op> __device__ __forceinline__ float lanes_fold(float v, Op op) {
    static_assert(N == 8 || N == 16 || N == 32 || N == 64, "whole groups of eight");
    v = op(v, lane_moved<0xb1>(v));            // quad_perm 1, 0, 3, 2
    v = op(v, lane_moved<0x4e>(v));            // quad_perm 2, 3, 0, 1
    v = op(v, lane_moved<0x141>(v));           // row_half_mirror
    if constexpr (N >= 16) v = op(v, lane_moved<0x140>(v));   // row_mirror
    if constexpr (N >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = op(__builtin_bit_cast(float, unsigned(r[0])), __builtin_bit_cast(float, unsigned(r[1])));
    }
    if constexpr (N >= 64) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = op(__builtin_bit_cast(float, unsigned(r[0])), __builtin_bit_cast(float, unsigned(r[1])));
    }
    return v;
}
template <int N> __device__ __forceinline__ float lanes_sum(float v) {
    return lanes_fold<N>(v, [](float a, float b) { return a + b; });
}
template <int N> __device__ __forceinline__ float lanes_max(float v) {
    return lanes_fold<N>(v, [](float a, float b) { return fmaxf(a, b); });
}

__host__ __device__ inline bool valid_dtype(int t) { return t == FLSTM_OP_F32 || t == FLSTM_OP_F16 || t == FLSTM_OP_BF16; }

// Calls `f` with a value of the element type that `dtype` names.
template <class F> inline int with_type(flstm_op_dtype dtype, F&& f) {
    switch (dtype) {
        case FLSTM_OP_F32: return f(float());
        case FLSTM_OP_F16: return f(half_t());
        case FLSTM_OP_BF16: return f(bfloat_t());
    }
    return FLSTM_E_INVALID;
}

inline int launched() { return int(hipGetLastError()); }

}  // namespace flstm_hip
