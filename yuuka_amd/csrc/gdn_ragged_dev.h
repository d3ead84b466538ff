// gdn_ragged_dev.h — what the kernels over ragged rows of the Gated DeltaNet
// layers share: element types, and the coefficients of a row.
#pragma once

#include "ragged_dev.h"
#include "refmath.h"

namespace yk {

struct RowF32 {
    typedef float T;
    static constexpr int kWide = 4;  // elements of 16 bytes
};
struct RowF16 {
    typedef _Float16 T;
    static constexpr int kWide = 8;
};
struct RowBF16 {
    typedef __bf16 T;
    static constexpr int kWide = 8;
};

typedef uint32_t Bytes16 __attribute__((ext_vector_type(4)));

// 16 bytes of a row as floats, and back (to the nearest, ties to even).
template <typename E> __device__ __forceinline__ void unpack(Bytes16 w, float (&x)[E::kWide]) {
    typename E::T v[E::kWide];
    __builtin_memcpy(v, &w, 16);
#pragma unroll
    for (int i = 0; i < E::kWide; i++) x[i] = (float)v[i];
}
template <typename E> __device__ __forceinline__ Bytes16 pack(const float (&x)[E::kWide]) {
    typename E::T v[E::kWide];
#pragma unroll
    for (int i = 0; i < E::kWide; i++) v[i] = (typename E::T)x[i];
    Bytes16 w;
    __builtin_memcpy(&w, v, 16);
    return w;
}

// The log of a row's decay and its step size (recurrent.go:66-70), in float32: the
// log is off by 2^-23 of itself.
__device__ __forceinline__ float log_decay_of(const GdnRows &b, const RaggedArgs &a, int64_t at, int h) {
    const float x = b.alpha[at];
    if (a.log_decay) return x;
    const float y = x + b.dt[h];
    return (y > 20.0f ? y : log1pf(expf(y))) * b.a[h];
}
__device__ __forceinline__ float beta_of(const GdnRows &b, const RaggedArgs &a, int64_t at) {
    const float x = b.beta[at];
    return a.log_decay ? x : 1.0f / (1.0f + expf(-x));
}

}  // namespace yk
