// sqd_vec.h — element types of the token operators (token_norm.hip, rotary.hip, attention*.hip): fp32, bf16 and fp16 rows read in 16-byte
// pieces, all arithmetic in fp32, one round-to-nearest-even at the store.
#pragma once
#include <algorithm>

#include "sqd_common.h"

namespace sqd {

struct bf16_t { unsigned short v; };
struct f16_t { _Float16 v; };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((unsigned)x.v << 16); }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x.v; }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) { return bf16_t{__builtin_bit_cast(unsigned short, (__bf16)x)}; }
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float x) { return f16_t{(_Float16)x}; }

// N elements of memory as fp32 values; one 16-byte (or, for N elements of less than 16 bytes, one scalar) access
template <typename T, int N> struct alignas(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Pack { T e[N]; };
template <typename T, int N> __device__ __forceinline__ void load_f32(const T *p, float (&out)[N]) {
    const Pack<T, N> v = *reinterpret_cast<const Pack<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_f32(v.e[i]);
}
template <typename T, int N> __device__ __forceinline__ void store_f32(T *p, const float (&in)[N]) {
    Pack<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = from_f32<T>(in[i]);
    *reinterpret_cast<Pack<T, N> *>(p) = v;
}

// workgroups of NTH threads that one launch takes: a grid counts its threads in 32 bits, and a larger one is cut modulo 2^32 without an error
constexpr int64_t max_blocks(int nth) { return ((1ll << 32) - 1) / nth; }

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// f(T{}) for the element type a `dtype` argument names
template <typename F> inline int for_dtype(int dtype, F &&f) {
    switch (dtype) {
        case SQD_F32: return f(float{});
        case SQD_BF16: return f(bf16_t{});
        case SQD_F16: return f(f16_t{});
    }
    set_error("element type %d unknown (SQD_F32 | SQD_BF16 | SQD_F16)", dtype);
    return SQD_EINVAL;
}
}  // namespace sqd
