// Element types of the token operators (qk_rotate.hip, block_sparse.hip): fp32, bf16 and fp16 tensors, all arithmetic in fp32.
#pragma once
#include <hip/hip_fp16.h>

#include <cmath>
#include <cstdint>

#include "av2x_common.hpp"

namespace {

enum TokDtype { kTokF32 = 0, kTokBF16 = 1, kTokF16 = 2 };      // dtype argument of the C-ABI

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T> struct tok_vec { typedef T v4 __attribute__((ext_vector_type(4))); typedef T v8 __attribute__((ext_vector_type(8))); };

template <typename T> __device__ __forceinline__ f32x4 tok_load4(const T* p) {      // four elements, aligned to their own size
    return __builtin_convertvector(*reinterpret_cast<const typename tok_vec<T>::v4*>(p), f32x4);
}
template <typename T> __device__ __forceinline__ void tok_store4(T* p, f32x4 v) {   // rounded to nearest even
    *reinterpret_cast<typename tok_vec<T>::v4*>(p) = __builtin_convertvector(v, typename tok_vec<T>::v4);
}

// f(std::integral_constant-like T{}) for the C-ABI's dtype
#define AV2X_TOK_DISPATCH(dtype, T, ...)                                   \
    do {                                                                   \
        if ((dtype) == kTokF32) { using T = float; __VA_ARGS__; }          \
        else if ((dtype) == kTokBF16) { using T = __bf16; __VA_ARGS__; }   \
        else { using T = _Float16; __VA_ARGS__; }                          \
    } while (0)

inline size_t tok_size(int dtype) { return dtype == kTokF32 ? 4 : 2; }
inline bool tok_aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
