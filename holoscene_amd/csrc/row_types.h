// row_types.h -- storage types of the row operators (dropout.hip, embed_rows.hip, gated_mlp.hip): elements to and from fp32, and loads and
// stores of several consecutive elements at the widest access the address allows.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "holoscene_hip.h"

namespace hs_row {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }      // round to nearest even

template <typename T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack { T v[N]; };      // an aligned group of elements
template <typename T, int N> struct __attribute__((packed, aligned(1))) Loose { T v[N]; };                  // the same at any address: gfx950 loads and stores unaligned dwords

__host__ inline int elem_bytes(int32_t dtype) { return dtype == HS_F32 ? 4 : 2; }
__host__ inline bool known_dtype(int32_t dtype) { return dtype == HS_F32 || dtype == HS_BF16 || dtype == HS_F16; }

}  // namespace hs_row

// Calls f with a value of the element type that `dtype` names (the caller has checked known_dtype).
#define HS_BY_DTYPE(dtype, ...)                                        \
    do {                                                               \
        if ((dtype) == HS_F32) { using T = float; __VA_ARGS__; }       \
        else if ((dtype) == HS_BF16) { using T = hs_row::bf16_t; __VA_ARGS__; } \
        else { using T = hs_row::f16_t; __VA_ARGS__; }                 \
    } while (0)
