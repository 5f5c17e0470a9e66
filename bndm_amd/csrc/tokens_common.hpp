// Shared by the kernels of libbndm_tokens.so (gfx950 only): element types, matrix-instruction wrappers, LDS tiles.
#pragma once
#include "common.hpp"
#include "../../include/bndm_tokens.h"

namespace bndm {

void tokens_error(const char *fmt, ...);

#define TOKENS_REQUIRE(cond, ...)                                                         \
    do {                                                                                  \
        if (!(cond)) {                                                                    \
            ::bndm::tokens_error(__VA_ARGS__);                                            \
            return BNDM_E_ARG;                                                            \
        }                                                                                 \
    } while (0)

static inline int tokens_launch_status(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        tokens_error("launch of %s failed: %s", what, hipGetErrorString(e));
        return (int)e;
    }
    return 0;
}

static inline int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

typedef _Float16 f16;
typedef __bf16 bf16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Vec;
template <> struct Vec<f16> {
    typedef f16 x8 __attribute__((ext_vector_type(8)));
    typedef f16 x4 __attribute__((ext_vector_type(4)));
};
template <> struct Vec<bf16> {
    typedef bf16 x8 __attribute__((ext_vector_type(8)));
    typedef bf16 x4 __attribute__((ext_vector_type(4)));
};

// D[32 x 32] += A[32 x 16] B[16 x 32].  Lane l holds row l % 32 of A and column l % 32 of B, k = 8 (l / 32) .. + 7, and of D column
// l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4 in register r.  The order of k is free as long as A and B agree.
template <typename T> __device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma32<f16>(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Vec<f16>::x8, a), __builtin_bit_cast(Vec<f16>::x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<bf16>(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Vec<bf16>::x8, a), __builtin_bit_cast(Vec<bf16>::x8, b), c, 0, 0, 0);
}

// D[16 x 16] += A[16 x 32] B[32 x 16].  Lane l: row l % 16 of A, column l % 16 of B, k = 8 (l / 16) .. + 7; of D column l % 16,
// rows 4 (l / 16) + r.
template <typename T> __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<f16>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Vec<f16>::x8, a), __builtin_bit_cast(Vec<f16>::x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<bf16>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Vec<bf16>::x8, a), __builtin_bit_cast(Vec<bf16>::x8, b), c, 0, 0, 0);
}

// Transposing LDS read: the 16 lanes of a group give the addresses of 16 pieces of 4 elements, lanes 4 j .. 4 j + 3 those of row j;
// lane i of the group receives column i of the four rows.
__device__ __forceinline__ s16x4 lds_read_tr(const void *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds_ptr_t)(p));
}

__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

template <typename T> __device__ __forceinline__ s16x8 pack8(float a, float b, float c, float d, float e, float f, float g, float h) {
    const typename Vec<T>::x8 v = {(T)a, (T)b, (T)c, (T)d, (T)e, (T)f, (T)g, (T)h};
    return __builtin_bit_cast(s16x8, v);
}
template <typename T> __device__ __forceinline__ s16x4 pack4(float a, float b, float c, float d) {
    const typename Vec<T>::x4 v = {(T)a, (T)b, (T)c, (T)d};
    return __builtin_bit_cast(s16x4, v);
}
template <typename T> __device__ __forceinline__ float widen(short s) { return (float)__builtin_bit_cast(T, s); }

// The 16-byte chunk in which chunk c of row `row` lies, for LDS tiles with rows of C chunks (C = 4, 8, 16, 32) that are read both as
// rows (32 consecutive rows at one c: ds_read_b128) and transposed (4 consecutive rows, 4 consecutive chunks: ds_read_b64_tr_b16).
// 16 / C rows fill the 64 banks once; of 16 such rows at one c no two share a bank, nor do the 4 x 4 chunks of a transposing read.
template <int C> __device__ __forceinline__ int swizzle(int row) {
    if constexpr (C == 4) return (row >> 2) & 3;
    else if constexpr (C == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return ((row & 3) << 2) | ((row >> 2) & 3);
}

// The same for tiles that are only read transposed: rows 8 apart are then a constant apart.
template <int C> __device__ __forceinline__ int swizzle_columns(int row) {
    static_assert(C >= 8, "four rows of 64 bytes need none");
    if constexpr (C == 8) return (row & 2) << 1;
    else return (row & 3) << 2;
}

// offset past every descriptor's range: the load returns zeros
constexpr uint32_t kNowhere = 0x80000000u;
constexpr int kAnywhere = 0x7ffffff0;

// the wave's copies into LDS have landed, and its reads of the tile before have been answered
__device__ __forceinline__ void wait_lds_dma() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

}  // namespace bndm
