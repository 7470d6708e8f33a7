// Quantised caches (PALU_LAYOUT_MX8 and MX4 with their V orders): 32 neighbouring channels of a position share one scale, a
// power of two kept as its 8-bit exponent (value 2^(byte - 127), 255: the block is NaN), and are held as fp8 (e4m3: 448 at
// most, steps of 1/8 of a power of two, 2^-9 below 2^-6) or fp4 (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6). What is held is exact in
// bf16: an element times its scale has 4 significant bits and stays within bf16's normal range.
//
// The scale of a block is the smallest power of two, from 2^-117 on, over which its largest value is at most 464 (7): it then
// is within half a step of 448 (6) and no element is further than that from what it is held as. 2^-117 is where every held
// value but 0 is a normal number; smaller blocks keep the absolute error of that scale (2^-127 in fp8, 2^-119 in fp4).
// Magnitudes past 1.75 2^127 are taken as that, so that what is read back is finite.
//
// A 32-position block of a cache w wide: its elements in the order that the attention's products take them, then the scales.
//   K order, position 8 t + 4 c + i (t < 4, c < 2, i < 4), n = 4 t + i:
//     fp8: [c][h][g][n] pieces of 16 bytes, channels 32 g + 16 h + 0 .. 15;   fp4: [c][g][n] pieces of 16, channels 32 g + 0 .. 31
//     scales [g][n][c]
//   V order, position 8 o + j (o < 4, j < 8):
//     fp8: [b][o][m][j] pairs of bytes, channels 32 b + 2 m and 2 m + 1;      fp4: [b][o][m][j] bytes of the same two
//     scales [b][position]
// In fp4 the lower channel is the lower half of a byte.
#pragma once
#include "palu_kernel.h"

namespace palu {

// An MX layout of the C-ABI: fp8 or fp4, K order or V order.
constexpr bool is_mx(int layout) { return layout >= PALU_LAYOUT_MX8 && layout <= PALU_LAYOUT_MX4_V; }
constexpr bool mx_fp8(int layout) { return layout == PALU_LAYOUT_MX8 || layout == PALU_LAYOUT_MX8_V; }
constexpr bool mx_k(int layout) { return layout == PALU_LAYOUT_MX8 || layout == PALU_LAYOUT_MX4; }

constexpr int mx_codes(bool fp8, int width) { return (fp8 ? 32 : 16) * width; }      // bytes of a block's elements
constexpr int mx_block(bool fp8, int width) { return (fp8 ? 33 : 17) * width; }      // and with its scales

// Ops over them, defined in palu_mx_cache.hip and palu_step_mx.hip.
int mx_append(void* cache, const void* rows, long long sb, long long sg, const int32_t* idx, const int32_t* page_table,
              int pt_stride, int n_pages, int batch, int n_groups, int seq_len, int width, int layout, const char* who,
              hipStream_t stream);
int mx_fill(void* pages, const void* rows, long long st, long long sg, const int32_t* cu, const int32_t* start,
            const int32_t* page_table, int n_rows, int batch, int n_groups, int n_pages, int page_shift, int pt_stride, int width,
            int layout, const char* who, hipStream_t stream);
int mx_flash_decode(const void* q, const void* k, const void* v, const int32_t* cur_pos, void* out, float scale, int batch,
                    int n_q, int n_kv, int positions, const int32_t* page_table, int pt_stride, int n_pages, int page_shift,
                    int head_dim_v, int out_dtype, int layout, void* workspace, size_t workspace_bytes, const char* who,
                    hipStream_t stream);

}  // namespace palu

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// The scale as the conversions take it. (byte 0, memory never written: 2^-127; 255: NaN)
__device__ __forceinline__ float mx_scale(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }
// Of byte j of a word (j a constant after unrolling): the conversions look at the exponent alone, so that the other bytes may be
// where sign and mantissa are.
__device__ __forceinline__ float mx_scale(unsigned word, int j) {
  return __builtin_bit_cast(float, j < 3 ? word << (23 - 8 * j) : word >> 1);
}

// Elements 2 p and 2 p + 1 of a word of codes as a pair of bf16 (p < 2 in fp8, < 4 in fp4; a constant after unrolling).
template <bool FP8>
__device__ __forceinline__ unsigned mx_pair(unsigned word, int p, float scale) {
  bf16x2 r;
  if constexpr (FP8) {
    r = p ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true)
          : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false);
  } else {
    r = p == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0)
        : p == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1)
        : p == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2)
                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
  }
  return __builtin_bit_cast(unsigned, r);
}

// The low (hi: high) halves of two words: lower half from x, upper from y.
__device__ __forceinline__ unsigned halves(unsigned x, unsigned y, bool hi) {
  return hi ? __builtin_amdgcn_perm(y, x, 0x07060302u) : __builtin_amdgcn_perm(y, x, 0x05040100u);
}

}  // namespace
