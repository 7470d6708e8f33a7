// Rows into quantised caches (palu_mx.h) and rows of any paged cache back out: palu_latent_append and its paged form,
// palu_latent_fill_paged in the MX layouts, palu_latent_read_paged in all.
#include "palu_mx.h"
#include "palu_packed.h"

#include <algorithm>

namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned max_halves(unsigned x, unsigned y) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
}
// Largest magnitudes of eight bf16 values, as their bits (which sort like the values, infinity and NaN above all numbers): of
// the even ones in the lower half, of the odd ones in the upper.
__device__ __forceinline__ unsigned top_halves(const bf16x8& x) {
  const u32x4 u = __builtin_bit_cast(u32x4, x) & 0x7fff7fffu;
  return max_halves(max_halves(u[0], u[1]), max_halves(u[2], u[3]));
}
// The same of two rows, over the four lanes that hold a block's 32 channels (lanes 4 k .. + 3, all active): row a's largest in
// the lower half, row b's in the upper.
__device__ __forceinline__ unsigned quad_tops(const bf16x8& a, const bf16x8& b) {
  const unsigned ta = top_halves(a), tb = top_halves(b);
  unsigned x = max_halves(halves(ta, tb, false), halves(ta, tb, true));
  x = max_halves(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));
  return max_halves(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));
}

constexpr unsigned INF_BITS = 0x7f80, MOST_BITS = 0x7f60;   // 1.75 2^127

// The scale byte of a block whose largest magnitude has these bits. Exact: 464 is 1.8125 2^8, 7 is 1.75 2^2.
template <bool FP8>
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
  if (top >= INF_BITS) return 255;
  top = min(top, MOST_BITS);
  const int e = (int)(top >> 7), m = (int)(top & 127);
  return (unsigned)max(FP8 ? e - 8 + (m > 104) : e - 2 + (m > 96), 10);
}

// Codes of eight values of a block whose largest magnitude is `top`: two words of fp8 or one of fp4. The conversion divides by the
// scale exactly and rounds once, to nearest even; fp4 stops at 6 by itself, fp8 would overflow past 464 scales, which only
// magnitudes past MOST_BITS are.
template <bool FP8>
struct Codes {
  unsigned w[FP8 ? 2 : 1];
};
template <bool FP8>
__device__ __forceinline__ Codes<FP8> encode8(bf16x8 x, unsigned top, unsigned byte) {
  u32x4 u = __builtin_bit_cast(u32x4, x);
  if (FP8 && top > MOST_BITS) {           // (rare)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = min(u[i] & 0x7fffu, MOST_BITS), hi = min(u[i] >> 16 & 0x7fffu, MOST_BITS);
      u[i] = (u[i] & 0x80008000u) | lo | hi << 16;
    }
  }
  const float scale = mx_scale(byte);
  Codes<FP8> c;
  auto pair = [&](int i) __attribute__((always_inline)) {
    const unsigned w = u[i];              // (an element of a vector is not cast as it stands)
    return __builtin_bit_cast(bf16x2, w);
  };
  if constexpr (FP8) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s16x2 w{0, 0};
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, pair(2 * i), scale, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, pair(2 * i + 1), scale, true);
      c.w[i] = __builtin_bit_cast(unsigned, w);
    }
  } else {
    unsigned w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, pair(0), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(1), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(2), scale, 2);
    c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(3), scale, 3);
  }
  if (byte == 255)                        // an infinity or NaN among the 32: all of them read back as NaN
#pragma unroll
    for (int i = 0; i < (FP8 ? 2 : 1); ++i) c.w[i] = 0;
  return c;
}
template <bool FP8>
__device__ __forceinline__ bf16x8 decode8(const Codes<FP8>& c, float scale) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = mx_pair<FP8>(c.w[FP8 ? i / 2 : 0], FP8 ? i & 1 : i, scale);
  return __builtin_bit_cast(bf16x8, r);
}

// Byte offsets inside a block: channels 8 v .. + 7 of position 8 o + j (K order: all of them; V order: channels 8 v and 8 v + 1,
// the next pair 8 positions' bytes further), and the scales of positions 8 o .. + 7 of channel block v / 4, eight bytes.
template <bool FP8>
__device__ __forceinline__ int k_codes(int o, int j, int v, int nb) {
  const int c = j >> 2, n = 4 * o + (j & 3), g = v >> 2;
  if constexpr (FP8) return ((c * 2 + ((v >> 1) & 1)) * nb + g) * 256 + n * 16 + (v & 1) * 8;
  else return (c * nb + g) * 256 + n * 16 + (v & 3) * 4;
}
template <bool FP8>
__device__ __forceinline__ int v_codes(int o, int v) { return (((v >> 2) * 4 + o) * 16 + 4 * (v & 3)) * (FP8 ? 16 : 8); }
__device__ __forceinline__ int scales_at(int codes, int o, int v) { return codes + (v >> 2) * 32 + 8 * o; }
// The scale of position 8 o + j in those eight bytes.
template <bool K>
__device__ __forceinline__ int scale_slot(int j) { return K ? 2 * (j & 3) + (j >> 2) : j; }

// ---- appends ------------------------------------------------------------------------------------
// cache[b][g][idx[b]] = rows[b][g]: a thread per eight channels. Single rows: latency.
struct AppendArgs {
  char* cache;
  const __bf16* rows;
  long long sb, sg;
  const int32_t* idx;
  const int32_t* table;                   // null: contiguous, row b's stream is "page" b
  int pt_stride, n_pages, B, G, S, width; // S: positions of a page (of a row)
};

template <bool FP8, bool K>
__global__ __launch_bounds__(256) void palu_mx_append_kernel(const AppendArgs a) {
  const int vec = a.width / 8, nb = a.width / 32;
  const long long total = (long long)a.B * a.G * vec;
  for (long long e = blockIdx.x * 256LL + threadIdx.x; e < total; e += gridDim.x * 256LL) {
    const int v = (int)(e % vec);
    const long long bg = e / vec;
    const int b = (int)(bg / a.G), g = (int)(bg - (long long)b * a.G);
    int p = a.idx[b];
    long long page = b;
    if (a.table) {
      if (p < 0 || p >= a.pt_stride * a.S) continue;       // (all four lanes of a block)
      page = a.table[(long long)b * a.pt_stride + p / a.S];
      if (page < 0 || page >= a.n_pages) continue;
      p %= a.S;
    } else if (p < 0 || p >= a.S) {
      continue;
    }
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(a.rows + b * a.sb + g * a.sg + 8 * v);
    const unsigned top = quad_tops(x, x) & 0xffffu, byte = scale_byte<FP8>(top);
    const Codes<FP8> c = encode8<FP8>(x, top, byte);
    const int o = (p >> 3) & 3, j = p & 7;
    char* blk = a.cache + ((page * a.G + g) * (a.S / 32) + (p >> 5)) * mx_block(FP8, a.width);
    if constexpr (K) {
      char* to = blk + k_codes<FP8>(o, j, v, nb);
      if constexpr (FP8) *reinterpret_cast<u32x2*>(to) = u32x2{c.w[0], c.w[1]};
      else *reinterpret_cast<unsigned*>(to) = c.w[0];
    } else {
      char* to = blk + v_codes<FP8>(o, v);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if constexpr (FP8) *reinterpret_cast<unsigned short*>(to + u * 16 + 2 * j) = (unsigned short)(c.w[u / 2] >> (16 * (u & 1)));
        else to[u * 8 + j] = (char)(c.w[0] >> (8 * u));
    }
    if ((v & 3) == 0) blk[scales_at(mx_codes(FP8, a.width), o, v) + scale_slot<K>(j)] = (char)byte;
  }
}

// ---- packed rows in and out ---------------------------------------------------------------------
// A workgroup takes one 32-position block of one sequence and a few groups, a thread eight positions of eight channels: their
// rows are whole 16-byte loads, and in V order its codes are whole pieces as well. Bound by memory: each row is read once and not
// kept in the caches, neither is what the read below writes (16 sequences of up to 4096 rows of 8 x 128 into fp4 and back,
// 78 MB: 23.4 -> 21.6 us; 13.9 and 9.5 us kept there).
struct MxFillArgs {
  PackedSeqs seqs;
  char* cache;
  const __bf16* rows;
  long long st, sg;
  int G, width, gpw;
};

template <bool FP8, bool K>
__global__ __launch_bounds__(256) void palu_mx_fill_kernel(const MxFillArgs a) {
  const PackedBlock p = packed_block(a.seqs, (int)blockIdx.x);
  if (p.b < 0 || p.pid < 0 || p.pid >= a.seqs.n_pages) return;   // as the append: ids outside the pool are skipped
  const int vec = a.width / 8, nb = a.width / 32, g0 = blockIdx.y * a.gpw, g1 = min(a.G, g0 + a.gpw);
  const int bpp = 1 << a.seqs.page_shift, codes = mx_codes(FP8, a.width);
  const __bf16* src = a.rows + (long long)p.row0 * a.st;
  for (int e = threadIdx.x; e < (g1 - g0) * 4 * vec; e += 256) {
    const int v = e % vec, o = e / vec & 3, g = g0 + e / (4 * vec), p0 = 32 * p.blk + 8 * o;
    if (p0 >= p.hi || p0 + 8 <= p.lo) continue;                  // (all four lanes of a block)
    Codes<FP8> c[8];
    unsigned byte[8];
    bf16x8 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __bf16* row = src + (long long)min(max(p0 + j, p.lo), p.hi - 1) * a.st + g * a.sg;
      x[j] = __builtin_nontemporal_load(reinterpret_cast<const bf16x8*>(row + 8 * v));
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const unsigned tops = quad_tops(x[j], x[j + 1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned top = i ? tops >> 16 : tops & 0xffffu;
        byte[j + i] = scale_byte<FP8>(top);
        c[j + i] = encode8<FP8>(x[j + i], top, byte[j + i]);
      }
    }
    char* blk = a.cache + (((long long)p.pid * a.G + g) * bpp + (p.blk & (bpp - 1))) * mx_block(FP8, a.width);
    const bool whole = p0 >= p.lo && p0 + 8 <= p.hi;
    auto inside = [&](int j) { return p0 + j >= p.lo && p0 + j < p.hi; };
    if constexpr (K) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!inside(j)) continue;
        char* to = blk + k_codes<FP8>(o, j, v, nb);
        if constexpr (FP8) *reinterpret_cast<u32x2*>(to) = u32x2{c[j].w[0], c[j].w[1]};
        else *reinterpret_cast<unsigned*>(to) = c[j].w[0];
      }
    } else {
      char* to = blk + v_codes<FP8>(o, v);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (whole) {
          if constexpr (FP8) {
            u32x4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = halves(c[2 * i].w[u / 2], c[2 * i + 1].w[u / 2], u & 1);
            *reinterpret_cast<u32x4*>(to + u * 16) = y;
          } else {
            u32x2 y;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              y[i] = 0;
#pragma unroll
              for (int j = 0; j < 4; ++j) y[i] |= ((c[4 * i + j].w[0] >> (8 * u)) & 255u) << (8 * j);
            }
            *reinterpret_cast<u32x2*>(to + u * 8) = y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (inside(j)) {
              if constexpr (FP8) *reinterpret_cast<unsigned short*>(to + u * 16 + 2 * j) = (unsigned short)(c[j].w[u / 2] >> (16 * (u & 1)));
              else to[u * 8 + j] = (char)(c[j].w[0] >> (8 * u));
            }
        }
      }
    }
    if ((v & 3) == 0) {
      char* to = blk + scales_at(codes, o, v);
      if (whole) {
        u32x2 y{0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) y[scale_slot<K>(j) / 4] |= byte[j] << (8 * (scale_slot<K>(j) & 3));
        *reinterpret_cast<u32x2*>(to) = y;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (inside(j)) to[scale_slot<K>(j)] = (char)byte[j];
      }
    }
  }
}

// Rows of the pages, out [T][G][width]: the fill the other way. Positions outside the table and pages outside the pool give
// zeros; packed rows of no sequence are left alone.
struct ReadArgs {
  PackedSeqs seqs;
  const char* cache;
  __bf16* out;
  int G, width, gpw;
};

template <int LAYOUT>
__global__ __launch_bounds__(256) void palu_read_pages_kernel(const ReadArgs a) {
  const PackedBlock p = packed_block<true>(a.seqs, (int)blockIdx.x);
  if (p.b < 0) return;
  const bool there = p.pid >= 0 && p.pid < a.seqs.n_pages;
  const int vec = a.width / 8, g0 = blockIdx.y * a.gpw, g1 = min(a.G, g0 + a.gpw), bpp = 1 << a.seqs.page_shift;
  for (int e = threadIdx.x; e < (g1 - g0) * 4 * vec; e += 256) {
    const int v = e % vec, o = e / vec & 3, g = g0 + e / (4 * vec), p0 = 32 * p.blk + 8 * o;
    if (p0 >= p.hi || p0 + 8 <= p.lo) continue;
    const long long block = ((long long)p.pid * a.G + g) * bpp + (p.blk & (bpp - 1));
    bf16x8 x[8];
    if (!there) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = bf16x8{};
    } else if constexpr (is_mx(LAYOUT)) {
      constexpr bool FP8 = mx_fp8(LAYOUT), K = mx_k(LAYOUT);
      const char* blk = a.cache + block * mx_block(FP8, a.width);
      const u32x2 s = *reinterpret_cast<const u32x2*>(blk + scales_at(mx_codes(FP8, a.width), o, v));
      Codes<FP8> c[8];
      if constexpr (K) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const char* from = blk + k_codes<FP8>(o, j, v, a.width / 32);
          if constexpr (FP8) {
            const u32x2 y = *reinterpret_cast<const u32x2*>(from);
            c[j].w[0] = y[0];
            c[j].w[1] = y[1];
          } else {
            c[j].w[0] = *reinterpret_cast<const unsigned*>(from);
          }
        }
      } else {
        const char* from = blk + v_codes<FP8>(o, v);
        if constexpr (FP8) {
          u32x4 y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) y[u] = *reinterpret_cast<const u32x4*>(from + u * 16);
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) c[j].w[i] = halves(y[2 * i][j / 2], y[2 * i + 1][j / 2], j & 1);
        } else {
          u32x2 y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) y[u] = *reinterpret_cast<const u32x2*>(from + u * 8);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            c[j].w[0] = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) c[j].w[0] |= ((y[u][j / 4] >> (8 * (j & 3))) & 255u) << (8 * u);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = decode8<FP8>(c[j], mx_scale(s[scale_slot<K>(j) / 4], scale_slot<K>(j) & 3));
    } else {
      const __bf16* blk = reinterpret_cast<const __bf16*>(a.cache) + block * 32 * a.width;
      if constexpr (LAYOUT == PALU_LAYOUT_TILED_V) {
        bf16x8 y[8];
        const __bf16* from = blk + tiled_v_offset(8 * o, 8 * v, a.width);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = *reinterpret_cast<const bf16x8*>(from + 8 * i);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j][i] = y[i][j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (LAYOUT == PALU_LAYOUT_ROWS) {
            x[j] = *reinterpret_cast<const bf16x8*>(blk + (8 * o + j) * a.width + 8 * v);
          } else {
            const __bf16* from = blk + tiled_k_offset(8 * o + j, 8 * v, a.width);
            if ((v >> 2) < (a.width >> 5)) {
              x[j] = *reinterpret_cast<const bf16x8*>(from);
            } else {                      // the half tile of a width that is an odd multiple of 16
              const bf16x4 lo = *reinterpret_cast<const bf16x4*>(from), hi = *reinterpret_cast<const bf16x4*>(from + 64);
              x[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
          }
        }
      }
    }
    __bf16* out = a.out + ((long long)p.row0 * a.G + g) * a.width + 8 * v;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (p0 + j >= p.lo && p0 + j < p.hi)
        __builtin_nontemporal_store(x[j], reinterpret_cast<bf16x8*>(out + (long long)(p0 + j) * a.G * a.width));
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
}

int check_mx(int width, int page, const char* who) {
  if (width <= 0 || width % 32 || width > 512)
    return fail(PALU_EINVAL, "%s: a quantised cache's width is a multiple of 32 up to 512, got %d", who, width);
  if (page % 32) return fail(PALU_EINVAL, "%s: a quantised cache holds whole 32-position blocks, got %d positions", who, page);
  return PALU_OK;
}

// Groups per workgroup: 64 values a thread.
int groups_per_wg(int n_groups, int width) { return std::min(n_groups, std::max(1, 512 / width)); }

template <typename F>
void for_mx(int layout, F&& go) {
  switch (layout) {
    case PALU_LAYOUT_MX8: return go(std::integral_constant<int, PALU_LAYOUT_MX8>());
    case PALU_LAYOUT_MX8_V: return go(std::integral_constant<int, PALU_LAYOUT_MX8_V>());
    case PALU_LAYOUT_MX4: return go(std::integral_constant<int, PALU_LAYOUT_MX4>());
    default: return go(std::integral_constant<int, PALU_LAYOUT_MX4_V>());
  }
}

}  // namespace

namespace palu {

int mx_append(void* cache, const void* rows, long long sb, long long sg, const int32_t* idx, const int32_t* page_table,
              int pt_stride, int n_pages, int batch, int n_groups, int seq_len, int width, int layout, const char* who,
              hipStream_t stream) {
  if (!cache || !rows || !idx) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  if (batch <= 0 || n_groups <= 0 || seq_len <= 0)
    return fail(PALU_EINVAL, "%s: batch, group and position counts must be positive", who);
  if (int rc = check_mx(width, seq_len, who)) return rc;
  if (!al16(cache) || !al16(rows)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  const AppendArgs a{static_cast<char*>(cache), static_cast<const __bf16*>(rows), sb, sg, idx, page_table, pt_stride, n_pages,
                     batch, n_groups, seq_len, width};
  const long long total = (long long)batch * n_groups * (width / 8);
  const dim3 grid((unsigned)std::min<long long>((total + 255) / 256, 4096));
  for_mx(layout, [&](auto l) {
    hipLaunchKernelGGL((palu_mx_append_kernel<mx_fp8(l.value), mx_k(l.value)>), grid, dim3(256), 0, stream, a);
  });
  return launched(who);
}

int mx_fill(void* pages, const void* rows, long long st, long long sg, const int32_t* cu, const int32_t* start,
            const int32_t* page_table, int n_rows, int batch, int n_groups, int n_pages, int page_shift, int pt_stride, int width,
            int layout, const char* who, hipStream_t stream) {
  if (int rc = check_mx(width, 32, who)) return rc;
  MxFillArgs a{{cu, start, page_table, n_rows, batch, n_pages, page_shift, pt_stride}, static_cast<char*>(pages),
               static_cast<const __bf16*>(rows), st, sg, n_groups, width, groups_per_wg(n_groups, width)};
  const dim3 grid(packed_blocks(n_rows, batch), (unsigned)((n_groups + a.gpw - 1) / a.gpw));
  for_mx(layout, [&](auto l) {
    hipLaunchKernelGGL((palu_mx_fill_kernel<mx_fp8(l.value), mx_k(l.value)>), grid, dim3(256), 0, stream, a);
  });
  return launched(who);
}

}  // namespace palu

extern "C" int palu_latent_read_paged(const void* cache_pages, void* out, const int32_t* cu_seqlens, const int32_t* start_pos,
                                      const int32_t* page_table, int n_rows, int batch, int n_groups, int num_pages,
                                      int page_size, int max_pages_per_seq, int width, int cache_layout, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_latent_read_paged";
  if (!cache_pages || !out || !cu_seqlens) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  int shift = 0;
  if (int rc = palu::check_pages(page_table, num_pages, page_size, max_pages_per_seq, &shift, who)) return rc;
  if (n_rows <= 0 || batch <= 0 || n_groups <= 0)
    return fail(PALU_EINVAL, "%s: row, sequence and group counts must be positive, got %d, %d, %d", who, n_rows, batch, n_groups);
  const bool mx = is_mx(cache_layout);
  if (!mx && cache_layout != PALU_LAYOUT_ROWS && cache_layout != PALU_LAYOUT_TILED && cache_layout != PALU_LAYOUT_TILED_V)
    return fail(PALU_EINVAL, "%s: cache layout must be PALU_LAYOUT_ROWS, _TILED, _TILED_V or one of the MX layouts, got %d", who,
                cache_layout);
  const int step = mx ? 32 : cache_layout == PALU_LAYOUT_ROWS ? 8 : 16;
  if (width <= 0 || width % step || width > 512)
    return fail(PALU_EINVAL, "%s: width must be a multiple of %d up to 512, got %d", who, step, width);
  if (!al16(cache_pages) || !al16(out)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  if (n_rows > (1 << 28) || batch > 65535 || n_groups > 65535) return fail(PALU_EUNSUPPORTED, "%s: counts exceed the grid", who);
  const ReadArgs a{{cu_seqlens, start_pos, page_table, n_rows, batch, num_pages, shift, max_pages_per_seq},
                   static_cast<const char*>(cache_pages), static_cast<__bf16*>(out), n_groups, width,
                   groups_per_wg(n_groups, width)};
  const dim3 grid(packed_blocks(n_rows, batch), (unsigned)((n_groups + a.gpw - 1) / a.gpw));
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, a); };
  if (mx) for_mx(cache_layout, [&](auto l) { go(palu_read_pages_kernel<l.value>); });
  else if (cache_layout == PALU_LAYOUT_TILED) go(palu_read_pages_kernel<PALU_LAYOUT_TILED>);
  else if (cache_layout == PALU_LAYOUT_TILED_V) go(palu_read_pages_kernel<PALU_LAYOUT_TILED_V>);
  else go(palu_read_pages_kernel<PALU_LAYOUT_ROWS>);
  return launched(who);
}
