// One new token per row over cached full K and V: the decode attention of quantised caches (palu_flash_decode and its paged
// form in the MX layouts) and of batches whose rows share prefixes (palu_flash_decode_shared, all layouts),
//   out[b][h] = sum_{p <= cur[b]} softmax_p(scale q[b][h] . k[p][j]) v[p][j],   j = h / rep, rep = n_q / n_kv.
// Included by one translation unit per family of layouts.
//
// A wave takes whole 32-position blocks, straight from memory into registers, the next block's loads under way while it
// computes, and the four waves of a workgroup take every fourth block. Its columns are up to 16 C queries:
//   S^T (keys x columns) = K Q^T, two v_mfma_f32_16x16x32_bf16 tiles of 16 keys, Q the B operand, in registers;
//   P^T = 2^(S^T - m), the running maximum m refreshed when a score exceeds it by more than 2^8;
//   O^T (channels x columns) += V^T P^T.
// The rows of the K operand are the keys in the order of the caches' K tiles: the two accumulators then leave a lane with
// the eight keys 8 g .. + 7 of its column, which is the B operand of the second product, and no value changes lanes. Tiled
// and quantised caches hold both operands as they are taken, 8 bytes or more of a lane in one piece; a quantised value is
// turned into bf16 (exactly) between memory and product, a lane's 32 channels of a key under one scale, two channels of a position
// under one scale of V, which two byte permutations make pairs of positions. Row-major V is read in the same pairs.
//
// Rounding: products of bf16 are exact in fp32, scores, statistics and sums are fp32; the probabilities are rounded to bf16
// for the second product, by up to 2^-8 of each, and it is the rounded ones that are summed to divide by.
#pragma once
#include "palu_mx.h"

#include <algorithm>

namespace palu {

// What a row has of a prefix: its blocks 0 .. blocks - 1 are read through row `lead`'s table; where pieces > 0 they have been
// read, and the row's queries are columns local * rep .. of the group's, in slots base + (tile * n_kv + kv) * pieces ..
struct RowPrefix {
  int lead, blocks, pieces, base, local, unused[3];
};

struct StepArgs {
  const __bf16* q;                        // [B][n_q][128]
  const char* k;
  const char* v;
  long long k_page, v_page, k_head, v_head;   // bytes: from a page (a row) to the next, from a head to the next
  int k_blk, v_blk;                       // bytes of a block
  const int32_t* cur;                     // [B] last position seen
  const int32_t* table;                   // [B][pt_stride], or null: "page" b is row b's stream
  int pt_stride, n_pages, page_shift, capacity;
  int B, n_q, n_kv, rep, dv;
  float qscale;                           // scale * log2 e
  void* out;                              // [B][n_q][dv]
  int f32_out;
  // Split items: partial results of 16 columns, [16][dv] O, m [16], l [16], and their done flags.
  float* part;
  unsigned long long* flags;
  unsigned long long epoch;
  // Shared prefixes (rows null: none).
  const int32_t* cu;                      // [n_groups + 1] first row of every group; null: one group
  const int32_t* shared;                  // [n_groups] positions shared
  int n_groups;
  RowPrefix* rows;                        // [B]
  float* pre;                             // pieces of the prefixes: [16 C][dv] O, m [16 C], l [16 C]
  int pre_slots, pre_cols;                // slots, 16 C
};

int step_bf16(const StepArgs& a, int layout, const char* who, hipStream_t s);   // defined in palu_step_bf16.hip

}  // namespace palu

namespace {

// ---- blocks --------------------------------------------------------------------------------------
// The registers of a block as it is loaded: K, V of NB blocks of 32 channels.
template <int L, int NB>
struct Raw {
  static constexpr bool MX = is_mx(L), FP8 = mx_fp8(L);
  u32x4 k[MX ? (FP8 ? 4 : 2) : 8];
  unsigned ks;                            // scales of half-blocks 0 and 1
  u32x4 v[MX ? (FP8 ? NB : (NB + 1) / 2) : 2 * NB];
  u32x2 vs[MX ? NB : 1];
};

// lane = 16 g + n
template <int L, int NB>
__device__ __forceinline__ void load_block(Raw<L, NB>& r, const char* k, const char* v, int dv) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  if constexpr (Raw<L, NB>::MX) {
    constexpr bool FP8 = Raw<L, NB>::FP8;
#pragma unroll
    for (int i = 0; i < (FP8 ? 4 : 2); ++i) r.k[i] = *reinterpret_cast<const u32x4*>(k + i * 1024 + lane * 16);
    r.ks = *reinterpret_cast<const unsigned short*>(k + mx_codes(FP8, HD) + 2 * lane);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (FP8) {
        r.v[b] = *reinterpret_cast<const u32x4*>(v + b * 1024 + lane * 16);
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(v + b * 512 + lane * 8);
        r.v[b / 2][2 * (b & 1)] = x[0];
        r.v[b / 2][2 * (b & 1) + 1] = x[1];
      }
      r.vs[b] = *reinterpret_cast<const u32x2*>(v + mx_codes(FP8, 32 * NB) + b * 32 + 8 * g);
    }
  } else if constexpr (L == PALU_LAYOUT_TILED) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.k[i] = *reinterpret_cast<const u32x4*>(k + i * 1024 + lane * 16);
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)      // (of a width that is an odd multiple of 16 the last tile twice)
      r.v[i] = *reinterpret_cast<const u32x4*>(v + min(i, dv / 16 - 1) * 1024 + lane * 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)           // key (c, n), channels 32 s + 8 g .. + 7
      r.k[i] = *reinterpret_cast<const u32x4*>(k + (8 * (n >> 2) + 4 * (i >> 2) + (n & 3)) * (2 * HD) + (i & 3) * 64 + g * 16);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 8; ++j)         // position 8 g + j, channels 32 b + 2 n and 2 n + 1
        r.v[2 * b + j / 4][j & 3] = *reinterpret_cast<const unsigned*>(v + (8 * g + j) * (2 * dv) + min(64 * b + 4 * n, 2 * dv - 4));
  }
}

// Channel of element j of product step s in lane group g's Q and K operands.
template <int L>
__device__ __forceinline__ int q_chan(int s, int g) { return is_mx(L) ? 32 * g + 8 * s : 32 * s + 8 * g; }

// K operand of half-block c and step s.
template <int L, int NB>
__device__ __forceinline__ bf16x8 k_operand(const Raw<L, NB>& r, int c, int s) {
  if constexpr (!is_mx(L)) {
    return __builtin_bit_cast(bf16x8, r.k[4 * c + s]);
  } else {
    const float scale = mx_scale(r.ks, c);
    u32x4 y;
    if constexpr (mx_fp8(L)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = mx_pair<true>(r.k[2 * c + (s >> 1)][2 * (s & 1) + (i >> 1)], i & 1, scale);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = mx_pair<false>(r.k[c][s], i, scale);
    }
    return __builtin_bit_cast(bf16x8, y);
  }
}

// The V^T operands of channel block b: row n of tile t is channel 32 b + 16 t + n of tiled caches, else 32 b + 2 n + t.
template <int L, int NB>
__device__ __forceinline__ void v_operands(const Raw<L, NB>& r, int b, u32x4 (&y)[2]) {
  if constexpr (L == PALU_LAYOUT_TILED) {
    y[0] = r.v[2 * b];
    y[1] = r.v[2 * b + 1];
  } else {
    unsigned u[8];                        // channels 32 b + 2 n and 2 n + 1 of position 8 g + j
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (L == PALU_LAYOUT_ROWS) {
        u[j] = r.v[2 * b + j / 4][j & 3];
      } else {
        const float scale = mx_scale(r.vs[b][j / 4], j & 3);
        if constexpr (mx_fp8(L)) u[j] = mx_pair<true>(r.v[b][j / 2], j & 1, scale);
        else u[j] = mx_pair<false>(r.v[b / 2][2 * (b & 1) + j / 4], j & 3, scale);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[0][i] = halves(u[2 * i], u[2 * i + 1], false);
      y[1][i] = halves(u[2 * i], u[2 * i + 1], true);
    }
  }
}

// ---- a wave's pass over blocks ------------------------------------------------------------------
// State of 16 C columns; lane 16 g + n has column n of every 16.
template <int L, int NB, int C>
struct Wave {
  bf16x8 q[C][4];
  f32x4 o[C][2 * NB];
  float m[C], l[C];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int x = 0; x < C; ++x) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) o[x][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[x] = NEG_INF;
      l[x] = 0.f;
    }
  }

  // The block's positions 0 .. seen - 1 (MASK: the rest may hold anything).
  template <bool MASK>
  __device__ __forceinline__ void add(const Raw<L, NB>& r, float qscale, int seen) {
    const int g = (threadIdx.x & 63) >> 4;
    f32x4 s[C][2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 k = k_operand<L, NB>(r, c, i);
#pragma unroll
        for (int x = 0; x < C; ++x) s[x][c] = mfma16(k, q[x][i], i == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[x][c]);
      }
    bf16x8 p[C];
#pragma unroll
    for (int x = 0; x < C; ++x) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[x][c][i] *= qscale;
          if (MASK && 8 * g + 4 * c + i >= seen) s[x][c][i] = NEG_INF;
        }
      const float top = max8(s[x][0], s[x][1]);
      if (__any(top > m[x] + LAZY_RESCALE_LOG2)) {
        const float all = wave_max_xor48(top), mn = all > m[x] + LAZY_RESCALE_LOG2 ? all : m[x];
        const float alpha = m[x] == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(m[x] - mn);
        if (__any(m[x] != NEG_INF)) {     // (not at the first block)
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) o[x][i] *= alpha;
          l[x] *= alpha;
        }
        m[x] = mn;
      }
      const float ref = m[x] == NEG_INF ? 0.f : m[x];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[x][j] = (__bf16)__builtin_amdgcn_exp2f(s[x][j >> 2][j & 3] - ref);
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        l[x] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[x][j], p[x][j + 1]}, bf16x2{(__bf16)1.f, (__bf16)1.f}, l[x], false);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      u32x4 y[2];
      v_operands<L, NB>(r, b, y);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (MASK)                         // 0 times what an unseen position holds may be NaN
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[t][i] &= (8 * g + 2 * i < seen ? 0xffffu : 0u) | (8 * g + 2 * i + 1 < seen ? 0xffff0000u : 0u);
#pragma unroll
        for (int x = 0; x < C; ++x) o[x][2 * b + t] = mfma16(__builtin_bit_cast(bf16x8, y[t]), p[x], o[x][2 * b + t]);
      }
    }
  }

  // Blocks first, first + step, .. below end of a sequence that is seen up to position seen - 1; where(blk, k, v) gives a
  // block's places.
  template <typename F>
  __device__ __forceinline__ void pass(int first, int end, int step, int seen, float qscale, int dv, F&& where) {
    if (first >= end) return;
    const int last = first + (end - 1 - first) / step * step;
    Raw<L, NB> a, b;
    const char *k, *v;
    auto load = [&](Raw<L, NB>& r, int blk) __attribute__((always_inline)) {
      where(min(blk, last), k, v);
      load_block<L, NB>(r, k, v, dv);
    };
    auto use = [&](const Raw<L, NB>& r, int blk) __attribute__((always_inline)) {
      if (32 * blk + 32 <= seen) add<false>(r, qscale, 32);
      else if (32 * blk < seen) add<true>(r, qscale, seen - 32 * blk);
    };
    load(a, first);
    for (int blk = first;; blk += 2 * step) {
      load(b, blk + step);
      use(a, blk);
      if (blk + step > last) break;
      load(a, blk + 2 * step);
      use(b, blk + step);
      if (blk + 2 * step > last) break;
    }
  }
};

// Column tile x of every wave's state to LDS, [wave][16][OS] O and [wave][16] m, l; barriers around it are the caller's.
template <int NB>
struct WaveLds {
  static constexpr int OS = 32 * NB + 4;
  float o[4][16][OS], m[4][16], l[4][16];
};
template <int L, int NB, int C>
__device__ __forceinline__ void to_lds(WaveLds<NB>& s, const Wave<L, NB, C>& st, int x) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, w = threadIdx.x >> 6;
  const float l = wave_sum_xor48(st.l[x]);
  if (g == 0) {
    s.m[w][n] = st.m[x];
    s.l[w][n] = l;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const f32x4 y = st.o[x][2 * b], z = st.o[x][2 * b + 1];    // rows 4 g .. + 3 of tiles 0 and 1
    if constexpr (L == PALU_LAYOUT_TILED) {
      *reinterpret_cast<f32x4*>(&s.o[w][n][32 * b + 4 * g]) = y;
      *reinterpret_cast<f32x4*>(&s.o[w][n][32 * b + 16 + 4 * g]) = z;
    } else {
      *reinterpret_cast<f32x4*>(&s.o[w][n][32 * b + 8 * g]) = f32x4{y[0], z[0], y[1], z[1]};
      *reinterpret_cast<f32x4*>(&s.o[w][n][32 * b + 8 * g + 4]) = f32x4{y[2], z[2], y[3], z[3]};
    }
  }
}

// Four channels of a column, summed from parts: y and l stand over 2^m.
struct Joined {
  f32x4 y{0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, l = 0.f;
  __device__ __forceinline__ void add(f32x4 py, float pm, float pl) {
    const float mn = fmaxf(m, pm);
    const float ref = mn == NEG_INF ? 0.f : mn;               // (then both have nothing, or NaN)
    const float wa = __builtin_amdgcn_exp2f(m - ref), wb = __builtin_amdgcn_exp2f(pm - ref);
    y = y * wa + py * wb;
    l = l * wa + pl * wb;
    m = mn;
  }
};
template <int NB>
__device__ __forceinline__ Joined join_waves(const WaveLds<NB>& s, int n, int d) {
  Joined j;
#pragma unroll
  for (int w = 0; w < 4; ++w) j.add(*reinterpret_cast<const f32x4*>(&s.o[w][n][d]), s.m[w][n], s.l[w][n]);
  return j;
}

// Exclusive prefix sum of x over the workgroup's 256 threads, and its total. `part`: 4 ints.
__device__ __forceinline__ int wg_scan(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, s = wave_scan(x);
  __syncthreads();
  if (lane == 63) part[w] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    before += i < w ? part[i] : 0;
    total += part[i];
  }
  return before + s - x;
}

__device__ __forceinline__ int seen_of(const StepArgs& a, int pos) { return min(max(pos, -1), a.capacity - 1) + 1; }

// Places of block blk of a row's KV head.
__device__ __forceinline__ void place_of(const StepArgs& a, int row, int kvh, int blk, const char*& k, const char*& v) {
  long long page = row;
  if (a.table) page = min(max(load_uniform(a.table, (long long)row * a.pt_stride + (blk >> a.page_shift)), 0), a.n_pages - 1);
  const int at = a.table ? blk & ((1 << a.page_shift) - 1) : blk;
  k = a.k + page * a.k_page + kvh * a.k_head + (long long)at * a.k_blk;
  v = a.v + page * a.v_page + kvh * a.v_head + (long long)at * a.v_blk;
}

// ---- the rows' own blocks -----------------------------------------------------------------------
// An item is a row's KV head: its blocks, but for those that have been read with the group's prefix. All items' blocks lie one
// after another, row by row, KV head by KV head. Where a workgroup's share of them (of STEP_WGS) is at least STEP_LEAST blocks
// each takes such a share, from wherever it begins to wherever it ends; below that an item is cut into even pieces of up
// to STEP_LEAST blocks, a workgroup each. An item in several workgroups is joined by the one that finds all parts done.
constexpr int STEP_WGS = 512;             // workgroups that the chip holds at once (two a CU)
constexpr int STEP_LEAST = 16;            // blocks

inline int step_grid(int B, int n_kv) { return STEP_WGS + B * n_kv; }          // pieces of STEP_LEAST, at most
inline int step_slots(int B, int n_kv) { return std::max(2 * STEP_WGS, step_grid(B, n_kv)); }
inline size_t step_bytes(int B, int n_kv, int rep, int dv) {
  return (size_t)step_slots(B, n_kv) * ((size_t)rep * (dv + 2) * sizeof(float) + sizeof(unsigned long long));
}

struct RowWork {
  int lead, first, end, seen, pieces;     // blocks first .. end - 1 (at least one, which may hold nothing), prefix pieces
  int base, local, pblocks;
};
__device__ __forceinline__ RowWork row_work(const StepArgs& a, int b) {
  const int seen = seen_of(a, a.cur[b]), end = (seen + 31) >> 5;
  RowWork r{b, 0, max(end, 1), seen, 0, 0, 0, 0};
  if (a.rows) {
    const RowPrefix p = a.rows[b];
    r.lead = p.lead;
    r.pblocks = p.blocks;
    if (p.pieces && seen >= 32 * p.blocks) {
      r.first = p.blocks;
      r.end = max(end, p.blocks + 1);
      r.pieces = p.pieces;
      r.base = p.base;
      r.local = p.local;
    }
  }
  return r;
}

__device__ __forceinline__ void store4(const StepArgs& a, long long at, f32x4 y) {
  if (a.f32_out) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = y;
  } else {
    bf16x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (__bf16)y[i];
    *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(a.out) + at) = x;
  }
}

template <int L, int NB>
__global__ __launch_bounds__(256, 2) void palu_step_kernel(const StepArgs a) {
  __shared__ WaveLds<NB> lds;
  __shared__ int scan[4], found[4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wg = blockIdx.x;
  const int per = (a.B + 255) / 256, r0 = min(tid * per, a.B), r1 = min(r0 + per, a.B);
  // this workgroup's part of the batch
  int mine = 0, total, pieces;
  for (int b = r0; b < r1; ++b) {
    const RowWork r = row_work(a, b);
    mine += r.end - r.first;
  }
  int before = wg_scan(mine, scan, total);
  total *= a.n_kv;
  const int share = (total + STEP_WGS - 1) / STEP_WGS;
  const bool cut = share < STEP_LEAST;    // items in pieces, not shares
  auto pieces_of = [](const RowWork& r) { return (r.end - r.first + STEP_LEAST - 1) / STEP_LEAST; };
  if (cut) {
    mine = 0;
    for (int b = r0; b < r1; ++b) mine += pieces_of(row_work(a, b));
    before = wg_scan(mine, scan, pieces);
  }
  if (!cut && wg >= STEP_WGS) return;     // uniform
  const int want = cut ? wg : wg * share;
  if (want >= (cut ? pieces * a.n_kv : total)) return;
  if (want >= before * a.n_kv && want < (before + mine) * a.n_kv) {
    int at = before * a.n_kv, b = r0;
    for (; b < r1; ++b) {
      const RowWork r = row_work(a, b);
      const int n = (cut ? pieces_of(r) : r.end - r.first) * a.n_kv;
      if (want < at + n) break;
      at += n;
    }
    found[0] = b;
    found[1] = at;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane(found[0]), at = __builtin_amdgcn_readfirstlane(found[1]);
  const int stop = cut ? want + 1 : min(total, want + share);
  const int n16 = lane & 15, g = lane >> 4;

  for (int here = want; here < stop;) {   // uniform
    RowWork r = row_work(a, b);
    const int unit = cut ? pieces_of(r) : r.end - r.first;  // of an item, in what `here` counts
    const int kvh = (here - at) / unit, in = here - at - kvh * unit;
    const int item = at + kvh * unit;                       // its first
    int lo, hi, chunk, chunks, wg0;
    if (cut) {
      const int len = (r.end - r.first + unit - 1) / unit;
      lo = r.first + in * len;
      hi = min(r.end, lo + len);
      chunk = in;
      chunks = unit;
      wg0 = item;
      here += 1;
    } else {
      const int n = min(unit - in, stop - here);
      lo = r.first + in;
      hi = lo + n;
      wg0 = item / share;
      chunk = wg - wg0;
      chunks = (item + unit - 1) / share - wg0 + 1;
      here += n;
    }
    const bool next_row = here - at >= unit * a.n_kv;

    Wave<L, NB, 1> st;
    st.clear();
    {
      const __bf16* q = a.q + ((long long)b * a.n_q + kvh * a.rep + min(n16, a.rep - 1)) * HD;
#pragma unroll
      for (int s = 0; s < 4; ++s) st.q[0][s] = *reinterpret_cast<const bf16x8*>(q + q_chan<L>(s, g));
    }
    st.pass(lo + w, min(hi, (r.seen + 31) >> 5), 4, r.seen, a.qscale, a.dv, [&](int blk, const char*& k, const char*& v) __attribute__((always_inline)) {
      place_of(a, blk < r.pblocks ? r.lead : b, kvh, blk, k, v);
    });
    __syncthreads();                      // lds may still be read for the item before
    to_lds(lds, st, 0);
    __syncthreads();
    const int vecs = a.dv / 4;
    auto slot = [&](int c) { return cut ? wg0 + c : 2 * (wg0 + c) + (c < chunks - 1 ? 1 : 0); };
    const long long part_size = (long long)a.rep * (a.dv + 2);
    bool join = true;
    if (chunks > 1) {
      float* po = a.part + slot(chunk) * part_size;
      for (int e = tid; e < a.rep * vecs; e += 256) {
        const int h = e / vecs, d = 4 * (e - h * vecs);
        const Joined j = join_waves(lds, h, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) __hip_atomic_store(po + h * a.dv + d + i, j.y[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        if (d == 0) {
          __hip_atomic_store(po + a.rep * a.dv + h, j.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
          __hip_atomic_store(po + a.rep * a.dv + a.rep + h, j.l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
      }
      // The parts' done flags, as the split items of the decode have them (chunks_all_done), but not next to each other.
      __builtin_amdgcn_s_waitcnt(0);      // this thread's part has been written
      __syncthreads();
      if (tid < 64) {
        if (tid == 0) __hip_atomic_store(a.flags + slot(chunk), a.epoch, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the flag is in memory before the others are read
        bool set = true;
        for (int c = tid; c < chunks; c += 64)
          set = set && __hip_atomic_load(a.flags + slot(c), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) == a.epoch;
        const bool all = __all(set);
        if (all)
          for (int c = tid; c < chunks; c += 64) __hip_atomic_store(a.flags + slot(c), 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        if (tid == 0) found[2] = all ? 1 : 0;
      }
      __syncthreads();
      join = found[2] != 0;
    }
    if (join) {
      for (int e = tid; e < a.rep * vecs; e += 256) {
        const int h = e / vecs, d = 4 * (e - h * vecs);
        Joined j;
        if (chunks == 1) {
          j = join_waves(lds, h, d);
        } else {
          for (int c = 0; c < chunks; ++c) {
            const float* po = a.part + slot(c) * part_size;
            f32x4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __hip_atomic_load(po + h * a.dv + d + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            j.add(y, __hip_atomic_load(po + a.rep * a.dv + h, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM),
                  __hip_atomic_load(po + a.rep * a.dv + a.rep + h, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM));
          }
        }
        if (r.pieces) {
          const int col = r.local * a.rep + h, tile = col / a.pre_cols, x = col - tile * a.pre_cols;
          const long long size = (long long)a.pre_cols * (a.dv + 2);
          const float* po = a.pre + (r.base + (long long)(tile * a.n_kv + kvh) * r.pieces) * size;
          for (int c = 0; c < r.pieces; ++c, po += size)
            j.add(*reinterpret_cast<const f32x4*>(po + x * a.dv + d), po[a.pre_cols * a.dv + x], po[a.pre_cols * (a.dv + 1) + x]);
        }
        const float inv = 1.f / j.l;
        const f32x4 y = r.seen == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : j.y * inv;   // a row that sees nothing: zeros
        store4(a, ((long long)b * a.n_q + kvh * a.rep + h) * a.dv + d, y);
      }
    }
    if (next_row) {
      at += unit * a.n_kv;
      ++b;
    }
  }
}

// ---- the groups' prefixes -----------------------------------------------------------------------
// An item is 16 C columns (queries of neighbouring rows) of a group and a KV head; its blocks are cut into the group's number
// of pieces, a workgroup each, so that all pieces fit the chip at once where they can. The first workgroups write what the
// second launch has to know of every row.

inline int pre_wgs(int C) { return C == 4 ? 256 : 512; }    // that the chip holds at once
inline int pre_tile(int B, int n_groups, int rep) {         // C by the average group
  const int cols = (B + n_groups - 1) / n_groups * rep;
  return cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
}
// Column tiles of all groups, at most, and pieces: tiles of n blocks are cut into at most n / len + 1 pieces, len at least the
// workgroups' even share of all blocks.
inline long long pre_tiles(int B, int n_groups, int rep, int C) { return (long long)B * rep / (16 * C) + std::min(B, n_groups); }
inline long long pre_slots(int B, int n_groups, int rep, int n_kv, int C) { return pre_wgs(C) + pre_tiles(B, n_groups, rep, C) * n_kv; }
inline size_t pre_bytes(int B, int n_groups, int rep, int n_kv, int dv) {
  const int C = pre_tile(B, n_groups, rep);
  return (size_t)pre_slots(B, n_groups, rep, n_kv, C) * 16 * C * (dv + 2) * sizeof(float) + (size_t)B * sizeof(RowPrefix);
}

struct Group {
  int row, rows, blocks;                  // blocks: of the prefix, 0 where nothing is shared
};
__device__ __forceinline__ Group group_of(const StepArgs& a, int gi) {
  const int c0 = a.cu ? a.cu[gi] : 0, c1 = a.cu ? a.cu[gi + 1] : a.B;
  Group g;
  g.row = min(max(c0, 0), a.B);
  g.rows = min(max(c1, g.row), a.B) - g.row;
  g.blocks = g.rows > 1 ? min(max(a.shared[gi], 0), a.capacity) >> 5 : 0;      // (a lone row has its blocks to itself)
  return g;
}

template <int L, int NB, int C>
__global__ __launch_bounds__(256, C == 4 ? 1 : 2) void palu_prefix_kernel(const StepArgs a) {
  __shared__ WaveLds<NB> lds;
  __shared__ int scan[4], found[2], bases[256];
  constexpr int COLS = 16 * C;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = (a.n_groups + 255) / 256, g0 = min(tid * per, a.n_groups), g1 = min(g0 + per, a.n_groups);
  constexpr int WGS = C == 4 ? 256 : 512;
  auto tiles_of = [&](const Group& g) { return g.blocks ? (g.rows * a.rep + COLS - 1) / COLS * a.n_kv : 0; };   // of all KV heads
  // blocks of a piece: the first of a few lengths whose pieces the chip holds at once
  int mine = 0, total, len = 8;
  for (int i = g0; i < g1; ++i) {
    const Group g = group_of(a, i);
    mine += tiles_of(g) * g.blocks;
  }
  wg_scan(mine, scan, total);
  int before, all;
  for (int t = 0; t < 4; ++t) {           // uniform
    len = max(8, (int)(((long long)(total + WGS - 1) / WGS) * (8 + t) / 8));
    mine = 0;
    for (int i = g0; i < g1; ++i) {
      const Group g = group_of(a, i);
      mine += tiles_of(g) * ((g.blocks + len - 1) / len);
    }
    before = wg_scan(mine, scan, all);
    if (all <= WGS) break;
  }
  const int row_wgs = (a.B + 255) / 256;
  if ((int)blockIdx.x < row_wgs) {        // the rows' records, a thread each
    bases[tid] = before;
    __syncthreads();
    const int b = (int)blockIdx.x * 256 + tid;
    if (b >= a.B) return;
    int gi = 0;
    for (int end = a.n_groups; end - gi > 1;) {   // the last group that begins at b or before it
      const int mid = (gi + end) >> 1;
      if (a.cu[mid] <= b) gi = mid;
      else end = mid;
    }
    RowPrefix r{b, 0, 0, 0, 0, {}};
    const Group g = group_of(a, gi);
    if (g.blocks && b >= g.row && b < g.row + g.rows) {
      int base = bases[gi / per];
      for (int i = gi / per * per; i < gi; ++i) {
        const Group x = group_of(a, i);
        base += tiles_of(x) * ((x.blocks + len - 1) / len);
      }
      const int pieces = (g.blocks + len - 1) / len;
      // (Groups that overlap, where the offsets make no sense, can be more pieces than the workspace was sized for.)
      r = RowPrefix{g.row, g.blocks, base >= 0 && base + tiles_of(g) * pieces <= a.pre_slots ? pieces : 0, base, b - g.row, {}};
    }
    a.rows[b] = r;
    return;
  }
  const int want = (int)blockIdx.x - row_wgs;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  if (want >= before && want < before + mine) {
    int at = before;
    for (int i = g0; i < g1; ++i) {
      const Group g = group_of(a, i);
      const int pieces = (g.blocks + len - 1) / len, n = tiles_of(g) * pieces;
      if (want >= at && want < at + n) {
        found[0] = i;
        found[1] = want - at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  const int gi = __builtin_amdgcn_readfirstlane(found[0]);
  if (gi < 0) return;                     // uniform: past the last piece
  const Group g = group_of(a, gi);
  const int in = __builtin_amdgcn_readfirstlane(found[1]), pieces = (g.blocks + len - 1) / len;
  const int tile = in / pieces, piece = in - tile * pieces, kvh = tile % a.n_kv, ct = tile / a.n_kv;
  const int each = (g.blocks + pieces - 1) / pieces, lo = piece * each, hi = min(g.blocks, lo + each);
  const int n16 = lane & 15, gl = lane >> 4;
  Wave<L, NB, C> st;
  st.clear();
#pragma unroll
  for (int x = 0; x < C; ++x) {
    const int col = min(ct * COLS + 16 * x + n16, g.rows * a.rep - 1), row = col / a.rep;   // columns past the group repeat its last
    const __bf16* q = a.q + ((long long)(g.row + row) * a.n_q + kvh * a.rep + (col - row * a.rep)) * HD;
#pragma unroll
    for (int s = 0; s < 4; ++s) st.q[x][s] = *reinterpret_cast<const bf16x8*>(q + q_chan<L>(s, gl));
  }
  st.pass(lo + w, hi, 4, 32 * g.blocks, a.qscale, a.dv, [&](int blk, const char*& k, const char*& v) __attribute__((always_inline)) {
    place_of(a, g.row, kvh, blk, k, v);
  });
  float* po = a.pre + (long long)want * COLS * (a.dv + 2);
  const int vecs = a.dv / 4;
#pragma unroll
  for (int x = 0; x < C; ++x) {
    if (x) __syncthreads();
    to_lds(lds, st, x);
    __syncthreads();
    for (int e = tid; e < 16 * vecs; e += 256) {
      const int n = e / vecs, d = 4 * (e - n * vecs), col = 16 * x + n;
      const Joined j = join_waves(lds, n, d);
      *reinterpret_cast<f32x4*>(po + col * a.dv + d) = j.y;
      if (d == 0) {
        po[COLS * a.dv + col] = j.m;
        po[COLS * (a.dv + 1) + col] = j.l;
      }
    }
  }
}

// ---- launches -----------------------------------------------------------------------------------
template <typename K>
int step_launch(K kern, unsigned grid, const StepArgs& a, const char* who, hipStream_t s) {
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
}

template <int L, int NB>
int step_run_nb(const StepArgs& a, const char* who, hipStream_t s) {
  if (a.rows) {
    const unsigned grid = (unsigned)((a.B + 255) / 256 + a.pre_slots);
    const int rc = a.pre_cols == 16   ? step_launch(palu_prefix_kernel<L, NB, 1>, grid, a, who, s)
                   : a.pre_cols == 32 ? step_launch(palu_prefix_kernel<L, NB, 2>, grid, a, who, s)
                                      : step_launch(palu_prefix_kernel<L, NB, 4>, grid, a, who, s);
    if (rc) return rc;
  }
  return step_launch(palu_step_kernel<L, NB>, (unsigned)step_grid(a.B, a.n_kv), a, who, s);
}

template <int L>
int step_run(const StepArgs& a, const char* who, hipStream_t s) {
  switch ((a.dv + 31) / 32) {
    case 1: return step_run_nb<L, 1>(a, who, s);
    case 2: return step_run_nb<L, 2>(a, who, s);
    case 3: return step_run_nb<L, 3>(a, who, s);
    default: return step_run_nb<L, 4>(a, who, s);
  }
}

}  // namespace
