// One new token per row over cached full K and V: the decode attention of quantised caches (palu_flash_decode and its paged
// form in the MX layouts) and of batches whose rows share prefixes (palu_flash_decode_shared, all layouts),
//   out[b][h] = sum_{p <= cur[b]} softmax_p(scale q[b][h] . k[p][j]) v[p][j],   j = h / rep, rep = n_q / n_kv.
// Included by one translation unit per family of layouts.
//
// A wave takes whole 32-position blocks, the four waves of a workgroup every fourth (in fp4 every fourth pair). Its columns are
// up to 16 C queries:
//   S^T (keys x columns) = K Q^T, two v_mfma_f32_16x16x32_bf16 tiles of 16 keys, Q the B operand, in registers;
//   P^T = 2^(S^T - m), the running maximum m refreshed when a score exceeds it by more than 2^8;
//   O^T (channels x columns) += V^T P^T.
// The rows of the K operand are the keys in the order of the caches' K tiles: the two accumulators then leave a lane with
// the eight keys 8 g .. + 7 of its column, which is the B operand of the second product, and no value changes lanes. Tiled
// and quantised caches hold both operands as they are taken, 8 bytes or more of a lane in one piece; a quantised value is
// turned into bf16 (exactly) between memory and product, a lane's 32 channels of a key under one scale, two channels of a
// position under one scale of V, which two byte permutations make pairs of positions. Row-major V is read in the same pairs.
//
// Bound by memory for long batches: 32 rows of 8192 positions, 8 KV heads, in fp8 554 MB in 88 us, 6.3 TB/s (a copy of this card
// reaches 4.9, a pure read 6.3), in fp4 285 MB in 52 us. For that a wave has a block of 8 KB or more on its way while it computes
// another: copies straight to LDS, which take no registers, and not kept in the caches (kept there fp8 took 102 us); the next copy
// goes out as soon as the block is in registers. A second block in registers spilled, and so did three workgroups a CU (115 us).
// Page ids are uniform and read as scalars a turn early: as vector loads each was waited for together with the blocks before it.
// Short ones are a chain of latencies: a launch 4 us, lengths, pages and queries 2, a first block 1 to 2, and where a row is cut, 3
// for the pieces to meet (one row of 300 positions: 9 us; of 2048: 12; of 32768: 21 in fp4, 23 in fp8).
//
// Rounding: products of bf16 are exact in fp32, scores, statistics and sums are fp32; the probabilities are rounded to bf16
// for the second product, by up to 2^-8 of each, and it is the rounded ones that are summed to divide by.
#pragma once
#include "palu_mx.h"

#include <algorithm>

namespace palu {

// What a row has of a prefix: its blocks 0 .. blocks - 1 are read through the table of its group's lead (lead_of), one of `rows`
// rows from `first` on; where pieces > 0 they have been read, and the row's queries are columns local * rep .. of the group's, in
// slots base + (tile * n_kv + kv) * pieces ..
struct RowPrefix {
  int first, rows, blocks, pieces, base, local, unused[2];
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
  // Shared prefixes (shared null: none; rows null: not read ahead).
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
// A block on its way: copied to LDS as it lies (row-major K in the order of its operands), a wave's own place, then read into
// registers at once, so that the next copy can go to the same place while this block is computed.
typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

// The registers of a block: K, V of NB blocks of 32 channels.
template <int L, int NB>
struct Raw {
  static constexpr bool MX = is_mx(L), FP8 = mx_fp8(L);
  static constexpr int KI = MX ? (FP8 ? 4 : 2) : 8, VI = MX ? (FP8 ? NB : (NB + 1) / 2) : 2 * NB;   // copies of a kilobyte
  static constexpr int COPIES = KI + VI + (MX ? 1 : 0);                                           // and one of the scales
  static constexpr int BYTES = (KI + VI) * 1024 + (MX ? 256 : 0);
  u32x4 k[KI];
  unsigned ks;                            // scales of half-blocks 0 and 1
  u32x4 v[VI];
  u32x2 vs[MX ? NB : 1];
};

// lane = 16 g + n. NT: not kept in the caches, as data that is read once. Rows that read their prefix by themselves read it
// several times, but are not slower for it (8 to 32 rows behind 500 to 1000 positions in any layout: within 0.2 us).
template <bool NT, int L, int NB>
__device__ __forceinline__ void copy_block(char* to, const char* k, const char* v, int dv) {
  using R = Raw<L, NB>;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;

  // Copy i of a run that lies the same way in memory and in LDS: the instruction's offset counts for both (up to 4 KB).
  auto run = [&](const char* from, char* at, auto count) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
    if constexpr (N > 0) __builtin_amdgcn_global_load_lds((gvoid*)from, (lvoid*)at, 16, 0, NT ? 2 : 0);
    if constexpr (N > 1) __builtin_amdgcn_global_load_lds((gvoid*)from, (lvoid*)at, 16, 1024, NT ? 2 : 0);
    if constexpr (N > 2) __builtin_amdgcn_global_load_lds((gvoid*)from, (lvoid*)at, 16, 2048, NT ? 2 : 0);
    if constexpr (N > 3) __builtin_amdgcn_global_load_lds((gvoid*)from, (lvoid*)at, 16, 3072, NT ? 2 : 0);
  };
  auto one = [&](const char* from, int i) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds((gvoid*)from, (lvoid*)(to + i * 1024), 16, 0, NT ? 2 : 0);
  };
  const unsigned l16 = lane * 16;
  if constexpr (L == PALU_LAYOUT_ROWS) {  // key (c, n), channels 32 s + 8 g .. + 7
#pragma unroll
    for (int i = 0; i < R::KI; ++i) {
      const int key = 8 * (n >> 2) + 4 * (i >> 2) + (n & 3);
      one(k + (unsigned)(key * (2 * HD) + (i & 3) * 64 + g * 16), i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < R::KI; i += 4)
      run(k + i * 1024 + l16, to + i * 1024, std::integral_constant<int, (R::KI > 4 ? 4 : R::KI)>());
  }
  char* tv = to + R::KI * 1024;
  if constexpr (L == PALU_LAYOUT_TILED || L == PALU_LAYOUT_ROWS) {
#pragma unroll
    for (int i = 0; i < R::VI; ++i)       // (of an odd multiple of 16 the last tile, or kilobyte, again)
      one(v + (L == PALU_LAYOUT_TILED ? min(i, dv / 16 - 1) * 1024 + l16 : min(i * 1024 + l16, 64u * dv - 16)), R::KI + i);
  } else {                                // (past the end, of half a kilobyte, the last piece again)
    constexpr int FULL = mx_codes(R::FP8, 32 * NB) / 1024;
    run(v + l16, tv, std::integral_constant<int, FULL>());
    if constexpr (FULL < R::VI) one(v + FULL * 1024 + min(l16, 512u - 16), R::KI + FULL);
    // 128 bytes of K's scales, then those of V
    const char *ks = k + mx_codes(R::FP8, HD), *vs = v + mx_codes(R::FP8, 32 * NB);
    const char* from = lane < 32 ? ks + 4 * lane : vs + min(4 * (lane - 32), 32 * NB - 4);
    __builtin_amdgcn_global_load_lds((gvoid*)from, (lvoid*)(to + (R::KI + R::VI) * 1024), 4, 0, NT ? 2 : 0);
  }
}
// K's part of the registers out of its elements and scales (a copy in LDS, or all but row-major ones as they lie in memory), then
// V's.
template <int L, int NB>
__device__ __forceinline__ void read_k(Raw<L, NB>& r, const char* k, const char* scales) {
  const unsigned lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < Raw<L, NB>::KI; ++i) r.k[i] = *reinterpret_cast<const u32x4*>(k + i * 1024 + lane * 16);
  if constexpr (is_mx(L)) r.ks = *reinterpret_cast<const unsigned short*>(scales + 2 * lane);
}
template <int L, int NB, bool LDS>
__device__ __forceinline__ void read_v(Raw<L, NB>& r, const char* v, const char* scales, int dv) {
  using R = Raw<L, NB>;
  const unsigned lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  if constexpr (R::MX) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (R::FP8) {
        r.v[b] = *reinterpret_cast<const u32x4*>(v + b * 1024 + lane * 16);
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(v + b * 512 + lane * 8);
        r.v[b / 2][2 * (b & 1)] = x[0];
        r.v[b / 2][2 * (b & 1) + 1] = x[1];
      }
      r.vs[b] = *reinterpret_cast<const u32x2*>(scales + b * 32 + 8 * g);
    }
  } else if constexpr (L == PALU_LAYOUT_TILED) {
#pragma unroll
    for (int i = 0; i < R::VI; ++i)
      r.v[i] = *reinterpret_cast<const u32x4*>(v + (LDS ? i : min(i, dv / 16 - 1)) * 1024 + lane * 16);
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 8; ++j) {       // position 8 g + j, channels 32 b + 2 n and 2 n + 1
        const char* pair = v + (8 * g + j) * (2 * dv) + min(64 * b + 4 * n, 2u * dv - 4);
        r.v[2 * b + j / 4][j & 3] = *reinterpret_cast<const unsigned*>(pair);
      }
  }
}
template <int L, int NB>
__device__ __forceinline__ void read_block(Raw<L, NB>& r, const char* s, int dv) {
  using R = Raw<L, NB>;
  const char* sc = s + (R::KI + R::VI) * 1024;
  read_k<L, NB>(r, s, sc);
  read_v<L, NB, true>(r, s + R::KI * 1024, sc + 128, dv);
}

// Neighbouring blocks that a wave takes together: some 8 KB or more on their way to it.
constexpr int step_group(int layout) { return layout == PALU_LAYOUT_MX4 ? 2 : 1; }

// This wave's copies have arrived, its reads from LDS are done.
__device__ __forceinline__ void wait_copies() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0)
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_reads() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xc07f);     // lgkmcnt(0)
  __builtin_amdgcn_sched_barrier(0);
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

  // One row's query, 16 bytes a piece. Its signs are turned for a negative scale, so that qscale is not, and the largest score
  // is that of the largest product.
  __device__ __forceinline__ void query(int x, const __bf16* from, bool neg) {
    const unsigned sign = neg ? 0x80008000u : 0u;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const u32x4 u = *reinterpret_cast<const u32x4*>(from + q_chan<L>(s, (threadIdx.x & 63) >> 4)) ^ sign;
      q[x][s] = __builtin_bit_cast(bf16x8, u);
    }
  }

  // The block's positions 0 .. seen - 1 (MASK: the rest may hold anything).
  template <bool MASK, typename AK, typename AV>
  __device__ __forceinline__ void add(const Raw<L, NB>& r, float qscale, int seen, AK&& after_k, AV&& after_v) {
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
    after_k();
    bf16x8 p[C];
#pragma unroll
    for (int x = 0; x < C; ++x) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (MASK && 8 * g + 4 * c + i >= seen) s[x][c][i] = NEG_INF;
      const float top = max8(s[x][0], s[x][1]) * qscale;
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
      for (int j = 0; j < 8; ++j) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][j >> 2][j & 3], qscale, -ref));
        p[x][j] = (__bf16)(MASK && 8 * g + j >= seen ? 0.f : e);               // (-inf times a scale of 0 would be NaN)
      }
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
    after_v();
  }
  template <bool MASK>
  __device__ __forceinline__ void add(const Raw<L, NB>& r, float qscale, int seen) {
    add<MASK>(r, qscale, seen, [] {}, [] {});
  }

  // The same over whole blocks straight from memory into the registers, the next block's K as soon as this one's scores are done,
  // its V after this one's products: for blocks that several workgroups read and the L2 holds, the way over LDS is the longer
  // one (64 rows with a prefix of 8192 in bf16: 24.4 -> 22.3 us). Blocks that are read once are longer on their way.
  template <int NW, typename P, typename F>
  __device__ __forceinline__ void pass_direct(int first, int end, float qscale, int dv, P&& page_at, F&& where) {
    first += __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (first >= end) return;
    Raw<L, NB> r;
    const char *k, *v;
    constexpr int KS = is_mx(L) ? mx_codes(mx_fp8(L), HD) : 0, VS = is_mx(L) ? mx_codes(mx_fp8(L), 32 * NB) : 0;
    where(page_at(first), first, k, v);
    int page = page_at(min(first + NW, end - 1));
    read_k<L, NB>(r, k, k + KS);
    read_v<L, NB, false>(r, v, v + VS, dv);
    for (int blk = first; blk < end; blk += NW) {
      const int next = min(blk + NW, end - 1);
      where(page, next, k, v);
      page = page_at(min(blk + 2 * NW, end - 1));
      add<false>(r, qscale, 32,
          [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            read_k<L, NB>(r, k, k + KS);
            __builtin_amdgcn_sched_barrier(0);
          },
          [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            read_v<L, NB, false>(r, v, v + VS, dv);
            __builtin_amdgcn_sched_barrier(0);
          });
    }
  }

  // This wave's blocks of first .. end - 1, of a sequence that is seen up to position seen - 1 (ALL: whole blocks only): a group
  // of them, then the one `waves` groups further, and so on. page_at(blk) gives a block's page, where(page, blk, k, v) its places;
  // s: the wave's place in LDS. While a group is computed the next one is on its way; its pages are asked for a turn earlier.
  template <bool ALL, typename P, typename F>
  __device__ __forceinline__ void pass(int first, int waves, int end, int seen, float qscale, int dv, char* s, P&& page_at,
                                       F&& where) {
    using R = Raw<L, NB>;
    constexpr int G = step_group(L);
    if (first >= end) return;
    int page[G];
    auto pages = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < G; ++i) page[i] = page_at(min(blk + i, end - 1));
    };
    auto fetch = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const char *k, *v;
        where(page[i], min(blk + i, end - 1), k, v);
        copy_block<!ALL, L, NB>(s + i * R::BYTES, k, v, dv);
      }
    };
    pages(first);
    wait_copies();                        // the queries are here (the pages took as long)
    fetch(first);
    for (int blk = first; blk < end;) {
      const int next = blk + waves * G;
      pages(min(next, end - 1));
      wait_copies();
      R r[G];
#pragma unroll
      for (int i = 0; i < G; ++i) read_block<L, NB>(r[i], s + i * R::BYTES, dv);
      wait_reads();
      if (next < end) fetch(next);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        if (ALL ? blk + i < end : 32 * (blk + i) + 32 <= seen && blk + i < end) add<false>(r[i], qscale, 32);
        else if (!ALL && blk + i < end) add<true>(r[i], qscale, seen - 32 * (blk + i));
      }
      blk = next;
    }
  }
};

// Column tile x of every wave's state in LDS: O [wave][cols][OS], then m and l [wave][cols]; only the first `cols` columns.
// Barriers around it are the caller's.
template <int NB>
struct WaveLds {
  static constexpr int OS = 32 * NB + 4;
  float* o;
  int cols;
  __host__ __device__ static constexpr int bytes(int cols) { return 4 * cols * (OS + 2) * (int)sizeof(float); }
  __device__ __forceinline__ float* row(int w, int n) const { return o + (w * cols + n) * OS; }
  __device__ __forceinline__ float& m(int w, int n) const { return o[4 * cols * OS + w * cols + n]; }
  __device__ __forceinline__ float& l(int w, int n) const { return o[4 * cols * (OS + 1) + w * cols + n]; }
};
// LDS of a workgroup: the waves' places for blocks on their way, afterwards their results.
template <int L, int NB>
constexpr int place_bytes() { return step_group(L) * Raw<L, NB>::BYTES; }
template <int L, int NB>
constexpr int step_lds() {
  return 4 * place_bytes<L, NB>() > WaveLds<NB>::bytes(16) ? 4 * place_bytes<L, NB>() : WaveLds<NB>::bytes(16);
}

template <int L, int NB, int C>
__device__ __forceinline__ void to_lds(const WaveLds<NB>& s, const Wave<L, NB, C>& st, int x) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, w = threadIdx.x >> 6;
  const float l = wave_sum_xor48(st.l[x]);
  if (n >= s.cols) return;
  if (g == 0) {
    s.m(w, n) = st.m[x];
    s.l(w, n) = l;
  }
  float* row = s.row(w, n);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const f32x4 y = st.o[x][2 * b], z = st.o[x][2 * b + 1];    // rows 4 g .. + 3 of tiles 0 and 1
    if constexpr (L == PALU_LAYOUT_TILED) {
      *reinterpret_cast<f32x4*>(row + 32 * b + 4 * g) = y;
      *reinterpret_cast<f32x4*>(row + 32 * b + 16 + 4 * g) = z;
    } else {
      *reinterpret_cast<f32x4*>(row + 32 * b + 8 * g) = f32x4{y[0], z[0], y[1], z[1]};
      *reinterpret_cast<f32x4*>(row + 32 * b + 8 * g + 4) = f32x4{y[2], z[2], y[3], z[3]};
    }
  }
}

// Four channels of a column, summed from parts: y and l stand over 2^m.
struct Joined {
  f32x4 y;
  float m, l;
  __device__ __forceinline__ void add(f32x4 py, float pm, float pl) {
    const float mn = fmaxf(m, pm);
    const float ref = mn == NEG_INF ? 0.f : mn;               // (then both have nothing, or NaN)
    const float wa = __builtin_amdgcn_exp2f(m - ref), wb = __builtin_amdgcn_exp2f(pm - ref);
    y = y * wa + py * wb;
    l = l * wa + pl * wb;
    m = mn;
  }
};
__device__ __forceinline__ Joined no_parts() { return Joined{{0.f, 0.f, 0.f, 0.f}, NEG_INF, 0.f}; }
template <int NB>
__device__ __forceinline__ Joined join_waves(const WaveLds<NB>& s, int n, int d) {
  Joined j = no_parts();
#pragma unroll
  for (int w = 0; w < 4; ++w) j.add(*reinterpret_cast<const f32x4*>(s.row(w, n) + d), s.m(w, n), s.l(w, n));
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
  total = __builtin_amdgcn_readfirstlane(total);            // what follows from it is uniform, and the page reads scalar
  return before + s - x;
}

// Sums of x and y over the workgroup's 256 threads, in every thread and uniform: of counts, exact up to 2^24. `part`: 8 floats.
__device__ __forceinline__ void wg_sum2(float& x, float& y, float* part) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    x += __shfl_xor(x, d);
    y += __shfl_xor(y, d);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6] = x;
    part[4 + (threadIdx.x >> 6)] = y;
  }
  __syncthreads();
  auto all = [](const float* p) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, p[0] + p[1] + p[2] + p[3])));
  };
  x = all(part);
  y = all(part + 4);
}
__device__ __forceinline__ float wg_sum(float x, float* part) {
  float none = 0.f;
  wg_sum2(x, none, part);
  return x;
}

// How items are cut into pieces of up to len blocks, a workgroup each: the first of a few lengths, from an even share of all
// blocks on (total: a float, since rows that share their pages can be more blocks than an int holds), of which the chip holds
// all pieces (`slots`) at once, and at least `least`. of(i) gives n items of some blocks each; a thread has i0 .. i1 - 1. Its
// pieces are number before .. before + mine - 1 of all; where they never fit, they are at most slots + all items. fit: that
// they can is likely, and lengths of up to 15/8 of a share are tried; otherwise 11/8 is taken. Whole shares of
// items, some workgroups with a little less to do, were faster than even shares that begin and end inside items and join more
// parts (64 rows of up to 2304 positions in fp4: 33 us against 37).
struct Cut {
  int len, before, mine, all;
  __device__ __forceinline__ int pieces(int blocks) const { return (blocks + len - 1) / len; }
};
struct Items {
  int n, blocks;
};
template <typename F>
__device__ __forceinline__ Cut cut_items(float total, int i0, int i1, int slots, int least, bool fit, int* scan, F&& of) {
  const float up = total < 0x1p24f ? 1.f : 1.f + 0x1p-14f;    // (the total may be rounded)
  const int share = max(least, (int)ceilf(total / (float)slots * up));
  Cut c;
  for (int t = fit ? 0 : 3; ; t += t < 3 ? 1 : 2) {           // (uniform)
    c.len = share + share / 8 * t + share % 8 * t / 8;
    c.mine = 0;
    for (int i = i0; i < i1; ++i) {
      const Items x = of(i);
      c.mine += x.n * c.pieces(x.blocks);
    }
    c.before = wg_scan(c.mine, scan, c.all);
    if (c.all <= slots || !fit || t == 7) break;
  }
  return c;
}

__device__ __forceinline__ int seen_of(const StepArgs& a, int pos) { return min(max(pos, -1), a.capacity - 1) + 1; }

// The page of block blk of a row, and the places of a KV head's block on it.
__device__ __forceinline__ int page_of(const StepArgs& a, int row, int blk) {
  if (!a.table) return row;
  return min(max(load_uniform(a.table, (long long)row * a.pt_stride + (blk >> a.page_shift)), 0), a.n_pages - 1);
}
__device__ __forceinline__ void place_of(const StepArgs& a, int page, int kvh, int blk, const char*& k, const char*& v) {
  const int at = a.table ? blk & ((1 << a.page_shift) - 1) : blk;
  k = a.k + page * a.k_page + kvh * a.k_head + (long long)at * a.k_blk;
  v = a.v + page * a.v_page + kvh * a.v_head + (long long)at * a.v_blk;
}

// ---- the rows' own blocks -----------------------------------------------------------------------
// An item is a row's KV head: its blocks, but for those that have been read with the group's prefix, cut into even pieces. The
// pieces of an item are joined by the workgroup that finds all of them done.
// Blocks of a piece, at least: four turns of its waves (fp4: two). With 8 a row of 2048 positions is 1.5 us faster, rows of 300
// and 512 are 1.5 to 3 us slower, for they are cut then.
constexpr int STEP_LEAST = 16;
constexpr int STEP_WGS = 512;             // workgroups that the chip holds at once, by the kernel's LDS and registers
// More items than those (MANY): rows of up to STEP_SHORT own blocks have four KV heads to a workgroup, one to a wave, which adds the
// prefix's pieces by itself, one after the other, where they are STEP_PIECES at most (a prefix of few rows can be hundreds: 65
// rows with 8 KV heads, two of them behind 32000 positions in fp8, 69 us if a wave joins its 63 pieces, 35 if a workgroup does; 600 rows
// with one, two of them behind 65000, 147 and 43; with 4 as the limit 65 rows behind 30000 take 78 us, with 8 or 16 76); of others a
// workgroup has a piece, as ever. Above 1024 items 512 workgroups take piece after
// piece, since one that finds no piece holds a place for 3 us to find that out (512 rows of up to 64 positions, 8 KV heads, fp8:
// 77 -> 18.5 us; 256 of up to 200: 37 -> 19; 256 behind a prefix of 2000: 37 -> 16). Up to there each piece has its own, which
// balances long rows better (66 rows of up to 4000: 68 us, 78 in such a loop). With 4 blocks as the limit 256 rows of 200 take 27
// us, with 16 32 rows of up to 1024 with 32 KV heads 46 against 37; with 256 items as the bound 64 rows of up to 250 take 13.8
// against 11.6.
constexpr int STEP_SHORT = 8;
constexpr int STEP_PIECES = 8;
inline bool step_many(int B, int n_kv) { return (long long)B * n_kv > STEP_WGS; }
inline int step_slots(int B, int n_kv) { return STEP_WGS + B * n_kv; }         // pieces, at most
inline int step_grid(int B, int n_kv) { return B * n_kv > 1024 ? STEP_WGS : step_slots(B, n_kv); }
inline size_t step_bytes(int B, int n_kv, int rep, int dv) {
  return (size_t)step_slots(B, n_kv) * ((size_t)rep * (dv + 2) * sizeof(float) + sizeof(unsigned long long));
}

struct Group {
  int row, rows, blocks;                  // blocks: of the prefix, 0 where nothing is shared
};
__device__ __forceinline__ Group group_of(const StepArgs& a, int gi, bool lone) {
  const int c0 = a.cu ? a.cu[gi] : 0, c1 = a.cu ? a.cu[gi + 1] : a.B;
  Group g;
  g.row = min(max(c0, 0), a.B);
  g.rows = min(max(c1, g.row), a.B) - g.row;
  g.blocks = g.rows > (lone ? 0 : 1) ? min(max(a.shared[gi], 0), a.capacity) >> 5 : 0;
  return g;
}

// The last group that begins at row b or before it.
__device__ __forceinline__ int last_group(const StepArgs& a, int b) {
  int gi = 0;
  for (int end = a.n_groups; end - gi > 1;) {
    const int mid = (gi + end) >> 1;
    if (a.cu[mid] <= b) gi = mid;
    else end = mid;
  }
  return gi;
}

// The row through whose table a group's prefix is read: the first whose table begins with a page of the pool, since a row that
// has ended has none, and its pages may be another request's; the group's first where there is no such row. Of a whole wave. It
// takes a call 0.1 to 0.2 us; with the first row's entry asked for together with the lengths the smallest call took the same, large ones
// 0.3 to 0.6 more.
__device__ __forceinline__ int lead_of(const StepArgs& a, int row, int rows) {
  const auto there = [&](int id) { return id >= 0 && id < a.n_pages; };
  if (rows == 1 || there(load_uniform(a.table, (long long)row * a.pt_stride))) return row;
  for (int i = 0; i < rows; i += 64) {    // (uniform)
    const int r = row + min(i + (int)(threadIdx.x & 63), rows - 1);
    const unsigned long long m = __ballot(there(a.table[(long long)r * a.pt_stride]));
    if (m) return row + min(i + __builtin_ctzll(m), rows - 1);
  }
  return row;
}

struct RowWork {
  int first, end, seen, pieces;           // blocks first .. end - 1 (at least one, which may hold nothing), prefix pieces
  int base, local;
  int pblocks, group, rows;               // blocks of the prefix, the group's first row and rows
};
__device__ __forceinline__ RowWork row_work(const StepArgs& a, int b) {
  const int seen = seen_of(a, a.cur[b]), end = (seen + 31) >> 5;
  RowWork r{0, max(end, 1), seen, 0, 0, 0, 0, b, 1};
  if (a.rows) {
    const RowPrefix p = a.rows[b];
    r.group = p.first;
    r.rows = p.rows;
    r.pblocks = p.blocks;
    if (p.pieces && seen >= 32 * p.blocks) {
      r.first = p.blocks;
      r.end = max(end, p.blocks + 1);
      r.pieces = p.pieces;
      r.base = p.base;
      r.local = p.local;
    }
  } else if (a.shared) {                  // nothing has been read: the prefix's blocks are the row's, by its group's table
    const Group g = group_of(a, last_group(a, b), false);
    if (b >= g.row && b < g.row + g.rows) {
      r.group = g.row;
      r.rows = g.rows;
      r.pblocks = g.blocks;
    }
  }
  return r;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ RowWork uniform(const RowWork& r) {
  return RowWork{uniform(r.first), uniform(r.end),     uniform(r.seen),  uniform(r.pieces), uniform(r.base),
                 uniform(r.local), uniform(r.pblocks), uniform(r.group), uniform(r.rows)};
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

// Parts of this launch go to memory and come from there, past the caches, whichever XCD wrote them: system-scope accesses of 4
// and of 16 bytes (which need not be one piece: a flag says that all of a part is there).
constexpr int SYSTEM_SCOPE = 1 | 16;      // sc0, sc1
__device__ __forceinline__ __amdgpu_buffer_rsrc_t parts_at(float* base) {
  return __builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7fffffff, 0x00027000);   // plain bytes
}
__device__ __forceinline__ void store_part(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
__device__ __forceinline__ float load_part(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
__device__ __forceinline__ void store_part4(__amdgpu_buffer_rsrc_t p, int at, f32x4 x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), p, at * 4, 0, SYSTEM_SCOPE);
}
__device__ __forceinline__ f32x4 load_part4(__amdgpu_buffer_rsrc_t p, int at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(p, at * 4, 0, SYSTEM_SCOPE));
}

// A wave's result (of column tile 0), joined with the prefix's pieces (STEP_PIECES at most) and written: row b's
// queries of a KV head. A lane has its channels of a piece as it has its own.
template <int L, int NB>
__device__ __forceinline__ void store_wave(const StepArgs& a, Wave<L, NB, 1>& st, int b, int head, const RowWork& r) {
  constexpr bool T = L == PALU_LAYOUT_TILED;
  int lane = threadIdx.x & 63;
  asm("" : "+v"(lane));                   // (what follows from it is not kept in registers from piece to piece)
  const int n = lane & 15, g = lane >> 4, d0 = (T ? 4 : 8) * g, d1 = d0 + (T ? 16 : 4);   // as in to_lds
  float l = wave_sum_xor48(st.l[0]), m = st.m[0];
  if (n >= a.rep) return;
  f32x4 y[2 * NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const f32x4 p = st.o[0][2 * i], q = st.o[0][2 * i + 1];
    y[2 * i] = T ? p : f32x4{p[0], q[0], p[1], q[1]};
    y[2 * i + 1] = T ? q : f32x4{p[2], q[2], p[3], q[3]};
  }
  if (r.pieces) {                         // (uniform)
    const int size = a.pre_cols * (a.dv + 2), col = r.local * a.rep + n, tile = col / a.pre_cols, x = col - tile * a.pre_cols;
    const float* pre = a.pre + (r.base + (long long)(tile * a.n_kv + head) * r.pieces) * size;
#pragma unroll 1
    for (int c = 0; c < r.pieces; ++c) {
      const float* piece = pre + (long long)c * size;
      const float pm = piece[a.pre_cols * a.dv + x], pl = piece[a.pre_cols * (a.dv + 1) + x];
      f32x4 py[2 * NB];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i)    // (past an odd multiple of 16 the last channels again)
        py[i] = *reinterpret_cast<const f32x4*>(piece + x * a.dv + min(32 * (i / 2) + (i & 1 ? d1 : d0), a.dv - 4));
      const float mn = fmaxf(m, pm), ref = mn == NEG_INF ? 0.f : mn;
      const float wa = __builtin_amdgcn_exp2f(m - ref), wb = __builtin_amdgcn_exp2f(pm - ref);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) y[i] = y[i] * wa + py[i] * wb;
      l = l * wa + pl * wb;
      m = mn;
    }
  }
  const float inv = 1.f / l;
  const long long at = ((long long)b * a.n_q + head * a.rep + n) * a.dv;
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
    const int d = 32 * (i / 2) + (i & 1 ? d1 : d0);
    if (d < a.dv) store4(a, at + d, r.seen == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : y[i] * inv);
  }
}

template <int L, int NB, bool MANY>
__global__ __launch_bounds__(256, 2) void palu_step_kernel(const StepArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[step_lds<L, NB>()];
  const WaveLds<NB> lds{reinterpret_cast<float*>(smem), a.rep};
  __shared__ int scan[8], found[2];
  __shared__ RowWork found_row;
  constexpr int U = 8, MAX_GROUPS = 4;   // parts that a thread has under way, and threads to a column's four channels, at most
  __shared__ union {
    float stats[2][U * MAX_GROUPS][16];   // m and l of parts
    Joined sums[256];
  } joining;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = (a.B + 255) / 256, r0 = min(tid * per, a.B), r1 = min(r0 + per, a.B);
  // this workgroup's piece
  RowWork own;                            // of a thread's only row
  if (r0 < r1) own = row_work(a, r0);
  auto row = [&](int b) { return per == 1 ? own : row_work(a, b); };
  float mine = 0.f;
  for (int i = r0; i < r1; ++i) {
    const RowWork r = row(i);
    mine += (float)a.n_kv * (float)(r.end - r.first);
  }
  // MANY: four KV heads of a short row to a workgroup, one to a wave
  auto to_waves = [&](const RowWork& r) { return MANY && r.end - r.first <= STEP_SHORT && r.pieces <= STEP_PIECES; };
  auto items_of = [&](const RowWork& r) { return to_waves(r) ? Items{(a.n_kv + 3) / 4, 1} : Items{a.n_kv, r.end - r.first}; };
  const bool fit = a.B * a.n_kv <= STEP_WGS * 3 / 4;
  const Cut cut = cut_items(wg_sum(mine, reinterpret_cast<float*>(scan)), r0, r1, STEP_WGS, STEP_LEAST, fit, scan,
                            [&](int i) { return items_of(row(i)); });
  int want = blockIdx.x;
  if (!MANY && want >= cut.all) return;   // uniform
  do {
    if (MANY) {
      if (want >= cut.all) return;        // uniform
      __syncthreads();                    // the piece before is done with LDS
    }
    if (want >= cut.before && want < cut.before + cut.mine) {
      int at = cut.before, b = r0;
      RowWork r = row(b);
      for (;;) {
        const Items x = items_of(r);
        const int n = x.n * cut.pieces(x.blocks);
        if (want < at + n || b + 1 >= r1) break;
        at += n;
        r = row(++b);
      }
      found[0] = b;
      found[1] = want - at;
      found_row = r;
    }
    __syncthreads();
    const int b = uniform(found[0]), in = uniform(found[1]);
    const RowWork r = uniform(found_row);
    const bool each = to_waves(r);          // (uniform)
    const int chunks = each ? 1 : uniform(cut.pieces(r.end - r.first)), head0 = each ? 4 * in : uniform(in / chunks);
    const int chunk = each ? 0 : in - head0 * chunks, wg0 = want - chunk;      // wg0: the item's first piece
    const int head = each ? min(head0 + w, a.n_kv - 1) : head0;                // this wave's
    const int len = uniform((r.end - r.first + chunks - 1) / chunks), lo = r.first + chunk * len, hi = min(r.end, lo + len);
    Wave<L, NB, 1> st;
    st.clear();
    st.query(0, a.q + ((long long)b * a.n_q + head * a.rep + min(lane & 15, a.rep - 1)) * HD, a.qscale < 0.f);
    const int lead = r.first < r.pblocks ? lead_of(a, r.group, r.rows) : b;    // (uniform)
    st.template pass<false>(
        lo + (each ? 0 : w * step_group(L)), each ? 1 : 4, min(hi, (r.seen + 31) >> 5), r.seen, fabsf(a.qscale), a.dv,
        smem + w * place_bytes<L, NB>(),
        [&](int blk) __attribute__((always_inline)) { return page_of(a, blk < r.pblocks ? lead : b, blk); },
        [&](int page, int blk, const char*& k, const char*& v) __attribute__((always_inline)) {
          place_of(a, page, head, blk, k, v);
        });
    if (each) {                           // (uniform)
      if (head0 + w < a.n_kv) store_wave<L, NB>(a, st, b, head, r);
      continue;
    }
    __syncthreads();                        // every wave is done with its places
    to_lds(lds, st, 0);
    __syncthreads();
    int tid = threadIdx.x;
    if (MANY) asm("" : "+v"(tid));        // (see store_wave)
    const int vecs = a.dv / 4, units = a.rep * vecs;
    const long long part_size = (long long)a.rep * (a.dv + 2);
    if (chunks > 1) {
      float* po = a.part + want * part_size;
      const __amdgpu_buffer_rsrc_t p4 = parts_at(po);
      for (int e = tid; e < units; e += 256) {
        const int h = e / vecs, d = 4 * (e - h * vecs);
        const Joined j = join_waves(lds, h, d);
        store_part4(p4, h * a.dv + d, j.y);
        if (d == 0) {
          store_part(po + a.rep * a.dv + h, j.m);
          store_part(po + a.rep * a.dv + a.rep + h, j.l);
        }
      }
      if (!chunks_all_done(a.flags + wg0, a.epoch, chunks, chunk, found)) continue; // uniform
    }
    const int kvh = head0;
    auto finish = [&](int h, int d, const Joined& j) __attribute__((always_inline)) {
      const float inv = 1.f / j.l;
      const f32x4 y = r.seen == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : j.y * inv;       // a row that sees nothing: zeros
      store4(a, ((long long)b * a.n_q + kvh * a.rep + h) * a.dv + d, y);
    };
    // The parts: this workgroup's own (in LDS), or all workgroups' (one of which is its own), and the prefix's pieces, which the
    // launch before wrote.
    const __amdgpu_buffer_rsrc_t parts = parts_at(a.part + wg0 * part_size);
    const int pre_size = a.pre_cols * (a.dv + 2);
    auto pieces_of = [&](int h, int& x) {   // the pieces of a head, in column x of theirs
      const int col = r.local * a.rep + h, tile = r.pieces ? col / a.pre_cols : 0;
      x = col - tile * a.pre_cols;
      return a.pre + (r.base + (long long)(tile * a.n_kv + kvh) * r.pieces) * pre_size;
    };
    const int groups = min(max(1, 256 / units), MAX_GROUPS), grp = groups > 1 ? tid / units : 0, batch = U * groups;
    for (int e0 = 0; e0 < units; e0 += 256) {                   // (uniform)
      const int e = groups > 1 ? tid - grp * units : e0 + tid;
      const bool on = e < units && grp < groups;
      const int h = on ? e / vecs : 0, d = on ? 4 * (e - h * vecs) : 0;
      Joined j = no_parts();
      // n parts, U to each of 256 / units threads at a time, whose loads are all under way together: stat(c, x, m, l) loads the
      // statistics of part c's column x, four(c) this thread's four channels.
      auto gather = [&](int n, auto&& stat, auto&& four) __attribute__((always_inline)) {
        for (int c0 = 0; c0 < n; c0 += batch) {                 // (uniform)
          float m[MAX_GROUPS], l[MAX_GROUPS];
#pragma unroll
          for (int i = 0; i < MAX_GROUPS; ++i) {
            if (16 * i >= batch || c0 + 16 * i >= n) break;     // (uniform)
            stat(min(c0 + 16 * i + (tid >> 4), n - 1), min(tid & 15, a.rep - 1), m[i], l[i]);
          }
          f32x4 y[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (c0 + u * groups >= n) break;                    // (uniform)
            y[u] = four(min(c0 + u * groups + min(grp, groups - 1), n - 1));
          }
          __syncthreads();                  // the batch before has been read
#pragma unroll
          for (int i = 0; i < MAX_GROUPS; ++i) {
            const int c = 16 * i + (tid >> 4);
            if (16 * i >= batch || c0 + 16 * i >= n) break;
            joining.stats[0][c][tid & 15] = m[i];
            joining.stats[1][c][tid & 15] = l[i];
          }
          __syncthreads();
          if (!on) continue;
          Joined b = no_parts();
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (c0 + u * groups + grp >= n) break;
            b.m = fmaxf(b.m, joining.stats[0][u * groups + grp][h]);
          }
          const float ref = b.m == NEG_INF ? 0.f : b.m;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (c0 + u * groups + grp >= n) break;
            const float f = __builtin_amdgcn_exp2f(joining.stats[0][u * groups + grp][h] - ref);
            b.l += f * joining.stats[1][u * groups + grp][h];
            b.y += f * y[u];
          }
          j.add(b.y, b.m, b.l);
        }
      };
      gather(chunks == 1 ? 0 : chunks, [&](int c, int x, float& m, float& l) __attribute__((always_inline)) {
               const float* p = a.part + (wg0 + c) * part_size + a.rep * a.dv + x;
               m = load_part(p);
               l = load_part(p + a.rep);
             }, [&](int c) __attribute__((always_inline)) { return load_part4(parts, c * (int)part_size + h * a.dv + d); });
      int col, stat_col;
      const float *pre = pieces_of(h, col), *stats = pieces_of(min(tid & 15, a.rep - 1), stat_col);
      gather(r.pieces, [&](int c, int x, float& m, float& l) __attribute__((always_inline)) {
               const float* p = stats + (long long)c * pre_size + a.pre_cols * a.dv + stat_col;
               m = p[0];
               l = p[a.pre_cols];
             }, [&](int c) __attribute__((always_inline)) {
               return *reinterpret_cast<const f32x4*>(pre + (long long)c * pre_size + col * a.dv + d);
             });
      if (on && chunks == 1 && grp == 0) {
        const Joined mine = join_waves(lds, h, d);
        j.add(mine.y, mine.m, mine.l);
      }
      if (groups == 1) {
        if (on) finish(h, d, j);
        continue;
      }
      __syncthreads();                      // the last batch has been read
      if (on) joining.sums[tid] = j;
      __syncthreads();
      if (tid < units) {
        for (int i = 1; i < groups; ++i) {
          const Joined x = joining.sums[tid + i * units];
          j.add(x.y, x.m, x.l);
        }
        finish(h, d, j);
      }
    }
  } while (MANY && (want += gridDim.x, true));
}

// ---- the groups' prefixes -----------------------------------------------------------------------
// An item is 16 C columns (queries of neighbouring rows) of a group and a KV head; its blocks are cut into the group's number
// of pieces, a workgroup each, so that all pieces fit the chip at once where they can. The first workgroups write what the
// second launch has to know of every row.

constexpr int PRE_WGS = 512;              // workgroups that the chip holds at once
// Blocks of a piece, at least. With 4 single short prefixes are 0.5 us faster, larger batches slower (64 rows behind 512 positions in
// tiles, both launches: 24.8 us, 26.5).
constexpr int PRE_LEAST = 8;
inline int pre_tile(int B, int n_groups, int rep) {         // C by the average group
  const int cols = (B + n_groups - 1) / n_groups * rep;
  return cols <= 16 ? 1 : 2;
}
// Column tiles of all groups, at most, and pieces: tiles of n blocks are cut into at most n / len + 1 pieces, len at least the
// workgroups' even share of all blocks.
inline long long pre_tiles(int B, int n_groups, int rep, int C) { return (long long)B * rep / (16 * C) + std::min(B, n_groups); }
inline long long pre_slots(int B, int n_groups, int rep, int n_kv, int C) {
  return PRE_WGS + pre_tiles(B, n_groups, rep, C) * n_kv;
}
inline size_t pre_bytes(int B, int n_groups, int rep, int n_kv, int dv) {
  const int C = pre_tile(B, n_groups, rep);
  return (size_t)pre_slots(B, n_groups, rep, n_kv, C) * 16 * C * (dv + 2) * sizeof(float) + (size_t)B * sizeof(RowPrefix);
}

template <int L, int NB, int C>
__global__ __launch_bounds__(256, 2) void palu_prefix_kernel(const StepArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[L == PALU_LAYOUT_ROWS ? step_lds<L, NB>() : WaveLds<NB>::bytes(16)];
  const WaveLds<NB> lds{reinterpret_cast<float*>(smem), 16};
  __shared__ int scan[8], found[4], bases[256];
  constexpr int COLS = 16 * C;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = (a.n_groups + 255) / 256, g0 = min(tid * per, a.n_groups), g1 = min(g0 + per, a.n_groups);
  auto tiles_of = [&](const Group& g) { return g.blocks ? (g.rows * a.rep + COLS - 1) / COLS * a.n_kv : 0; };   // of all KV heads
  // What a lone row shares with itself is read here too if it is no more than the larger groups' blocks: the second launch would
  // have a few workgroups busy with it when all others are done (64 rows in 16 groups, one of them of a single row, over up to
  // 2048 positions: 40 -> 31 us for both launches). Otherwise that launch is the better place, which reads past the caches.
  Group own{0, 0, 0};                     // a thread's only group
  float of_lone = 0.f, of_larger = 0.f;
  for (int i = g0; i < g1; ++i) {
    own = group_of(a, i, true);
    (own.rows > 1 ? of_larger : of_lone) += (float)tiles_of(own) * (float)own.blocks;
  }
  wg_sum2(of_lone, of_larger, reinterpret_cast<float*>(scan));
  const bool lone = of_lone <= of_larger;
  if (!lone && own.rows == 1) own.blocks = 0;
  auto group = [&](int i) { return per == 1 ? own : group_of(a, i, lone); };
  const Cut cut = cut_items(of_larger + (lone ? of_lone : 0.f), g0, g1, PRE_WGS, PRE_LEAST, true, scan, [&](int i) {
    const Group g = group(i);
    return Items{tiles_of(g), g.blocks};
  });
  const int row_wgs = (a.B + 255) / 256;
  // The rows' records, a thread each: the last workgroups, which are the first to have no piece.
  const int rec = (int)(gridDim.x - 1 - blockIdx.x), b = rec * 256 + tid;
  if (rec < row_wgs) {                    // (uniform)
    bases[tid] = cut.before;
    __syncthreads();
  }
  if (rec < row_wgs && b < a.B) {
    const int gi = last_group(a, b);
    RowPrefix r{b, 1, 0, 0, 0, 0, {}};
    const Group g = group_of(a, gi, lone);
    if (g.blocks && b >= g.row && b < g.row + g.rows) {
      int base = bases[gi / per];
      for (int i = gi / per * per; i < gi; ++i) {
        const Group x = group_of(a, i, lone);
        base += tiles_of(x) * cut.pieces(x.blocks);
      }
      const int pieces = cut.pieces(g.blocks);
      r = RowPrefix{g.row, g.rows, g.blocks, base >= 0 && base + tiles_of(g) * pieces <= a.pre_slots ? pieces : 0, base, b - g.row, {}};
    }
    a.rows[b] = r;
  }
  // (Groups that overlap, where the offsets make no sense, can be more pieces than the workspace was sized for, or than can be
  // counted: those are left out.)
  for (int want = blockIdx.x; want < min(cut.all, a.pre_slots); want += gridDim.x) {   // (uniform)
    __syncthreads();                      // the piece before is done with LDS
    if (tid == 0) found[0] = -1;
    __syncthreads();
    if (want >= cut.before && want < cut.before + cut.mine) {
      int at = cut.before;
      for (int i = g0; i < g1; ++i) {
        const Group g = group(i);
        const int n = tiles_of(g) * cut.pieces(g.blocks);
        if (want >= at && want < at + n) {
          found[0] = want - at;
          found[1] = g.row;
          found[2] = g.rows;
          found[3] = g.blocks;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
    const int in = __builtin_amdgcn_readfirstlane(found[0]);
    if (in < 0) continue;                   // (uniform)
    const Group g{uniform(found[1]), uniform(found[2]), uniform(found[3])};
    const int pieces = uniform(cut.pieces(g.blocks)), tile = uniform(in / pieces), piece = in - tile * pieces;
    const int ct = uniform(tile / a.n_kv), kvh = tile - ct * a.n_kv;
    const int each = uniform((g.blocks + pieces - 1) / pieces), lo = piece * each, hi = min(g.blocks, lo + each);
    Wave<L, NB, C> st;
    st.clear();
#pragma unroll
    for (int x = 0; x < C; ++x) {
      const int col = min(ct * COLS + 16 * x + (lane & 15), g.rows * a.rep - 1);    // (those past the group repeat its last)
      const int row = col / a.rep;
      st.query(x, a.q + ((long long)(g.row + row) * a.n_q + kvh * a.rep + (col - row * a.rep)) * HD, a.qscale < 0.f);
    }
    const int lead = lead_of(a, g.row, g.rows);
    auto page_at = [&](int blk) __attribute__((always_inline)) { return page_of(a, lead, blk); };
    auto where = [&](int page, int blk, const char*& k, const char*& v) __attribute__((always_inline)) {
      place_of(a, page, kvh, blk, k, v);
    };
    if constexpr (L == PALU_LAYOUT_ROWS) {  // (V's operands are gathered: out of LDS)
      st.template pass<true>(lo + w * step_group(L), 4, hi, 32 * g.blocks, fabsf(a.qscale), a.dv, smem + w * place_bytes<L, NB>(),
                             page_at, where);
    } else {
      st.template pass_direct<4>(lo, hi, fabsf(a.qscale), a.dv, page_at, where);
    }
    float* po = a.pre + (long long)want * COLS * (a.dv + 2);
    const int vecs = a.dv / 4;
#pragma unroll
    for (int x = 0; x < C; ++x) {
      __syncthreads();                      // every wave is done with its places, or with the results before
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
}

// ---- launches -----------------------------------------------------------------------------------
template <typename K>
int step_launch(K kern, unsigned grid, int lds, const StepArgs& a, const char* who, hipStream_t s) {
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), lds, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
}

template <int L, int NB>
int step_run_nb(const StepArgs& a, const char* who, hipStream_t s) {
  if (a.rows) {
    const int rc = a.pre_cols == 16   ? step_launch(palu_prefix_kernel<L, NB, 1>, PRE_WGS, 0, a, who, s)
                                      : step_launch(palu_prefix_kernel<L, NB, 2>, PRE_WGS, 0, a, who, s);
    if (rc) return rc;
  }
  const unsigned grid = (unsigned)step_grid(a.B, a.n_kv);
  return step_many(a.B, a.n_kv) ? step_launch(palu_step_kernel<L, NB, true>, grid, 0, a, who, s)
                                : step_launch(palu_step_kernel<L, NB, false>, grid, 0, a, who, s);
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
