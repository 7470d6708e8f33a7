// Causal attention of packed sequences of different lengths over full K and V, the prompt's counterpart of the stock
// flash-decode (palu_flash_decode): new row i of sequence b stands at position p = start_b + i and sees keys 0 .. p,
//   out[row][h] = sum_t softmax_t(scale q[row][h] . k[t][j]) v[t][j],   j = h / (n_q / n_kv),
// K and V either the packed rows themselves (start 0) or page pools, row-major or in the caches' tile order.
//
// One pass over the keys per tile of queries. The rows of a tile are (position, head of the KV group) pairs of one
// sequence and one KV head, position-major: the heads of a group share every K and V tile, and a tile of 128 rows is 128 / rep
// positions tall, so that little of its last key tiles lies past the diagonal. A workgroup's 4 waves take 32 rows
// each and share 64-key tiles of K and V in LDS, copied straight there (global_load_lds) one tile ahead.
//   S^T (keys x rows) = K Q^T, Q the B operand of v_mfma_f32_32x32x16_bf16, in registers for the whole pass;
//   P^T = 2^(S^T - m), the running maximum m refreshed when a score exceeds it by more than 2^8;
//   O^T (dims x rows) += V^T P^T.
// The K operand's rows are the keys in the order of the caches' K tiles: the accumulators then leave a lane with
// keys 8 g .. + 7 in pairs of registers, which is the B operand of the second product, and no value changes lanes.
// V^T comes from the caches' V tiles as it stands, from rows by transposing LDS reads (ds_read_b64_tr_b16).
//
// Rounding: scores, statistics and sums are fp32 (products of bf16 are exact in them); the probabilities are rounded to
// bf16 for the second product, half a step of 2^-9 of each, less in their weighted sum than the output's own rounding.
#include "palu_kernel.h"

#include <algorithm>

namespace {

constexpr int FP_ROWS = 128;              // rows of a tile: 4 waves of 32
constexpr int FP_KEYS = 64;               // keys of a K / V tile: two 32-position blocks
constexpr int FP_MIN_SPLIT = 4;           // key tiles of a split, at least
constexpr int FP_WGS = 512;               // workgroups that the chip holds at once (two a CU)

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

enum Source { PACKED, PAGED_ROWS, PAGED_TILED };

struct FlashPrefillArgs {
  const __bf16* q;
  long long q_st, q_sh;                   // element strides: row, head
  const __bf16* k;
  const __bf16* v;
  long long k_st, k_sh, v_st, v_sh;       // packed: row and head strides; pools: page and head strides
  const int32_t* cu;                      // [B + 1] first packed row of every sequence
  const int32_t* start;                   // [B] position of its first row, or null (0)
  const int32_t* page_table;              // [B][pt_stride]
  int pt_stride, n_pages, page_shift, capacity;
  int T, B, n_q, n_kv, rep, dv;
  float qscale;                           // |scale| * log2 e (1 for a scale of 0: a masked score times 0 would be NaN)
  int sign;                               // of the scale: -1, 0, 1; Q is taken times that
  __bf16* out;                            // [T][n_q][dv]
  int nsplit;                             // parts that the keys of a tile may be split into
  float* part;                            // nsplit > 1: unnormalised O of every (item, split) [FP_ROWS][dv], then m and l [FP_ROWS] each
};

// Key tiles first .. last of split s of an item of nt key tiles, and how many splits that item has.
__device__ __forceinline__ int split_tiles(int nt, int nsplit) { return max(FP_MIN_SPLIT, (nt + nsplit - 1) / nsplit); }

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The packed rows of sequence b, whatever cu holds: [beg, beg + len) inside [0, T).
struct Seq {
  int beg, len, start;
};
__device__ __forceinline__ Seq lane_seq(const FlashPrefillArgs& a, int b) {
  const int c0 = a.cu[b], c1 = a.cu[b + 1];
  const int beg = min(max(c0, 0), a.T), end = min(max(c1, beg), a.T);
  const int s = a.start ? a.start[b] : 0;
  return Seq{beg, end - beg, min(max(s, -(1 << 24)), 1 << 24)};
}

// Work order: all tiles of the batch, those with the most keys first, so that the last ones to run are short. A tile's
// level is its distance from position 0 in tiles, rounded down; item w of the descending order is found by halving over
// levels, each lane counting the tiles of one sequence (all waves do it, without a barrier).
struct Tile {
  int b, j;                               // j: tile of sequence b; b < 0: none
};
__device__ __forceinline__ Tile find_tile(const FlashPrefillArgs& a, int w) {
  const int lane = threadIdx.x & 63;
  const int per = FP_ROWS / a.rep > 0 ? FP_ROWS / a.rep : 1;
  auto seq_levels = [&](int b, int& base, int& n) {
    const Seq s = lane_seq(a, min(b, a.B - 1));
    n = b < a.B ? (int)(((long long)s.len * a.rep + FP_ROWS - 1) / FP_ROWS) : 0;
    base = max(s.start, 0) / per;
  };
  int base0, n0;
  seq_levels(lane, base0, n0);            // the first 64 sequences stay in registers
  auto count = [&](int t, int& top) {     // tiles at level t or above; top: one past the highest level
    int c = min(max(base0 + n0 - t, 0), n0), hi = n0 ? base0 + n0 : 0;
    for (int b0 = 64; b0 < a.B; b0 += 64) {
      int base, n;
      seq_levels(b0 + lane, base, n);
      c += min(max(base + n - t, 0), n);
      hi = max(hi, n ? base + n : 0);
    }
    top = hi;
    return wave_sum_i(c);
  };
  int top;
  if (w >= count(0, top)) return Tile{-1, 0};
#pragma unroll
  for (int o = 32; o; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
  int lo = 0, hi = __builtin_amdgcn_readfirstlane(top), unused;   // count(lo) > w, count(hi) = 0 <= w
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (count(mid, unused) > w) lo = mid;
    else hi = mid;
  }
  int r = w - count(lo + 1, unused);      // which of the sequences that have level lo
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int base = base0, n = n0;
    if (b0) seq_levels(b0 + lane, base, n);
    const unsigned long long m = __ballot(n > 0 && base <= lo && lo < base + n);
    const int c = __popcll(m);
    if (r < c) {
      const int before = __popcll(m & ((1ull << lane) - 1));
      const unsigned long long me = __ballot(((m >> lane) & 1) && before == r);
      const int l = __builtin_ctzll(me);
      return Tile{b0 + l, lo - __builtin_amdgcn_readlane(base, l)};
    }
    r -= c;
  }
  return Tile{-1, 0};
}

// dv = V width (a multiple of 16), DV32 its 32-wide tiles; row-major V rows stand DVP wide in LDS.
template <Source SRC, int DV32>
__global__ __launch_bounds__(256, 2) void palu_flash_prefill_kernel(const FlashPrefillArgs a) {
  constexpr bool TILED = SRC == PAGED_TILED;
  constexpr int DVP = DV32 == 3 && !TILED ? 128 : 32 * DV32;
  constexpr int CPR = DVP / 8;            // 16-byte chunks of a V row
  constexpr int VI = DVP / 32;            // 1 KB copies of V per wave and tile
  // One array per stage: the compiler then knows that a copy into one stage is no store to the stage being read.
  __shared__ __attribute__((aligned(1024))) __bf16 sk0[FP_KEYS * HD], sk1[FP_KEYS * HD], sv0[FP_KEYS * DVP], sv1[FP_KEYS * DVP];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // A KV head's workgroups are n_kv ids apart, for 8 heads all on one XCD, whose L2 then holds that head's K and V.
  const int kvh = blockIdx.x % a.n_kv;
  const int item = blockIdx.x / a.n_kv / a.nsplit, split = blockIdx.x / a.n_kv - item * a.nsplit;
  const Tile tile = find_tile(a, item);
  if (tile.b < 0) return;                 // uniform, before any barrier
  Seq sq = lane_seq(a, tile.b);
  sq.beg = __builtin_amdgcn_readfirstlane(sq.beg);
  sq.len = __builtin_amdgcn_readfirstlane(sq.len);
  sq.start = __builtin_amdgcn_readfirstlane(sq.start);
  const int rows = sq.len * a.rep, row0 = tile.j * FP_ROWS, last_row = min(row0 + FP_ROWS, rows) - 1;
  auto key_pos = [&](int row) { return min(sq.start + row / a.rep, a.capacity - 1); };
  const int kv_end = key_pos(last_row) + 1;               // keys of this workgroup
  const int row = min(row0 + 32 * w + n, rows - 1);       // rows past the sequence repeat its last, unstored
  const int ri = row / a.rep, pos = key_pos(row);
  const long long head = (long long)kvh * a.rep + (row - ri * a.rep);
  const int w_lo = __builtin_amdgcn_readfirstlane(key_pos(min(row0 + 32 * w, rows - 1)));
  const int w_hi = row0 + 32 * w >= rows ? -1             // a wave without rows copies only
                                         : __builtin_amdgcn_readfirstlane(key_pos(min(row0 + 32 * w + 31, rows - 1)));
  const int nt_all = kv_end > 0 ? (kv_end + FP_KEYS - 1) / FP_KEYS : 0;
  const int per_split = split_tiles(nt_all, a.nsplit);
  const int t_lo = split * per_split, nt = min(nt_all, t_lo + per_split);
  if (t_lo >= nt && split > 0) return;    // uniform

  // ---- copies to LDS ------------------------------------------------------------------------
  const int32_t* pt = SRC == PACKED ? nullptr : a.page_table + (long long)tile.b * a.pt_stride;
  auto page_of = [&](int t, int blk) {                    // page of block blk of tile t (past the end: the last block's)
    if constexpr (SRC == PACKED) return 0;
    const int p = load_uniform(pt, min(2 * t + blk, (kv_end - 1) >> 5) >> a.page_shift);
    return min(max(p, 0), a.n_pages - 1);
  };
  const int last_blk = (kv_end - 1) >> 5;
  const __bf16* kh = a.k + (long long)kvh * a.k_sh + (SRC == PACKED ? (long long)sq.beg * a.k_st : 0);
  const __bf16* vh = a.v + (long long)kvh * a.v_sh + (SRC == PACKED ? (long long)sq.beg * a.v_st : 0);
  auto copy_tile = [&](__bf16* sk, __bf16* sv, int t, int p0, int p1) __attribute__((always_inline)) {
    if constexpr (TILED) {
      const int inpage = (1 << a.page_shift) - 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {                       // kilobyte 4 w + i of the tile: block w / 2
        const int blk = min(2 * t + (w >> 1), last_blk);
        const __bf16* src = kh + (long long)(w >> 1 ? p1 : p0) * a.k_st + (long long)(blk & inpage) * (BLK * HD) +
                            ((w & 1) * 4 + i) * 512 + lane * 8;
        __builtin_amdgcn_global_load_lds((gvoid*)src, (lvoid*)(sk + (4 * w + i) * 512), 16, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < DV32; ++i) {
        const int c = w * DV32 + i, b = c / (2 * DV32), mt = min(c - b * 2 * DV32, a.dv / 16 - 1);
        const int blk = min(2 * t + b, last_blk);
        const __bf16* src = vh + (long long)(b ? p1 : p0) * a.v_st + (long long)(blk & inpage) * (BLK * a.dv) + mt * 512 + lane * 8;
        __builtin_amdgcn_global_load_lds((gvoid*)src, (lvoid*)(sv + c * 512), 16, 0, 0);
      }
    } else {
      // Row r of the tile in memory: packed, clamped to the last key; in pages, a row of its block's page.
      auto row_at = [&](const __bf16* base, long long st, long long pst, int width, int r) {
        if constexpr (SRC == PACKED) return base + (long long)min(t * FP_KEYS + r, kv_end - 1) * st;
        const int blk = min(2 * t + (r >> 5), last_blk);
        const int in = ((blk & ((1 << a.page_shift) - 1)) << 5) + (r & 31);
        return base + (long long)(r >> 5 ? p1 : p0) * pst + in * width;
      };
      // 16-byte chunks of a row are permuted by the row, so that the reads below meet all banks.
#pragma unroll
      for (int i = 0; i < 4; ++i) {                       // rows 4 (4 w + i) .. + 3
        const int r = 4 * (4 * w + i) + (lane >> 4);
        const int c = (lane & 15) ^ (4 * ((r >> 3) & 3) + (r & 3));
        __builtin_amdgcn_global_load_lds((gvoid*)(row_at(kh, a.k_st, a.k_st, HD, r) + 8 * c), (lvoid*)(sk + (4 * w + i) * 512), 16, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int e = (VI * w + i) * 64 + lane, r = e / CPR;
        const int g = CPR == 16 ? 2 * (r & 3) + ((r >> 2) & 1) : CPR == 8 ? 2 * ((r >> 1) & 1) : 0;
        const int c = min((e % CPR) ^ (2 * g), a.dv / 8 - 1);
        __builtin_amdgcn_global_load_lds((gvoid*)(row_at(vh, a.v_st, a.v_st, a.dv, r) + 8 * c), (lvoid*)(sv + (VI * w + i) * 512), 16, 0, 0);
      }
    }
  };

  // ---- operands from LDS --------------------------------------------------------------------
  const int c16 = n >> 4, nn = n & 15;
  int kaddr[TILED ? 1 : 8];                               // byte offsets of a lane's K operand, dim block kk
  if constexpr (TILED) {
    kaddr[0] = c16 * 4096 + h * 256 + nn * 16;
  } else {
    const int p = 8 * (nn >> 2) + 4 * c16 + (nn & 3);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) kaddr[kk] = p * 256 + (((2 * kk + h) ^ nn) * 16);
  }
  auto read_k = [&](const __bf16* sk, int blk, int kk) {
    const char* base = reinterpret_cast<const char*>(sk) + blk * 8192;
    if constexpr (TILED) return *reinterpret_cast<const bf16x8*>(base + kaddr[0] + (kk >> 1) * 1024 + (kk & 1) * 512);
    else return *reinterpret_cast<const bf16x8*>(base + kaddr[kk]);
  };
  // V^T operand of dims 32 md .. + 31 and keys 32 blk + 16 t .. + 15: lane (n, h) holds keys 8 (2 t + h) .. + 7 of a dim.
  int vaddr[TILED ? 1 : 2 * DV32];
  if constexpr (TILED) {
    vaddr[0] = c16 * 1024 + h * 256 + nn * 16;
  } else {
    // a 16-lane group reads 4 keys of 16 dims and gets, per lane, the 4 keys of one dim
    const int r = 8 * h + ((lane & 15) >> 2);
#pragma unroll
    for (int md = 0; md < DV32; ++md)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int rr = r + 4 * u, pr = 2 * md + ((lane >> 4) & 1);
        const int g = CPR == 16 ? 2 * (rr & 3) + ((rr >> 2) & 1) : CPR == 8 ? 2 * ((rr >> 1) & 1) : 0;
        vaddr[2 * md + u] = rr * (2 * DVP) + ((pr ^ g) * 32) + 8 * (lane & 3);
      }
  }
  auto read_v = [&](const __bf16* sv, int blk, int t, int md) {
    const char* base = reinterpret_cast<const char*>(sv);
    if constexpr (TILED) {
      return *reinterpret_cast<const bf16x8*>(base + vaddr[0] + blk * (DV32 * 2048) + md * 2048 + t * 512);
    } else {
      base += (32 * blk + 16 * t) * (2 * DVP);
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(base + vaddr[2 * md]));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(base + vaddr[2 * md + 1]));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };

  // ---- state ----------------------------------------------------------------------------------
  bf16x8 q[8];
  {
    const __bf16* qp = a.q + (sq.beg + ri) * a.q_st + head * a.q_sh + 8 * h;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      q[kk] = *reinterpret_cast<const bf16x8*>(qp + 16 * kk);
      if (a.sign < 0) q[kk] = -q[kk];
      if (a.sign == 0) q[kk] = bf16x8{};
    }
  }
  f32x16 O[DV32];
#pragma unroll
  for (int md = 0; md < DV32; ++md)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[md][i] = 0.f;
  float m_run = NEG_INF, l_run = 0.f;

  auto step = [&](const __bf16* sk, const __bf16* sv, int t) __attribute__((always_inline)) {
    const int base = t * FP_KEYS;
    if (base > w_hi) return;                              // uniform per wave: keys past all its rows
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = mfma32(read_k(sk, b, kk), q[kk], s[b]);
    const bool masked = base + FP_KEYS - 1 > w_lo;
    if (masked) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = i >> 2, key = base + 32 * b + 8 * (2 * (j & 1) + h) + 4 * (j >> 1) + (i & 3);
          if (key > pos) s[b][i] = NEG_INF;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, s[b][i]);
    mx *= a.qscale;
    if (__any(mx > m_run + LAZY_RESCALE_LOG2)) {
      // Rows refresh by their own scores alone, so that a row's roundings do not depend on its neighbours'.
      const float top = fmaxf(mx, __shfl_xor(mx, 32, 64)), mn = top > m_run + LAZY_RESCALE_LOG2 ? top : m_run;
      const float alpha = m_run == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(m_run - mn);
#pragma unroll
      for (int md = 0; md < DV32; ++md)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[md][i] *= alpha;
      l_run *= alpha;
      m_run = mn;
    }
    const float mref = m_run == NEG_INF ? 0.f : m_run;
    bf16x8 p[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(s[b][4 * tt + 8 * (i >> 2) + (i & 3)], a.qscale, -mref));
          p[b][tt][i] = (__bf16)e[i];
        }
        l_run += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
      }
    if (masked) {
      // A key that some rows do not see may hold an infinity or NaN in V, and 0 times that is NaN: such a tile (rare) is
      // added one key at a time, to the rows that see it.
      float bad = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int md = 0; md < DV32; ++md) {
            const bf16x8 v = read_v(sv, b, tt, md);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              bad = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[2 * i], v[2 * i + 1]}, bf16x2{(__bf16)0.f, (__bf16)0.f}, bad, false);
          }
      if (__any(bad != bad)) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
            for (int x = 0; x < 16; ++x) {
              const int key = base + 32 * b + 16 * tt + x;
              if (key > w_hi) break;
#pragma unroll
              for (int md = 0; md < DV32; ++md) {
                bf16x8 v = read_v(sv, b, tt, md);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 8 * h + i == x ? v[i] : (__bf16)0.f;
                const f32x16 y = mfma32(v, p[b][tt], O[md]);
#pragma unroll
                for (int i = 0; i < 16; ++i) O[md][i] = key <= pos ? y[i] : O[md][i];
              }
            }
        return;
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int md = 0; md < DV32; ++md) O[md] = mfma32(read_v(sv, b, tt, md), p[b][tt], O[md]);
  };
  // A tile's copies are asked for while the one before it is computed; past the wait and the barrier they have arrived in
  // every wave, and every wave is done with the stage that the next copies overwrite.
  auto turn = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  if (t_lo < nt) {
    int a0 = page_of(t_lo, 0), a1 = page_of(t_lo, 1);
    copy_tile(sk0, sv0, t_lo, a0, a1);
    a0 = page_of(t_lo + 1, 0), a1 = page_of(t_lo + 1, 1);
    for (int t = t_lo; t < nt; t += 2) {
      turn();
      if (t + 1 < nt) copy_tile(sk1, sv1, t + 1, a0, a1);
      a0 = page_of(t + 2, 0), a1 = page_of(t + 2, 1);
      step(sk0, sv0, t);
      turn();
      if (t + 1 >= nt) break;
      if (t + 2 < nt) copy_tile(sk0, sv0, t + 2, a0, a1);
      a0 = page_of(t + 3, 0), a1 = page_of(t + 3, 1);
      step(sk1, sv1, t + 1);
    }
  }

  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (row0 + 32 * w + n >= rows) return;
  if (nt_all > per_split) {               // one of several splits
    const long long slot = ((long long)item * a.n_kv + kvh) * a.nsplit + split;
    float* po = a.part + slot * FP_ROWS * (a.dv + 2);
    const int r = 32 * w + n;
    if (h == 0) {
      po[FP_ROWS * a.dv + r] = m_run;
      po[FP_ROWS * (a.dv + 1) + r] = l;
    }
#pragma unroll
    for (int md = 0; md < DV32; ++md)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * md + 8 * j < a.dv)
          *reinterpret_cast<f32x4*>(po + r * a.dv + 32 * md + 8 * j + 4 * h) =
              f32x4{O[md][4 * j], O[md][4 * j + 1], O[md][4 * j + 2], O[md][4 * j + 3]};
    return;
  }
  const float inv = 1.f / l;
  __bf16* o = a.out + ((long long)(sq.beg + ri) * a.n_q + head) * a.dv + 4 * h;
#pragma unroll
  for (int md = 0; md < DV32; ++md)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (32 * md + 8 * j < a.dv) {
        bf16x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pos < 0 ? (__bf16)0.f : (__bf16)(O[md][4 * j + i] * inv);
        *reinterpret_cast<bf16x4*>(o + 32 * md + 8 * j) = x;
      }
    }
}

// Joins the splits of an item: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. One workgroup per (item, KV head, 32 rows),
// eight threads to a row.
__global__ __launch_bounds__(256) void palu_flash_prefill_join_kernel(const FlashPrefillArgs a) {
  const int kvh = blockIdx.x % a.n_kv, rest = blockIdx.x / a.n_kv, item = rest >> 2;
  const Tile tile = find_tile(a, item);
  if (tile.b < 0) return;
  const Seq sq = lane_seq(a, tile.b);
  const int rows = sq.len * a.rep, row0 = tile.j * FP_ROWS;
  const int last = min(sq.start + (min(row0 + FP_ROWS, rows) - 1) / a.rep, a.capacity - 1);
  const int nt = last >= 0 ? last / FP_KEYS + 1 : 0, per = split_tiles(nt, a.nsplit);
  const int r = (rest & 3) * 32 + (threadIdx.x >> 3), row = row0 + r;
  if (nt <= per || row >= rows) return;
  const int ns = (nt + per - 1) / per, ri = row / a.rep;
  const long long stride = (long long)FP_ROWS * (a.dv + 2);
  const float* part = a.part + ((long long)item * a.n_kv + kvh) * a.nsplit * stride;
  const float* ml = part + FP_ROWS * a.dv + r;
  float M = NEG_INF, l = 0.f;
  for (int s = 0; s < ns; ++s) M = fmaxf(M, ml[s * stride]);
  const float ref = M == NEG_INF ? 0.f : M;
  for (int s = 0; s < ns; ++s) l += __builtin_amdgcn_exp2f(ml[s * stride] - ref) * ml[s * stride + FP_ROWS];
  const float inv = 1.f / l;
  __bf16* o = a.out + ((long long)(sq.beg + ri) * a.n_q + (long long)kvh * a.rep + (row - ri * a.rep)) * a.dv;
  for (int d = 4 * (threadIdx.x & 7); d < a.dv; d += 32) {
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ns; ++s)
      y += *reinterpret_cast<const f32x4*>(part + s * stride + r * a.dv + d) * __builtin_amdgcn_exp2f(ml[s * stride] - ref);
    bf16x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = sq.start + ri < 0 ? (__bf16)0.f : (__bf16)(y[i] * inv);
    *reinterpret_cast<bf16x4*>(o + d) = x;
  }
}

// Tiles of a batch, at most: a sequence's last tile may hold fewer rows.
long long most_tiles(int T, int B, int rep) { return (long long)T * rep / FP_ROWS + std::min(T, B); }

// Splits per tile: enough workgroups for the chip where the tiles are few, none of them under FP_MIN_SPLIT key tiles.
int split_count(int T, int B, int n_q, int n_kv, long long max_keys) {
  const long long items = most_tiles(T, B, n_q / n_kv) * n_kv;
  return (int)std::max<long long>(1, std::min<long long>(FP_WGS / items, max_keys / (FP_MIN_SPLIT * FP_KEYS)));
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t part_bytes(int T, int B, int n_q, int n_kv, long long max_keys, int dv) {
  const int ns = split_count(T, B, n_q, n_kv, max_keys);
  return ns == 1 ? 0 : (size_t)most_tiles(T, B, n_q / n_kv) * n_kv * ns * FP_ROWS * (dv + 2) * sizeof(float);
}

int check_dims(int T, int B, int n_q, int n_kv, int dv, const char* who) {
  if (T <= 0 || B <= 0 || n_q <= 0 || n_kv <= 0)
    return fail(PALU_EINVAL, "%s: row, sequence and head counts must be positive, got %d, %d, %d, %d", who, T, B, n_q, n_kv);
  if (n_q % n_kv) return fail(PALU_EINVAL, "%s: n_q = %d must be a multiple of the KV head count %d", who, n_q, n_kv);
  if (dv < 16 || dv > HD || dv % 16)
    return fail(PALU_EUNSUPPORTED, "%s: head_dim_v %d (multiples of 16 up to %d)", who, dv, HD);
  if ((long long)T * n_q > (1ll << 30) || (long long)B > (1 << 24))
    return fail(PALU_EUNSUPPORTED, "%s: %d rows of %d heads in %d sequences exceed the grid", who, T, n_q, B);
  return PALU_OK;
}

template <Source SRC>
int launch_prefill(FlashPrefillArgs& a, long long max_keys, void* workspace, size_t workspace_bytes, const char* who, hipStream_t s) {
  a.nsplit = split_count(a.T, a.B, a.n_q, a.n_kv, max_keys);
  const size_t need = part_bytes(a.T, a.B, a.n_q, a.n_kv, max_keys, a.dv);
  if (need && (!workspace || workspace_bytes < need || !al16(workspace)))
    return fail(PALU_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes needed (palu_flash_prefill_workspace_bytes), got %zu", who,
                need, workspace ? workspace_bytes : 0);
  a.part = static_cast<float*>(workspace);
  const unsigned items = (unsigned)(most_tiles(a.T, a.B, a.rep) * a.n_kv);
  auto go = [&](auto kern, unsigned grid) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
  };
  int rc = PALU_OK;
  switch ((a.dv + 31) / 32) {
    case 1: rc = go(palu_flash_prefill_kernel<SRC, 1>, items * a.nsplit); break;
    case 2: rc = go(palu_flash_prefill_kernel<SRC, 2>, items * a.nsplit); break;
    case 3: rc = go(palu_flash_prefill_kernel<SRC, 3>, items * a.nsplit); break;
    default: rc = go(palu_flash_prefill_kernel<SRC, 4>, items * a.nsplit); break;
  }
  if (rc == PALU_OK && a.nsplit > 1) rc = go(palu_flash_prefill_join_kernel, items * 4);
  return rc;
}

bool stride_ok(long long st, long long least) { return st >= least && st % 8 == 0; }

}  // namespace

extern "C" size_t palu_flash_prefill_workspace_bytes(int rows, int batch, int n_q, int n_kv, int max_keys, int head_dim_v) {
  palu::g_err[0] = 0;
  if (max_keys <= 0 || check_dims(rows, batch, n_q, n_kv, head_dim_v, "palu_flash_prefill_workspace_bytes")) return 0;
  return part_bytes(rows, batch, n_q, n_kv, max_keys, head_dim_v);
}

extern "C" int palu_flash_prefill(const void* q, long long q_row_stride, long long q_head_stride, const void* k,
                                  long long k_row_stride, long long k_head_stride, const void* v, long long v_row_stride,
                                  long long v_head_stride, const int32_t* cu_seqlens, void* out, float scale, int rows,
                                  int batch, int n_q, int n_kv, int head_dim_v, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_flash_prefill";
  if (!q || !k || !v || !cu_seqlens || !out) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  if (int rc = check_dims(rows, batch, n_q, n_kv, head_dim_v, who)) return rc;
  if (!stride_ok(q_row_stride, 0) || !stride_ok(q_head_stride, 0) || !stride_ok(k_row_stride, 0) || !stride_ok(k_head_stride, 0) ||
      !stride_ok(v_row_stride, 0) || !stride_ok(v_head_stride, 0))
    return fail(PALU_EINVAL, "%s: strides must be non-negative multiples of 8", who);
  if (!al16(q) || !al16(k) || !al16(v) || !al16(out)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  FlashPrefillArgs a{static_cast<const __bf16*>(q), q_row_stride, q_head_stride, static_cast<const __bf16*>(k),
                     static_cast<const __bf16*>(v), k_row_stride, k_head_stride, v_row_stride, v_head_stride, cu_seqlens, nullptr,
                     nullptr, 0, 0, 0, 0x7fffffff, rows, batch, n_q, n_kv, n_q / n_kv, head_dim_v,
                     scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f, (scale > 0.f) - (scale < 0.f),
                     static_cast<__bf16*>(out), 1, nullptr};
  return launch_prefill<PACKED>(a, rows, workspace, workspace_bytes, who, stream);
}

extern "C" int palu_flash_prefill_paged(const void* q, long long q_row_stride, long long q_head_stride, const void* k_pages,
                                        const void* v_pages, const int32_t* cu_seqlens, const int32_t* start_pos,
                                        const int32_t* page_table, void* out, float scale, int rows, int batch, int n_q,
                                        int n_kv, int num_pages, int page_size, int max_pages_per_seq, int head_dim_v,
                                        int cache_layout, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_flash_prefill_paged";
  if (!q || !k_pages || !v_pages || !cu_seqlens || !out) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  int shift = 0;
  if (int rc = palu::check_pages(page_table, num_pages, page_size, max_pages_per_seq, &shift, who)) return rc;
  if (int rc = check_dims(rows, batch, n_q, n_kv, head_dim_v, who)) return rc;
  if (cache_layout != PALU_LAYOUT_ROWS && cache_layout != PALU_LAYOUT_TILED)
    return fail(PALU_EINVAL, "%s: cache layout must be PALU_LAYOUT_ROWS or PALU_LAYOUT_TILED, got %d", who, cache_layout);
  if (!stride_ok(q_row_stride, 0) || !stride_ok(q_head_stride, 0))
    return fail(PALU_EINVAL, "%s: strides must be non-negative multiples of 8", who);
  if (!al16(q) || !al16(k_pages) || !al16(v_pages) || !al16(out)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  const long long k_sh = (long long)page_size * HD, v_sh = (long long)page_size * head_dim_v;
  const int capacity = max_pages_per_seq * page_size;
  FlashPrefillArgs a{static_cast<const __bf16*>(q), q_row_stride, q_head_stride, static_cast<const __bf16*>(k_pages),
                     static_cast<const __bf16*>(v_pages), k_sh * n_kv, k_sh, v_sh * n_kv, v_sh, cu_seqlens, start_pos, page_table,
                     max_pages_per_seq, num_pages, shift, capacity, rows, batch, n_q, n_kv, n_q / n_kv, head_dim_v,
                     scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f, (scale > 0.f) - (scale < 0.f),
                     static_cast<__bf16*>(out), 1, nullptr};
  if (cache_layout == PALU_LAYOUT_TILED) return launch_prefill<PAGED_TILED>(a, capacity, workspace, workspace_bytes, who, stream);
  return launch_prefill<PAGED_ROWS>(a, capacity, workspace, workspace_bytes, who, stream);
}
