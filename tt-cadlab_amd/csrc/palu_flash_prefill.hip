// Causal attention of packed sequences of different lengths over full K and V, the prompt's counterpart of the stock
// flash-decode (palu_flash_decode): new row i of sequence b stands at position p = start_b + i and sees keys 0 .. p,
//   out[row][h] = sum_t softmax_t(scale q[row][h] . k[t][j]) v[t][j],   j = h / (n_q / n_kv),
// K and V either the packed rows themselves (start 0) or page pools, row-major or in the caches' tile order.
//
// One pass over the keys per tile of queries. The rows of a tile are (position, head of the KV group) pairs of one
// sequence and one KV head, position-major: the heads of a group share every K and V tile, and a tile of 128 rows is
// 128 / rep positions tall, so that little of its last key tiles lies past the diagonal. A workgroup's 4 waves take 32 rows
// each and share 64-key tiles of K and V in LDS, copied straight there (global_load_lds), K two tiles ahead and V one.
//   S^T (keys x rows) = K Q^T, Q the B operand of v_mfma_f32_32x32x16_bf16, in registers for the whole pass;
//   P^T = 2^(S^T - m), the running maximum m refreshed when a score exceeds it by more than 2^8;
//   O^T (dims x rows) += V^T P^T.
// The K operand's rows are the keys in the order of the caches' K tiles: the accumulators then leave a lane with
// keys 8 g .. + 7 in pairs of registers, which is the B operand of the second product, and no value changes lanes.
// V^T comes from the caches' V tiles as it stands, from rows by transposing LDS reads (ds_read_b64_tr_b16).
//
// Bound by the matrix cores where sequences are long: they are busy 57 % of a CU's cycles over a prompt of 8192 positions,
// at the 1.65 GHz that the card's power limit leaves; S of the next tile runs beside the exponentials of this one, and two
// workgroups share a CU. 32 query heads over 8 KV heads, widths 128: a prompt of 8192 takes 526 us (1.05 PFLOP/s), of 16384
// 2.02 ms (1.09); 2048 rows behind 30000 positions in pages 0.95 ms (1.09); 64 rows, one behind each of 8000 positions,
// 365 us (5.7 TB/s). Short sequences pay for each tile's search, first loads and masked keys, some 17 thousand cycles together (not
// measured apart) beside 2100 to 2900 per 64 keys: 8 prompts of 2 to 2048 82 us (0.71 PFLOP/s), 128 of 128 127 us. At width
// 128 four to seven registers spill, 20 to 32 bytes a thread.
//
// Rounding: scores, statistics and sums are fp32 (products of bf16 are exact in them); the probabilities are rounded to bf16
// for the second product, by up to 2^-8 of each, and it is the rounded ones that are summed to divide by. So a result is a mean of V
// with weights off by that much: by at most 2^-8 sum_t p_t |v_t - out| before its own rounding to bf16, which is more than the latter
// where values cancel, and nothing where they are equal. (Divided by the sum of the unrounded ones, one dominating key alone
// was off by up to 2^-8; a prompt of 8192 takes 3 % longer for it. A second bf16 plane for what the rounding drops, which
// would leave 2^-16, takes another 37 %.)
#include "palu_kernel.h"

#include <algorithm>

namespace {

constexpr int FP_ROWS = 128;              // rows of a tile: 4 waves of 32
constexpr int FP_KEYS = 64;               // keys of a K / V tile: two 32-position blocks
constexpr int FP_MIN_KEYS = 256;          // keys of a piece of a split tile, about, at least
constexpr int FP_SORTED = 256;            // sequences whose tiles are taken longest first
constexpr int FP_WGS = 512;               // workgroups that the chip holds at once (two a CU)
// Keys of a piece over a workgroup slot's part of the batch's, about, at most. Measured on two batches only: 8 sequences of up to 300
// rows over up to 32000 positions 136 us, with 0.8 175, with 0.55 151; one row over 32000 32, 39 and 43. What counts is how a
// batch's pieces fall on the slots, so no rule follows for others, but that a little over one part each leaves no second turn.
constexpr float FP_PIECE = 1.05f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

enum Source { PACKED, PAGED_ROWS, PAGED_TILED };

// What the join reads of an item: of a tile's first piece the number of pieces and its rows, else 0 pieces.
struct Record {
  int pieces, rows, beg, start, pos0, rem, unused[2];
};

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
  float* part;                            // where keys may be cut: a piece's unnormalised O [FP_ROWS][dv], m, l [FP_ROWS]
  Record* records;                        // of the items that may be pieces: `cut` per KV head
  int cut;
};

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
  const int s = a.start ? a.start[b] : 0;                 // (rows past the capacity see all keys, before 0 none, however far)
  return Seq{beg, end - beg, min(max(s, -(1 << 30)), a.capacity)};
}

// Work order: all tiles of the batch, those with the most keys first, so that the last ones to run are short. A tile's
// level is its distance from position 0 in tiles (of a power of two positions), rounded down; item w of the descending
// order is found by halving over levels, the lanes counting the tiles of up to four sequences each (all waves do it, without
// a barrier; one sequence's is found directly). Batches of more than FP_SORTED sequences are taken sequence by sequence
// instead, in one pass over their lengths.
// Where a.part is given, a tile of level t is cut along its keys into t / len + 3 / 4 pieces (one below 1.25 len), items of
// their own, next to each other: len levels are FP_PIECE times what a workgroup slot gets of the whole batch, so the batch
// is cut only where single tiles are long for it (few new rows over long contexts).
struct Tile {
  int b, j;                               // j: tile of sequence b; b < 0: none
  int piece, pieces;
  Seq seq;
};
__device__ __forceinline__ Tile find_tile(const FlashPrefillArgs& a, int w) {
  constexpr int R = FP_SORTED / 64;
  const int lane = threadIdx.x & 63;
  const int shift = 31 - __builtin_clz(max(1, FP_ROWS / a.rep));
  struct Levels {
    int base, n;
  };
  auto load = [&](int b) {
    const Seq s = lane_seq(a, min(b, a.B - 1));
    return b < a.B ? s : Seq{0, 0, 0};
  };
  auto levels = [&](const Seq& s) { return Levels{max(s.start, 0) >> shift, (s.len * a.rep + FP_ROWS - 1) / FP_ROWS}; };
  auto the_seq = [](const Seq& s, int x) {                // lane x's
    return Seq{__builtin_amdgcn_readlane(s.beg, x), __builtin_amdgcn_readlane(s.len, x), __builtin_amdgcn_readlane(s.start, x)};
  };
  if (a.B > FP_SORTED) {
    int before = 0;
    Seq next = load(lane);
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Seq s = next;
      next = load(b0 + 64 + lane);        // (past the batch: none)
      const int n = levels(s).n, upto = before + wave_scan(n);
      const unsigned long long m = __ballot(w < upto);
      if (m) {
        const int x = __builtin_ctzll(m);
        return Tile{b0 + x, __builtin_amdgcn_readlane(upto, x) - 1 - w, 0, 1, the_seq(s, x)};   // its last tile first
      }
      before = __builtin_amdgcn_readlane(upto, 63);
    }
    return Tile{-1, 0, 0, 1, {}};
  }
  Seq own[R];
  Levels lv[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    own[r] = Seq{0, 0, 0};
    lv[r] = Levels{0, 0};
    if (64 * r < a.B) {
      own[r] = load(64 * r + lane);
      lv[r] = levels(own[r]);
    }
  }
  if (a.B == 1 && !a.part) {              // one sequence: its tiles from the last on
    const Seq s = the_seq(own[0], 0);
    const int n = levels(s).n;
    return Tile{w < n ? 0 : -1, n - 1 - w, 0, 1, s};
  }
  // a sum over all sequences' levels
  auto over_all = [&](auto f) {
    auto x = f(lv[0]);
    if (a.B > 64)
#pragma unroll
      for (int r = 1; r < R; ++r) x += f(lv[r]);
    return x;
  };
  FDiv len = make_fdiv(1 << 30);          // levels of a piece
  if (a.part) {
    float keys = over_all([](Levels l) { return (float)l.n * ((float)l.base + 0.5f * (float)(l.n + 1)); });
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) keys += __shfl_xor(keys, o, 64);
    const float most = fmaxf((float)(FP_MIN_KEYS >> shift), ceilf(keys * (float)a.n_kv * (FP_PIECE / FP_WGS)));
    len = make_fdiv((int)fminf(fmaxf(most, 2.f), 1e9f));
  }
  const int round = len.d - (len.d >> 2) - 1;
  auto pieces_below = [&](int t) {        // of one tile at each of levels 0 .. t - 1
    if (!a.part) return t;
    const int u = t + round, q = fdiv(u, len);            // the sum of u / len, and 1 in place of each 0
    return q * (q - 1) / 2 * len.d + (u - q * len.d) * q + min(t, len.d - round);
  };
  auto count = [&](int t) {               // pieces at level t or above
    return wave_sum_i(over_all([&](Levels l) {
      const int end = l.base + l.n;
      return end > t ? pieces_below(end) - pieces_below(max(l.base, t)) : 0;
    }));
  };
  int top = lv[0].n ? lv[0].base + lv[0].n : 0;            // one past the highest level
  if (a.B > 64)
#pragma unroll
    for (int r = 1; r < R; ++r) top = max(top, lv[r].n ? lv[r].base + lv[r].n : 0);
  int lo = 0, hi = wave_max_i(top), above = 0;            // the level lies in [lo, hi); above = count(hi) <= w
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, c = count(mid);
    if (c > w) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  const int pieces = a.part ? max(1, __builtin_amdgcn_readfirstlane(fdiv(lo + round, len))) : 1;
  int r = w - above;                      // which piece of the sequences that have level lo
  const int piece = r % pieces;
  r /= pieces;
  Tile found{-1, 0, 0, 1, {}};
  auto pick = [&](int b0, const Seq& s) {
    const Levels l = levels(s);
    const unsigned long long m = __ballot(l.n > 0 && l.base <= lo && lo < l.base + l.n);
    const int c = __popcll(m);
    if (r >= 0 && r < c) {
      const unsigned long long me = __ballot(((m >> lane) & 1) && __popcll(m & ((1ull << lane) - 1)) == r);
      const int x = __builtin_ctzll(me);
      found = Tile{b0 + x, lo - __builtin_amdgcn_readlane(l.base, x), piece, pieces, the_seq(s, x)};
    }
    r -= c;
  };
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (64 * k < a.B) pick(64 * k, own[k]);
  return found;
}

// The item of workgroup w (of n per KV head). The first `half` go to a CU each, the next as many beside them: in reverse, so
// that the longest items have the shortest of these for neighbours (one prompt of 2048: 52 us instead of 56).
__device__ __forceinline__ int place(int w, int n, int half) {
  const int upto = min(2 * half, n);
  return w >= half && w < upto ? half + upto - 1 - w : w;
}

// A tile's rows are rows row0 .. of the sequence, row = position * rep + head: position and head of row row0 + x.
struct RowSplit {
  int pos0, rem;
  FDiv rep;
};
__device__ __forceinline__ RowSplit split_rows(int row0, int rep) {
  const int p = (int)((unsigned)row0 / (unsigned)rep);
  return RowSplit{p, row0 - p * rep, make_fdiv(rep)};
}
__device__ __forceinline__ int row_pos(const RowSplit& s, int x) { return s.pos0 + fdiv(s.rem + x, s.rep); }

// dv = V width (a multiple of 16), DV32 its 32-wide tiles; row-major V rows stand DVP wide in LDS.
//
// LDS: K in the order of the caches' K tiles (kilobyte (block, half-block c, dim block kb): slot 16 g + n is key 8 (n / 4) + 4 c +
// n % 4 and dims 32 kb + 8 g .. + 7), V in that of their V tiles or, from rows, in lines of rows 4 apart: the four
// consecutive keys that a transposing read wants are a kilobyte and 64 bytes apart, so that they meet different banks.
template <Source SRC, int DV32>
__global__ __launch_bounds__(256, 2) void palu_flash_prefill_kernel(const FlashPrefillArgs a) {
  constexpr bool TILED = SRC == PAGED_TILED;
  constexpr int DVP = DV32 == 3 && !TILED ? 128 : 32 * DV32;
  constexpr int VI = DVP / 32;            // 1 KB copies of V per wave and tile
  constexpr int VKB = TILED || DVP == 32 ? 1024 : 1088;   // a kilobyte of V and its padding
  // One array per stage: the compiler then knows that a copy into one stage is no store to the stage being read.
  __shared__ __attribute__((aligned(1024))) char sk0[FP_KEYS * HD * 2], sk1[FP_KEYS * HD * 2], sv0[4 * VI * VKB], sv1[4 * VI * VKB];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // A KV head's workgroups are n_kv ids apart, for 8 heads all on one XCD, whose L2 then holds that head's K and V.
  const int kvh = blockIdx.x % a.n_kv;
  const int item = place(blockIdx.x / a.n_kv, gridDim.x / a.n_kv, FP_WGS / 2 / a.n_kv);
  const Tile tile = find_tile(a, item);
  const bool recorded = item < a.cut;
  auto record = [&](const Record& r) {
    if (recorded && threadIdx.x == 0) a.records[item * a.n_kv + kvh] = r;
  };
  if (tile.b < 0) {                       // uniform, before any barrier
    record(Record{});
    return;
  }
  const Seq sq = tile.seq;
  const int row0 = tile.j * FP_ROWS, rows = min(sq.len * a.rep - row0, FP_ROWS);   // rows of this tile
  const RowSplit rs = split_rows(row0, a.rep);
  // the last key that a row sees, of row x of the tile, x uniform
  auto key_pos = [&](int x) { return __builtin_amdgcn_readfirstlane(min(sq.start + row_pos(rs, x), a.capacity - 1)); };
  const int kv_end = key_pos(rows - 1) + 1;               // keys of this workgroup
  const int nt_all = kv_end > 0 ? (kv_end + FP_KEYS - 1) / FP_KEYS : 0;
  const int per_piece = (nt_all + tile.pieces - 1) / tile.pieces;
  const int t_lo = tile.piece * per_piece, nt = min(nt_all, t_lo + per_piece);
  const int n_pieces = nt_all > per_piece ? (nt_all + per_piece - 1) / per_piece : 1;
  // (Sequences that overlap, where the offsets make no sense, can be more tiles than the workspace was sized for.)
  const bool fits = SRC == PACKED || item - tile.piece + n_pieces <= a.cut;
  record(n_pieces > 1 && fits && tile.piece == 0 ? Record{n_pieces, rows, sq.beg, sq.start, rs.pos0, rs.rem, {}} : Record{});
  if ((t_lo >= nt && tile.piece > 0) || (n_pieces > 1 && !fits)) return;   // uniform

  // ---- copies to LDS: wave w copies keys 16 w .. + 15 of a tile (half-block w % 2 of block w / 2 for K) ---------
  const int last_blk = (kv_end - 1) >> 5, inpage = (1 << a.page_shift) - 1;
  const int32_t* pt = SRC == PACKED ? nullptr : a.page_table + (long long)tile.b * a.pt_stride;
  auto page_of = [&](int t) {                             // the page of this wave's block of tile t (past the end: the last block's)
    if constexpr (SRC == PACKED) return 0;
    const int p = load_uniform(pt, min(2 * t + (w >> 1), last_blk) >> a.page_shift);
    return min(max(p, 0), a.n_pages - 1);
  };
  const __bf16* kh = a.k + (long long)kvh * a.k_sh + (SRC == PACKED ? (long long)sq.beg * a.k_st : 0);
  const __bf16* vh = a.v + (long long)kvh * a.v_sh + (SRC == PACKED ? (long long)sq.beg * a.v_st : 0);
  // a lane's K row in its block (K-tile order) and V row, chunk in the 16 of its wave
  const int g4 = lane >> 4, n16 = lane & 15;
  const int krow = 8 * (n16 >> 2) + 4 * (w & 1) + (n16 & 3);
  constexpr int CPR = DVP / 8;            // 16-byte chunks of a V row in LDS
  const int vline = lane / CPR, vchunk = min(lane % CPR, a.dv / 8 - 1);
  // V row (of its block) that copy i of wave w brings to line vline of its kilobyte
  auto vrow = [&](int i) {
    if constexpr (DVP == 32) return 16 * (w & 1) + vline;
    else if constexpr (DVP == 64) return 4 * vline + 2 * (w & 1) + i;
    else return 16 * (w & 1) + 4 * vline + i;
  };
  auto vkb = [&](int i) { return DVP == 64 ? 4 * (w >> 1) + 2 * (w & 1) + i : VI * w + i; };
  // A row of the packed K or V: a uniform base and a lane's 32-bit offset (bytes), rows clamped to the last key.
  const int rows16 = 32 * (w >> 1);
  auto copy_k = [&](char* sk, int t, int pid) __attribute__((always_inline)) {
    const char* src;
    unsigned off;
    if constexpr (SRC == PACKED) {
      const int r0 = min(t * FP_KEYS + rows16, kv_end - 1);
      src = reinterpret_cast<const char*>(kh + (long long)r0 * a.k_st);
      off = __umul24(min(krow, kv_end - 1 - r0), (unsigned)a.k_st * 2) + 16 * g4;
    } else {
      const int blk = min(2 * t + (w >> 1), last_blk);
      src = reinterpret_cast<const char*>(kh + (long long)pid * a.k_st + (long long)(blk & inpage) * (BLK * HD));
      off = TILED ? (w & 1) * 4096 + lane * 16 : krow * (2 * HD) + 16 * g4;
    }
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
      __builtin_amdgcn_global_load_lds((gvoid*)(src + off + kb * (TILED ? 1024 : 64)), (lvoid*)(sk + (4 * w + kb) * 1024), 16, 0, 0);
  };
  auto copy_v = [&](char* sv, int t, int pid) __attribute__((always_inline)) {
    const int r0 = min(t * FP_KEYS + rows16, kv_end - 1), blk = min(2 * t + (w >> 1), last_blk);
    const char* src = reinterpret_cast<const char*>(
        SRC == PACKED ? vh + (long long)r0 * a.v_st : vh + (long long)pid * a.v_st + (long long)(blk & inpage) * (BLK * a.dv));
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int kb = TILED ? w * DV32 + i : vkb(i);
      unsigned off;
      if constexpr (SRC == PACKED) off = __umul24(min(vrow(i), kv_end - 1 - r0), (unsigned)a.v_st * 2) + 16 * vchunk;
      else if constexpr (TILED) off = min(kb - (w >> 1) * 2 * DV32, a.dv / 16 - 1) * 1024 + lane * 16;
      else off = vrow(i) * (2 * a.dv) + 16 * vchunk;
      __builtin_amdgcn_global_load_lds((gvoid*)(src + off), (lvoid*)(sv + kb * VKB), 16, 0, 0);
    }
  };
  // A tile's copies are asked for while the ones before it are computed; past the wait and the barrier they have arrived
  // in every wave, and every wave is done with the stages that the next copies overwrite.
  auto turn = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // Stage of iteration t: K of tile t + 2 over that of tile t, whose scores are there, and V of t + 1.
  int page1 = 0, page2 = 0;               // pages of tiles t + 1 and t + 2
  auto ahead = [&](char* sk, char* sv, int t) __attribute__((always_inline)) {
    if (t + 1 < nt) copy_v(sv, t + 1, page1);
    if (t + 2 < nt) copy_k(sk, t + 2, page2);
    page1 = page2;
    page2 = page_of(t + 3);
  };
  if (t_lo < nt) {
    const int p = page_of(t_lo);
    page1 = page_of(t_lo + 1);
    page2 = page_of(t_lo + 2);
    copy_k(sk0, t_lo, p);
    copy_v(sv0, t_lo, p);
    if (t_lo + 1 < nt) copy_k(sk1, t_lo + 1, page1);
  }
  if (32 * w >= rows) {                   // a wave without rows copies only
    for (int t = t_lo; t < nt; t += 2) {
      if (t == t_lo) turn();
      turn();
      ahead(sk0, sv1, t);
      if (t + 1 >= nt) break;
      turn();
      ahead(sk1, sv0, t + 1);
    }
    return;
  }

  // ---- this wave's rows ---------------------------------------------------------------------------
  const int row = min(32 * w + n, rows - 1);              // rows past the sequence repeat its last, unstored
  const int ri = row_pos(rs, row), pos = min(sq.start + ri, a.capacity - 1);
  const long long head = (long long)kvh * a.rep + (rs.rem + row - (ri - rs.pos0) * a.rep);
  const int w_hi = key_pos(min(32 * w + 31, rows - 1));
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
  const int c16 = n >> 4, nn = n & 15;
  const int kaddr = c16 * 4096 + h * 256 + nn * 16;
  auto read_k = [&](const char* sk, int blk, int kk) {
    return *reinterpret_cast<const bf16x8*>(sk + kaddr + blk * 8192 + (kk >> 1) * 1024 + (kk & 1) * 512);
  };
  // V^T operand of dims 32 md .. + 31 and keys 32 blk + 16 t .. + 15: lane (n, h) holds keys 8 (2 t + h) .. + 7 of a dim.
  // From rows, a 16-lane group reads 4 keys of 16 dims (lanes 4 x .. + 3 key x) and gets, per lane, the 4 keys of one dim.
  const int x4 = n16 >> 2, vcol = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  const int vaddr = TILED ? c16 * 1024 + h * 256 + nn * 16
                  : DVP == 32 ? (8 * h + x4) * 64 + vcol
                  : DVP == 64 ? x4 * VKB + h * 256 + vcol : x4 * VKB + h * 512 + vcol;
  auto read_v = [&](const char* sv, int blk, int t, int md) {
    if constexpr (TILED) {
      return *reinterpret_cast<const bf16x8*>(sv + vaddr + blk * (DV32 * 2048) + md * 2048 + t * 512);
    } else {
      constexpr int U = DVP == 32 ? 256 : DVP == 64 ? 128 : 256;   // from keys 0 .. 3 to 4 .. 7 of a lane's eight
      const int o = md * 64 + (DVP == 32 ? (32 * blk + 16 * t) * 64 : DVP == 64 ? blk * 4 * VKB + t * 512 : (2 * blk + t) * 4 * VKB);
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(sv + vaddr + o));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(sv + vaddr + o + U));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  f32x16 O[DV32];
#pragma unroll
  for (int md = 0; md < DV32; ++md)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[md][i] = 0.f;
  float m_run = NEG_INF, l_run = 0.f;
  auto zero = [](f32x16 (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
  };
  auto fence = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };

  // The running maximum of every row after scores s; what was summed before is scaled to it. Refreshed by the row's own scores
  // alone, so that a row's roundings do not depend on its neighbours'. Returns the reference of the exponents.
  auto maximum = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, s[b][i]);
    mx *= a.qscale;
    if (__any(mx > m_run + LAZY_RESCALE_LOG2)) {
      const float top = fmaxf(mx, __shfl_xor(mx, 32, 64)), mn = top > m_run + LAZY_RESCALE_LOG2 ? top : m_run;
      const float alpha = m_run == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(m_run - mn);
      if (__any(m_run != NEG_INF)) {                      // (not at the first tile)
#pragma unroll
        for (int md = 0; md < DV32; ++md)
#pragma unroll
          for (int i = 0; i < 16; ++i) O[md][i] *= alpha;
        l_run *= alpha;
      }
      m_run = mn;
    }
    return m_run == NEG_INF ? 0.f : m_run;
  };
  // An eighth of a tile's probabilities, four scores of half tt of block b: rounded, and their sum. (Two accumulators, the sums an
  // eighth later, or beside the products with V: within 1 % of this, the last 4 % slower.)
  auto eighth = [&](const f32x16 (&s)[2], bf16x8 (&p)[2][2], int c, float mref) __attribute__((always_inline)) {
    const int b = c >> 2, tt = (c >> 1) & 1, lo = 4 * (c & 1);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[b][tt][lo + i] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[b][4 * tt + 2 * lo + i], a.qscale, -mref));
#pragma unroll
    for (int i = lo; i < lo + 4; i += 2)
      l_run = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[b][tt][i], p[b][tt][i + 1]}, bf16x2{(__bf16)1.f, (__bf16)1.f}, l_run, false);
    asm volatile("" : "+v"(l_run));                       // now: put off, the sums would keep more registers live
  };
  // Operand c of a tile's products with V, md innermost: consecutive products have different accumulators. Operands are
  // read ahead of their products, K two eighths and V three products: a read from LDS takes as long as some four products.
  bf16x8 vq[4];
  auto next_v = [&](const char* sv, int c) __attribute__((always_inline)) {
    if (c < 4 * DV32) vq[c & 3] = read_v(sv, c / (2 * DV32), c / DV32 % 2, c % DV32);
  };
  // O += V^T P^T, the first `ready` operands read.
  auto values = [&](const char* sv, const bf16x8 (&p)[2][2], int ready) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 3; ++c)
      if (c >= ready) next_v(sv, c);
    fence();
#pragma unroll
    for (int c = 0; c < 4 * DV32; ++c) {
      next_v(sv, c + 3);
      fence();
      O[c % DV32] = mfma32(vq[c & 3], p[c / (2 * DV32)][c / DV32 % 2], O[c % DV32]);
    }
    fence();
  };
  auto scores = [&](f32x16 (&s)[2], const char* sk) __attribute__((always_inline)) {
    zero(s);
    bf16x8 kq[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) kq[0][b] = read_k(sk, b, 0);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c < 7)
#pragma unroll
        for (int b = 0; b < 2; ++b) kq[(c + 1) & 1][b] = read_k(sk, b, c + 1);
      fence();
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = mfma32(kq[c & 1][b], q[c], s[b]);
    }
  };

  // A tile that all rows see whole: the scores of the next one (sn) beside the softmax of this one's (s), then its V. The
  // products of the next tile's scores and this one's exponentials are independent and alternate. (Behind the last tile
  // the products are of what the stage holds, and unused.)
  auto step = [&](f32x16 (&s)[2], f32x16 (&sn)[2], const char* skn, const char* sv) __attribute__((always_inline)) {
    const float mref = maximum(s);
    bf16x8 p[2][2], kq[3][2];
    auto next_k = [&](int c) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; ++b) kq[c % 3][b] = read_k(skn, b, c);
    };
    zero(sn);
    fence();
    next_k(0);
    next_k(1);
    fence();
    __builtin_amdgcn_s_setprio(1);                        // ahead of the SIMD's other wave, whose products with V need few slots
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c < 6) next_k(c + 2);
      else next_v(sv, c - 6);
      fence();
#pragma unroll
      for (int b = 0; b < 2; ++b) sn[b] = mfma32(kq[c % 3][b], q[c], sn[b]);
      eighth(s, p, c, mref);
      fence();
    }
    __builtin_amdgcn_s_setprio(0);
    values(sv, p, 2);
  };
  // A tile of which some rows do not see some keys; s becomes the next tile's scores.
  auto tail = [&](f32x16 (&s)[2], const char* skn, const char* sv, int t) __attribute__((always_inline)) {
    const int base = t * FP_KEYS;
    if (base > w_hi) return;                              // uniform per wave: keys past all its rows
    const int seen = pos - base - 8 * h;                  // register i of block b holds key 32 b + 16 (j % 2) + 4 (j / 2) + i % 4,
#pragma unroll                                            // j = i / 4, from base + 8 h on
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * b + 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3) > seen) s[b][i] = NEG_INF;
    const float mref = maximum(s);
    bf16x8 p[2][2];
#pragma unroll
    for (int c = 0; c < 8; ++c) eighth(s, p, c, mref);
    fence();
    // A key that some rows do not see may hold an infinity or NaN in V, and 0 times that is NaN: such a tile (rare) is
    // added one key at a time, to the rows that see it.
    float bad[4] = {0.f, 0.f, 0.f, 0.f};
    next_v(sv, 0);
    next_v(sv, 1);
    next_v(sv, 2);
#pragma unroll
    for (int c = 0; c < 4 * DV32; ++c) {
      next_v(sv, c + 3);
      fence();
      const bf16x8 v = vq[c & 3];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        bad[i] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[2 * i], v[2 * i + 1]}, bf16x2{(__bf16)0.f, (__bf16)0.f}, bad[i], false);
    }
    const float b4 = (bad[0] + bad[1]) + (bad[2] + bad[3]);
    if (__any(b4 != b4)) {
#pragma unroll
      for (int md = 0; md < DV32; ++md)
        for (int x = 0; x < FP_KEYS && base + x <= w_hi; ++x) {
          const int bt = x >> 4;
          bf16x8 px = p[0][0];
#pragma unroll
          for (int i = 1; i < 4; ++i)
            if (bt == i) px = p[i >> 1][i & 1];
          bf16x8 v = read_v(sv, bt >> 1, bt & 1, md);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = i == (x & 15) - 8 * h ? v[i] : (__bf16)0.f;
          const f32x16 y = mfma32(v, px, O[md]);
#pragma unroll
          for (int i = 0; i < 16; ++i) O[md][i] = base + x <= pos ? y[i] : O[md][i];
        }
    } else {
      values(sv, p, 0);
    }
    if (base + FP_KEYS <= w_hi) scores(s, skn);
  };
  if (t_lo < nt) {
    f32x16 s0[2];
    turn();
    if (t_lo * FP_KEYS <= w_hi) scores(s0, sk0);
    int t = t_lo;
    const int nfull = min(nt, (key_pos(0) + 1) / FP_KEYS);   // tiles that all rows of the workgroup see whole
    // An odd last one of packed rows is a step, too (128 sequences of 128 rows: 123 us instead of 133). Over pages it is a
    // tail: the exit in the loop's middle costs the loop 1.5 to 3 % there (2048 rows behind 30000: 748 us instead of 726).
    const int whole = SRC == PACKED ? nfull : t_lo + ((nfull - t_lo) & ~1);
    bool odd = false;                     // which stages hold tile t
    while (t < whole) {
      f32x16 s1[2];
      turn();
      ahead(sk0, sv1, t);
      step(s0, s1, sk1, sv0);
      ++t;
      if (SRC == PACKED && t >= whole) {
#pragma unroll
        for (int b = 0; b < 2; ++b) s0[b] = s1[b];
        odd = true;
        break;
      }
      turn();
      ahead(sk1, sv0, t);
      step(s1, s0, sk0, sv1);
      ++t;
    }
    while (t < nt) {
      if (!odd) {
        turn();
        ahead(sk0, sv1, t);
        tail(s0, sk1, sv0, t);
        if (++t >= nt) break;
      }
      odd = false;
      turn();
      ahead(sk1, sv0, t);
      tail(s0, sk0, sv1, t);
      ++t;
    }
  }

  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (32 * w + n >= rows) return;
  if (n_pieces > 1) {                     // one of several pieces (which are the first of all items)
    float* po = a.part + ((long long)item * a.n_kv + kvh) * FP_ROWS * (a.dv + 2);
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

// Joins the pieces of a tile: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. One workgroup per (item, KV head, 32 rows),
// those of a first piece work; what the item is stands in its record. 32 threads to a row, N rows of a thread (8 apart).
// Bound by latency (the record, the statistics, the results): the rows' and pieces' loads are on their way together, which
// took it from 15.4 to 8.4 us for 8 sequences of up to 300 rows over up to 32000 positions, and the whole call of one row
// over 32000 from 41 to 31.
constexpr int JOIN_ROWS = 32;
template <int N>
__device__ __forceinline__ void join_rows(const FlashPrefillArgs& a, const Record& rec, const float* part, int kvh, int r0) {
  constexpr int U = N == 1 ? 8 : 1;       // pieces at a time (4 for N = 4: 1 to 4 % more time for the whole call)
  const int sub = threadIdx.x & 31, ns = rec.pieces, rw = r0 + (threadIdx.x >> 5), d = 4 * sub;
  const RowSplit rs{rec.pos0, rec.rem, make_fdiv(a.rep)};
  const long long stride = (long long)FP_ROWS * (a.dv + 2) * a.n_kv;   // pieces are n_kv places apart
  const float *ml[N], *o[N];
  float M[N], l[N], w[N];
  f32x4 y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = min(rw + 8 * i, rec.rows - 1);
    ml[i] = part + FP_ROWS * a.dv + r;
    o[i] = part + r * a.dv + min(d, a.dv - 4);
    M[i] = NEG_INF;
    l[i] = 0.f;
    y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int s = sub; s < ns; s += 32)
#pragma unroll
    for (int i = 0; i < N; ++i) M[i] = fmaxf(M[i], ml[i][s * stride]);
#pragma unroll
  for (int x = 1; x < 32; x <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) M[i] = fmaxf(M[i], __shfl_xor(M[i], x, 32));
  for (int s0 = 0; s0 < ns; s0 += 32) {
    const int s = s0 + sub;
#pragma unroll
    for (int i = 0; i < N; ++i) {         // lane `sub` has the weight of piece s0 + sub
      const float x = ml[i][min(s, ns - 1) * stride], z = ml[i][min(s, ns - 1) * stride + FP_ROWS];
      w[i] = s < ns ? __builtin_amdgcn_exp2f(x - (M[i] == NEG_INF ? 0.f : M[i])) : 0.f;
      l[i] += s < ns ? w[i] * z : 0.f;
    }
    for (int c = s0; c < min(s0 + 32, ns); c += U) {
      f32x4 v[U][N];
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) v[k][i] = *reinterpret_cast<const f32x4*>(o[i] + min(c + k, ns - 1) * stride);
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const f32x4 t = v[k][i] * __shfl(w[i], c + k - s0, 32);
          if (c + k < ns) y[i] += t;
        }
    }
  }
#pragma unroll
  for (int x = 1; x < 32; x <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] += __shfl_xor(l[i], x, 32);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = rw + 8 * i, pos = row_pos(rs, r);
    if (d >= a.dv || r >= min(r0 + JOIN_ROWS, rec.rows)) continue;
    const float inv = 1.f / l[i];
    bf16x4 x;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = rec.start + pos < 0 ? (__bf16)0.f : (__bf16)(y[i][k] * inv);
    *reinterpret_cast<bf16x4*>(a.out + ((long long)(rec.beg + pos) * a.n_q + (long long)kvh * a.rep +
                                        (rs.rem + r - (pos - rs.pos0) * a.rep)) * a.dv + d) = x;
  }
}

__global__ __launch_bounds__(256) void palu_flash_prefill_join_kernel(const FlashPrefillArgs a) {
  const int rest = blockIdx.x / a.n_kv, kvh = blockIdx.x - rest * a.n_kv, item = rest / (FP_ROWS / JOIN_ROWS);
  const Record rec = a.records[item * a.n_kv + kvh];
  const int r0 = rest % (FP_ROWS / JOIN_ROWS) * JOIN_ROWS;
  if (rec.pieces == 0 || r0 >= rec.rows) return;
  const float* part = a.part + ((long long)item * a.n_kv + kvh) * FP_ROWS * (a.dv + 2);
  if (rec.rows - r0 <= 8) join_rows<1>(a, rec, part, kvh, r0);
  else join_rows<JOIN_ROWS / 8>(a, rec, part, kvh, r0);
}

// Tiles of a batch, at most: a sequence's last tile may hold fewer rows.
long long most_tiles(int T, int B, int rep) { return (long long)T * rep / FP_ROWS + std::min(T, B); }

// Whether tiles may be cut along their keys: where contexts stand before the rows. (Packed prompts stand on their own keys;
// cutting their longest tiles, one prompt of 1024 positions took 42 us instead of 27 and one of 2048 82 instead of 55.)
// Up to 2^28 rows of heads, which keeps find_tile's levels below 2^22, and up to FP_SORTED sequences, whose lengths a wave holds
// in registers. (Single rows, one behind 60000 positions and the others behind 500, 8 KV heads: 256 take 180 us, 300 1039.)
bool may_split(int T, int B, int n_q, bool paged, long long max_keys) {
  return paged && B <= FP_SORTED && max_keys > FP_MIN_KEYS && (long long)T * n_q <= (1ll << 28);
}

// Items of a KV head that may be pieces of cut tiles (they are the first of all items), at most; 0: no tile is cut. With len levels to a
// piece (find_tile), a tile of level t is cut into t / len + 3 / 4 pieces where t >= 1.25 len, so into fewer than 2 t / len; all
// tiles' levels together are at most FP_WGS / (FP_PIECE n_kv) times len; len is not below `least`, no level above `top`.
long long cut_items(int T, int B, int n_q, int n_kv, long long max_keys) {
  const int rep = n_q / n_kv, shift = 31 - __builtin_clz(std::max(1, FP_ROWS / rep)), least = std::max(2, FP_MIN_KEYS >> shift);
  const long long tiles = most_tiles(T, B, rep), top = (max_keys >> shift) + ((long long)T * rep + FP_ROWS - 1) / FP_ROWS - 1;
  const long long of_tile = (top + least - least / 4 - 1) / least, share = (long long)(FP_WGS / FP_PIECE) / n_kv + 1;
  return of_tile < 2 ? 0 : std::min({tiles * of_tile, share + tiles, 2 * share});
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workspace: the pieces' partial results, then the items' records.
size_t part_bytes(int n_q, int n_kv, int T, int B, bool paged, long long max_keys, int dv) {
  if (!may_split(T, B, n_q, paged, max_keys)) return 0;
  return (size_t)cut_items(T, B, n_q, n_kv, max_keys) * n_kv * (FP_ROWS * (dv + 2) * sizeof(float) + sizeof(Record));
}

int check_dims(int T, int B, int n_q, int n_kv, int dv, const char* who) {
  if (T <= 0 || B <= 0 || n_q <= 0 || n_kv <= 0)
    return fail(PALU_EINVAL, "%s: row, sequence and head counts must be positive, got %d, %d, %d, %d", who, T, B, n_q, n_kv);
  if (n_q % n_kv) return fail(PALU_EINVAL, "%s: n_q = %d must be a multiple of the KV head count %d", who, n_q, n_kv);
  if (dv < 16 || dv > HD || dv % 16)
    return fail(PALU_EUNSUPPORTED, "%s: head_dim_v %d (multiples of 16 up to %d)", who, dv, HD);
  if ((long long)T * n_q > (1ll << 30) || n_q > 65535 || B > 65535 || most_tiles(T, B, n_q / n_kv) * n_kv > (1ll << 23))
    return fail(PALU_EUNSUPPORTED, "%s: %d rows of %d heads in %d sequences exceed the grid", who, T, n_q, B);
  return PALU_OK;
}

template <Source SRC>
int launch_prefill(FlashPrefillArgs& a, long long max_keys, void* workspace, size_t workspace_bytes, const char* who,
                   hipStream_t s) {
  const size_t need = part_bytes(a.n_q, a.n_kv, a.T, a.B, SRC != PACKED, max_keys, a.dv);
  if (need && (!workspace || workspace_bytes < need || !al16(workspace)))
    return fail(PALU_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes needed (palu_flash_prefill_workspace_bytes), got %zu",
                who, need, workspace ? workspace_bytes : 0);
  a.cut = need ? (int)cut_items(a.T, a.B, a.n_q, a.n_kv, max_keys) : 0;
  a.part = need ? static_cast<float*>(workspace) : nullptr;
  a.records = reinterpret_cast<Record*>(a.part + (size_t)a.cut * a.n_kv * FP_ROWS * (a.dv + 2));
  const unsigned grid = (unsigned)((most_tiles(a.T, a.B, a.rep) + a.cut) * a.n_kv);
  auto go = [&](auto kern, unsigned wgs) {
    hipLaunchKernelGGL(kern, dim3(wgs), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
  };
  int rc = PALU_OK;
  switch ((a.dv + 31) / 32) {
    case 1: rc = go(palu_flash_prefill_kernel<SRC, 1>, grid); break;
    case 2: rc = go(palu_flash_prefill_kernel<SRC, 2>, grid); break;
    case 3: rc = go(palu_flash_prefill_kernel<SRC, 3>, grid); break;
    default: rc = go(palu_flash_prefill_kernel<SRC, 4>, grid); break;
  }
  if (rc == PALU_OK && need) rc = go(palu_flash_prefill_join_kernel, (unsigned)(a.cut * a.n_kv) * (FP_ROWS / JOIN_ROWS));
  return rc;
}

// (a lane's offset in a block of 32 rows is a 24-bit product)
bool stride_ok(long long st) { return st >= 0 && st % 8 == 0; }
bool row_stride_ok(long long st) { return stride_ok(st) && st < (1 << 22); }

}  // namespace

extern "C" size_t palu_flash_prefill_workspace_bytes(int rows, int batch, int n_q, int n_kv, int max_keys, int head_dim_v) {
  palu::g_err[0] = 0;
  if (max_keys <= 0 || check_dims(rows, batch, n_q, n_kv, head_dim_v, "palu_flash_prefill_workspace_bytes")) return 0;
  return part_bytes(n_q, n_kv, rows, batch, true, max_keys, head_dim_v);
}

extern "C" int palu_flash_prefill(const void* q, long long q_row_stride, long long q_head_stride, const void* k,
                                  long long k_row_stride, long long k_head_stride, const void* v, long long v_row_stride,
                                  long long v_head_stride, const int32_t* cu_seqlens, void* out, float scale, int rows,
                                  int batch, int n_q, int n_kv, int head_dim_v, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_flash_prefill";
  if (!q || !k || !v || !cu_seqlens || !out) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  if (int rc = check_dims(rows, batch, n_q, n_kv, head_dim_v, who)) return rc;
  if (!stride_ok(q_row_stride) || !stride_ok(q_head_stride) || !row_stride_ok(k_row_stride) || !stride_ok(k_head_stride) ||
      !row_stride_ok(v_row_stride) || !stride_ok(v_head_stride))
    return fail(PALU_EINVAL, "%s: strides must be non-negative multiples of 8, rows of k and v less than 2^22 apart", who);
  if (!al16(q) || !al16(k) || !al16(v) || !al16(out)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  FlashPrefillArgs a{static_cast<const __bf16*>(q), q_row_stride, q_head_stride, static_cast<const __bf16*>(k),
                     static_cast<const __bf16*>(v), k_row_stride, k_head_stride, v_row_stride, v_head_stride, cu_seqlens, nullptr,
                     nullptr, 0, 0, 0, 0x7fffffff, rows, batch, n_q, n_kv, n_q / n_kv, head_dim_v,
                     scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f, (scale > 0.f) - (scale < 0.f),
                     static_cast<__bf16*>(out), nullptr, nullptr, 0};
  return launch_prefill<PACKED>(a, 0, nullptr, 0, who, stream);
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
  if (!stride_ok(q_row_stride) || !stride_ok(q_head_stride))
    return fail(PALU_EINVAL, "%s: strides must be non-negative multiples of 8", who);
  if (!al16(q) || !al16(k_pages) || !al16(v_pages) || !al16(out)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  const long long k_sh = (long long)page_size * HD, v_sh = (long long)page_size * head_dim_v;
  const int capacity = max_pages_per_seq * page_size;
  FlashPrefillArgs a{static_cast<const __bf16*>(q), q_row_stride, q_head_stride, static_cast<const __bf16*>(k_pages),
                     static_cast<const __bf16*>(v_pages), k_sh * n_kv, k_sh, v_sh * n_kv, v_sh, cu_seqlens, start_pos, page_table,
                     max_pages_per_seq, num_pages, shift, capacity, rows, batch, n_q, n_kv, n_q / n_kv, head_dim_v,
                     scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f, (scale > 0.f) - (scale < 0.f),
                     static_cast<__bf16*>(out), nullptr, nullptr, 0};
  if (cache_layout == PALU_LAYOUT_TILED) return launch_prefill<PAGED_TILED>(a, capacity, workspace, workspace_bytes, who, stream);
  return launch_prefill<PAGED_ROWS>(a, capacity, workspace, workspace_bytes, who, stream);
}
