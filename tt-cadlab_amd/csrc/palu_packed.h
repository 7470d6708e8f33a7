// The 32-position blocks that the packed rows of a batch touch in their pages: shared by the ops that move packed rows into
// page pools and out of them.
#pragma once
#include "palu_kernel.h"

namespace {

// Packed sequences over a page table. cu [B + 1]: sequence b's rows are cu[b] .. cu[b + 1] - 1 of T; row i of it stands at
// position start[b] + i (start null: i).
struct PackedSeqs {
  const int32_t* cu;
  const int32_t* start;
  const int32_t* table;
  int T, B, n_pages, page_shift, pt_stride;   // pages of 32 << page_shift positions
};

// Sequence b's packed rows inside [0, T) and the position of its first.
__device__ __forceinline__ void packed_seq(const PackedSeqs& a, int b, int& beg, int& len, int& start) {
  const int c0 = a.cu[b], c1 = a.cu[b + 1];
  beg = min(max(c0, 0), a.T);
  len = min(max(c1, beg), a.T) - beg;
  start = a.start ? a.start[b] : 0;
  start = min(max(start, -(1 << 29)), 1 << 29);            // (farther is as far: at most 2^28 rows, 2^16 positions)
}

// Block number `want` of the batch, counted sequence by sequence: sequence b's block blk (b < 0: past the last one), whose
// positions lo .. hi - 1 are packed rows row0 + lo .., on page pid (as the table has it, possibly outside the pool). Only
// blocks inside the table are counted, or with ALL those before and behind it as well, whose pid is -1.
struct PackedBlock {
  int b, blk, lo, hi, row0, pid;
};
template <bool ALL = false>
__device__ __forceinline__ PackedBlock packed_block(const PackedSeqs& a, int want) {
  const int lane = threadIdx.x & 63, cap_blocks = a.pt_stride << a.page_shift;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int lb, ll, ls;
    packed_seq(a, min(b0 + lane, a.B - 1), lb, ll, ls);
    const int first = (ALL ? ls : max(ls, 0)) >> 5, past = (ls + ll + 31) >> 5;
    const int end = ALL ? past : min(past, cap_blocks);   // blocks first .. end - 1
    const int n = b0 + lane < a.B && ll > 0 && end > first ? end - first : 0;
    const int upto = before + wave_scan(n);
    const unsigned long long m = __ballot(want < upto);
    if (m) {
      const int l = __builtin_ctzll(m);
      const int beg = __builtin_amdgcn_readlane(lb, l), len = __builtin_amdgcn_readlane(ll, l);
      const int start = __builtin_amdgcn_readlane(ls, l);
      const int blk = __builtin_amdgcn_readlane(first, l) + want - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
      const bool in_table = !ALL || (blk >= 0 && blk < cap_blocks);
      const int pid = in_table ? a.table[(long long)(b0 + l) * a.pt_stride + (blk >> a.page_shift)] : -1;
      return PackedBlock{b0 + l, blk, max(start, 32 * blk), min(start + len, 32 * blk + 32), beg - start, pid};
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return PackedBlock{-1, 0, 0, 0, 0, 0};
}

// Workgroups that take a block each: a sequence of n rows touches at most n / 32 + 2 blocks, and at most n.
inline unsigned packed_blocks(int rows, int batch) {
  const long long most = rows / 32 + 2LL * batch;
  return (unsigned)(rows < most ? rows : most);
}

}  // namespace
