// Page pools of several sequences: rows of a packed batch into their pages, and the bookkeeping of a page table with the
// copies of pages that it asks for. The pools of all layers share one page table; a page is free when no row's
// used entries name it, so nothing but the table and the lengths has to be kept.
#include "palu_kernel.h"

#include <algorithm>

namespace {

// ---- packed rows into pages -------------------------------------------------------------------
// cache[table[b][p / page]][g][p % page] = rows[cu[b] + i][g], p = start[b] + i. A workgroup takes one 32-position block of one
// sequence and a few groups (64 bytes a thread); blocks are numbered sequence by sequence, found by a wave-wide sum over the
// lengths. Bound by memory: the rows in, as many bytes out; a block at a sequence's end keeps its other positions. 34 MB of
// rows of 16 sequences into K tiles take 13.1 us (5.2 TB/s read and written), into V tiles, whose regrouping goes through registers, 20.2
// (3.4), 57 rows 3.7 us.
struct FillArgs {
  __bf16* cache;                          // [n_pages][G][page][width]
  const __bf16* rows;
  long long st, sg;                       // source strides: row, group
  const int32_t* cu;
  const int32_t* start;                   // or null
  const int32_t* table;
  int T, B, G, width, n_pages, page_shift, pt_stride, gpw;   // gpw: groups per workgroup
};

// Sequence b's packed rows inside [0, T) and the position of its first.
__device__ __forceinline__ void fill_seq(const FillArgs& a, int b, int& beg, int& len, int& start) {
  const int c0 = a.cu[b], c1 = a.cu[b + 1];
  beg = min(max(c0, 0), a.T);
  len = min(max(c1, beg), a.T) - beg;
  start = a.start ? a.start[b] : 0;
  start = min(max(start, -(1 << 29)), 1 << 29);            // (farther is as far: at most 2^28 rows, 2^16 positions)
}

template <int LAYOUT>
__global__ __launch_bounds__(256) void palu_fill_pages_kernel(const FillArgs a) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int cap_blocks = a.pt_stride << a.page_shift;
  // this workgroup's block: number blockIdx.x of the batch
  int beg = 0, len = 0, start = 0, blk = -1, b = 0;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int lb, ll, ls;
    fill_seq(a, min(b0 + lane, a.B - 1), lb, ll, ls);
    const int first = max(ls, 0) >> 5, end = min((ls + ll + 31) >> 5, cap_blocks);   // blocks first .. end - 1
    const int n = b0 + lane < a.B && ll > 0 && end > first ? end - first : 0;
    const int upto = before + wave_scan(n), want = (int)blockIdx.x;
    const unsigned long long m = __ballot(want < upto);
    if (m) {
      const int l = __builtin_ctzll(m);
      beg = __builtin_amdgcn_readlane(lb, l);
      len = __builtin_amdgcn_readlane(ll, l);
      start = __builtin_amdgcn_readlane(ls, l);
      blk = __builtin_amdgcn_readlane(first, l) + want - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
      b = b0 + l;
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  if (blk < 0) return;
  const int pid = a.table[(long long)b * a.pt_stride + (blk >> a.page_shift)];
  if (pid < 0 || pid >= a.n_pages) return;                // as the append: ids outside the pool are skipped
  const int lo = max(start, 32 * blk), hi = min(start + len, 32 * blk + 32);   // the block's positions lo .. hi - 1
  const int vec = a.width / 8, page = 32 << a.page_shift, g0 = blockIdx.y * a.gpw, g1 = min(a.G, g0 + a.gpw);
  const int inpage = (blk & ((1 << a.page_shift) - 1)) * 32;
  const __bf16* src = a.rows + (long long)(beg - start) * a.st;
  __bf16* dst = a.cache + (long long)pid * a.G * page * a.width;
  if constexpr (LAYOUT == PALU_LAYOUT_TILED_V) {
    // 8 positions x 8 columns a thread: eight 16-byte loads, regrouped, eight 16-byte slots
    for (int e = tid; e < (g1 - g0) * 4 * vec; e += 256) {
      const int v = e % vec, o = e / vec & 3, g = g0 + e / (4 * vec), p0 = 32 * blk + 8 * o;
      if (p0 >= hi || p0 + 8 <= lo) continue;
      bf16x8 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = *reinterpret_cast<const bf16x8*>(src + (long long)min(max(p0 + i, lo), hi - 1) * a.st + g * a.sg + 8 * v);
      __bf16* out = dst + (long long)g * page * a.width + tiled_v_offset(inpage + 8 * o, 8 * v, a.width);
      if (p0 >= lo && p0 + 8 <= hi) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          bf16x8 y;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i][c];
          *reinterpret_cast<bf16x8*>(out + 8 * c) = y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p0 + i >= lo && p0 + i < hi)
#pragma unroll
            for (int c = 0; c < 8; ++c) out[8 * c + i] = x[i][c];
      }
    }
  } else {
    for (int e = tid; e < (g1 - g0) * 32 * vec; e += 256) {
      int v, t;
      const int g = g0 + e / (32 * vec), x = e % (32 * vec);
      if constexpr (LAYOUT == PALU_LAYOUT_TILED) {        // 16 positions of a chunk after the other, as the tiles lie
        const int nn = x & 15, rest = x >> 4, c = rest / vec;
        v = rest - c * vec;
        t = 8 * (nn >> 2) + 4 * c + (nn & 3);
      } else {
        t = x / vec;
        v = x - t * vec;
      }
      const int p = 32 * blk + t;
      if (p < lo || p >= hi) continue;
      const bf16x8 y = *reinterpret_cast<const bf16x8*>(src + (long long)p * a.st + g * a.sg + 8 * v);
      __bf16* out = dst + (long long)g * page * a.width;
      if constexpr (LAYOUT == PALU_LAYOUT_TILED) store_k8(out, inpage + t, 8 * v, a.width, y);
      else *reinterpret_cast<bf16x8*>(out + (long long)(inpage + t) * a.width + 8 * v) = y;
    }
  }
}

// ---- the page table -----------------------------------------------------------------------------
// One workgroup plans (the table is small: 64 rows of 64 entries are 16 KB), a second launch copies. The plan keeps a bit
// per page in LDS: set where a row's used entries name the page.
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_LDS = 156 << 10;       // dynamic LDS of a plan, at most
constexpr int MAX_POOLS = 128;            // pools of one copy launch

struct PlanArgs {
  const int32_t* table;                   // [B][slots]
  const int32_t* len;                     // [B]
  const int32_t* parents;                 // [B] or null (every row its own)
  const int32_t* new_len;                 // [B] or null (as long as the parent)
  int32_t* table_out;
  int32_t* len_out;
  int B, slots, n_pages, page, log2_page;
  int hash;                               // entries of the update's hash table, a power of two
  int32_t* ws;                            // [4]: number of copies; then src[n], dst[n]; then a list of n_pages
  int max_copies;
};

// Pages of n positions.
__device__ __forceinline__ int pages_of(const PlanArgs& a, int n) { return (n + a.page - 1) >> a.log2_page; }

// Exclusive prefix sum of x over the workgroup's threads, and its total. `part`: PLAN_THREADS / 64 + 1 ints.
__device__ __forceinline__ int block_scan(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int s = wave_scan(x);
  __syncthreads();                        // part may still be read from the call before
  if (lane == 63) part[w] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < PLAN_THREADS / 64; ++i) {
    before += i < w ? part[i] : 0;
    all += part[i];
  }
  total = all;
  return before + s - x;
}

__device__ __forceinline__ bool in_pool(int p, int n) { return p >= 0 && p < n; }
__device__ __forceinline__ void set_bit(unsigned* bits, int p) { atomicOr(&bits[p >> 5], 1u << (p & 31)); }
__device__ __forceinline__ bool get_bit(const unsigned* bits, int p) { return bits[p >> 5] >> (p & 31) & 1; }

// Rows of the table by waves, four at a time so that their loads are on their way together: use(b, j, entry) for the first
// n(b) slots of every row's source row from(b).
template <typename N, typename From, typename Use>
__device__ __forceinline__ void each_entry(const PlanArgs& a, N n, From from, Use use) {
  constexpr int R = 4, WAVES = PLAN_THREADS / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int b0 = w; b0 < a.B; b0 += R * WAVES) {
    const int32_t* row[R];
    int cnt[R], most = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int b = b0 + r * WAVES;
      cnt[r] = b < a.B ? n(b) : 0;
      row[r] = a.table + (long long)(cnt[r] ? from(b) : 0) * a.slots;
      most = max(most, cnt[r]);
    }
    for (int j = lane; j < most; j += 64) {
      int x[R];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = row[r][min(j, max(cnt[r], 1) - 1)];
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (j < cnt[r]) use(b0 + r * WAVES, j, x[r]);
    }
  }
}

// A row's whole kept pages stay shared. The page that a row writes next, the one its kept positions end inside, has to be
// its own: the first row in order that would write it keeps it, unless another row holds it as a whole page; the others get
// copies. New pages are the lowest free ones, in the order of rows and slots; when they run out, a row's length is cut to
// what it has. All choices go by row and page order, none by the order in which threads arrive.
// Bound by latency, three loads deep (a row's parent, its length, its page) and a barrier for each step of the plan: 8 rows
// of 64 slots 4.5 us, 64 rows 10 us; with rows one after the other, each with loads of its own at every step, 64 took 14.8.
__global__ __launch_bounds__(PLAN_THREADS) void palu_update_pages_kernel(const PlanArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned lds[];
  __shared__ int part[PLAN_THREADS / 64 + 1], n_copies;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int words = (a.n_pages + 31) >> 5;
  unsigned* bits = lds;
  int* key = reinterpret_cast<int*>(bits + words);        // page -> first row that would write it
  int* first = key + a.hash;
  int* parent = first + a.hash;                           // [B]; later the row's first new page's place in the free list
  int* keep = parent + a.B;                               // [B] positions kept of the parent's; later the pages a row has
  int* want = keep + a.B;                                 // [B] positions in all
  int* last = want + a.B;                                 // [B] the page that the kept positions end inside, or -1
  for (int b = tid; b < a.B; b += PLAN_THREADS) {
    const int most = a.slots * a.page;
    int p = a.parents ? a.parents[b] : b;
    const int asked = a.new_len ? a.new_len[b] : 0;
    if (!in_pool(p, a.B)) p = -1;
    const int have = p < 0 ? 0 : min(max(a.len[p], 0), most);
    const int all = a.new_len ? min(max(asked, 0), most) : have, kept = min(have, all);
    int page = -1;
    if (kept & (a.page - 1)) page = a.table[(long long)p * a.slots + (kept >> a.log2_page)];
    parent[b] = p;
    keep[b] = kept;
    want[b] = all;
    last[b] = in_pool(page, a.n_pages) ? page : -1;
  }
  for (int i = tid; i < words; i += PLAN_THREADS) bits[i] = 0;
  for (int i = tid; i < a.hash; i += PLAN_THREADS) key[i] = -1, first[i] = 0x7fffffff;
  if (tid == 0) n_copies = 0;
  __syncthreads();
  each_entry(a, [&](int b) { return keep[b] >> a.log2_page; }, [&](int b) { return parent[b]; }, [&](int b, int j, int p) {
    a.table_out[(long long)b * a.slots + j] = p;
    if (in_pool(p, a.n_pages)) set_bit(bits, p);
  });
  for (int b = w; b < a.B; b += PLAN_THREADS / 64)
    for (int j = pages_of(a, want[b]) + lane; j < a.slots; j += 64) a.table_out[(long long)b * a.slots + j] = -1;
  __syncthreads();
  const int per = (a.B + PLAN_THREADS - 1) / PLAN_THREADS;   // rows of a thread, next to each other
  const int b_lo = min(a.B, tid * per), b_hi = min(a.B, b_lo + per);
  for (int b = b_lo; b < b_hi; ++b) {
    const int p = last[b];
    if (p < 0 || get_bit(bits, p)) continue;
    unsigned s = (unsigned)p * 2654435761u & (a.hash - 1);
    while (true) {
      const int k = atomicCAS(&key[s], -1, p);
      if (k == -1 || k == p) break;
      s = (s + 1) & (a.hash - 1);                         // at most half the entries are taken
    }
    atomicMin(&first[s], b);
  }
  __syncthreads();
  int demand = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int p = last[b], full = keep[b] >> a.log2_page;
    bool mine = false;                                    // (a page that another row holds whole is in no entry)
    if (p >= 0) {
      unsigned s = (unsigned)p * 2654435761u & (a.hash - 1);
      while (key[s] != p && key[s] != -1) s = (s + 1) & (a.hash - 1);
      mine = key[s] == p && first[s] == b;
    }
    if (mine) {
      set_bit(bits, p);
      a.table_out[(long long)b * a.slots + full] = p;
      last[b] = -1;
    }
    keep[b] = full + mine;
    demand += pages_of(a, want[b]) - keep[b];
  }
  int total;
  int at = block_scan(demand, part, total);
  for (int b = b_lo; b < b_hi; ++b) {
    parent[b] = at;
    at += pages_of(a, want[b]) - keep[b];
  }
  // The lowest free pages in order, as many as are asked for.
  int32_t* list = total <= 2 * a.hash ? key : a.ws + 4 + 2 * a.max_copies;   // (the hash table is done with)
  const int wper = (words + PLAN_THREADS - 1) / PLAN_THREADS, w_lo = min(words, tid * wper), w_hi = min(words, w_lo + wper);
  auto free_bits = [&](int i) { return ~bits[i] & (32 * i + 32 <= a.n_pages ? ~0u : (1u << (a.n_pages & 31)) - 1); };
  __syncthreads();                                        // all bits are set
  int mine = 0;
  for (int i = w_lo; i < w_hi; ++i) mine += __popc(free_bits(i));
  int n_free;
  int rank = block_scan(mine, part, n_free);
  for (int i = w_lo; i < w_hi && rank < total; ++i)
    for (unsigned f = free_bits(i); f; f &= f - 1, ++rank)
      if (rank < total) list[rank] = 32 * i + __builtin_ctz(f);
  __syncthreads();
  for (int b = w; b < a.B; b += PLAN_THREADS / 64) {
    const int have = keep[b], need = pages_of(a, want[b]), o = parent[b];
    const int got = min(need - have, max(n_free - o, 0));
    int32_t* out = a.table_out + (long long)b * a.slots;
    for (int j = have + lane; j < need; j += 64) {
      const int p = j - have < got ? list[o + j - have] : -1;
      out[j] = p;
      if (j == have && got > 0 && last[b] >= 0) {
        const int c = atomicAdd(&n_copies, 1);            // the copies do not touch each other: any order
        a.ws[4 + c] = last[b];
        a.ws[4 + a.max_copies + c] = p;
      }
    }
    if (lane == 0) a.len_out[b] = min(want[b], (have + got) * a.page);
  }
  __syncthreads();
  if (tid == 0) a.ws[0] = n_copies;
}

// The n pages in use move to pages 0 .. n - 1: those at n or above, in order, to the free ones below n, in order. Bound by
// latency: 48 rows of 128 slots 10 us.
__global__ __launch_bounds__(PLAN_THREADS) void palu_compact_pages_kernel(const PlanArgs a, int32_t* n_live_out) {
  extern __shared__ __attribute__((aligned(16))) unsigned bits[];
  __shared__ int part[PLAN_THREADS / 64 + 1], low;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int words = (a.n_pages + 31) >> 5;
  for (int i = tid; i < words; i += PLAN_THREADS) bits[i] = 0;
  __syncthreads();
  auto used = [&](int b) { return pages_of(a, min(max(a.len[b], 0), a.slots * a.page)); };
  auto itself = [](int b) { return b; };
  each_entry(a, used, itself, [&](int, int, int p) {
    if (in_pool(p, a.n_pages)) set_bit(bits, p);
  });
  __syncthreads();
  const int wper = (words + PLAN_THREADS - 1) / PLAN_THREADS, w_lo = min(words, tid * wper), w_hi = min(words, w_lo + wper);
  int mine = 0;
  for (int i = w_lo; i < w_hi; ++i) mine += __popc(bits[i]);
  int n_live;
  const int before = block_scan(mine, part, n_live);      // pages in use below this thread's words
  int32_t *src = a.ws + 4, *dst = src + a.max_copies, *to = dst + a.max_copies;
  auto below = [&](int i) {                               // bits of word i that are pages under n_live
    return 32 * i + 32 <= n_live ? ~0u : 32 * i >= n_live ? 0u : (1u << (n_live & 31)) - 1;
  };
  int mine_low = 0, n_low;
  for (int i = w_lo; i < w_hi; ++i) mine_low += __popc(bits[i] & below(i));
  block_scan(mine_low, part, n_low);
  int live = before;
  for (int i = w_lo; i < w_hi; ++i) {
    const unsigned x = bits[i], m = below(i);
    for (unsigned f = x & ~m; f; f &= f - 1) {
      const int bit = __builtin_ctz(f);
      src[live + __popc(x & ((1u << bit) - 1)) - n_low] = 32 * i + bit;
    }
    for (unsigned f = ~x & m; f; f &= f - 1) {
      const int bit = __builtin_ctz(f);
      dst[32 * i + bit - live - __popc(x & ((1u << bit) - 1))] = 32 * i + bit;
    }
    live += __popc(x);
  }
  if (tid == 0) low = n_live - n_low;
  __syncthreads();
  for (int i = tid; i < low; i += PLAN_THREADS) to[src[i]] = dst[i];
  __syncthreads();
  each_entry(a, used, itself, [&](int b, int j, int p) {
    a.table_out[(long long)b * a.slots + j] = in_pool(p, a.n_pages) && p >= n_live ? to[p] : p;
  });
  for (int b = w; b < a.B; b += PLAN_THREADS / 64)
    for (int j = used(b) + lane; j < a.slots; j += 64) a.table_out[(long long)b * a.slots + j] = -1;
  if (tid == 0) {
    a.ws[0] = low;
    n_live_out[0] = n_live;
  }
}

// Page copies of a plan in every pool: 16 KB pieces, a workgroup to a piece, as many workgroups as the chip holds. Bound by
// memory: 840 MB read and written take 173 us (4.9 TB/s, the rate of one large copy).
constexpr int COPY_VECS = 4;              // 16-byte vectors of a thread in flight
constexpr int COPY_BYTES = 256 * 16 * COPY_VECS;

struct CopyArgs {
  const int32_t* ws;
  int max_copies, n_pools, pieces;        // pieces of the largest page
  char* pool[MAX_POOLS];
  long long bytes[MAX_POOLS];             // of a page
};

__global__ __launch_bounds__(256) void palu_copy_pages_kernel(const CopyArgs a) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const int n = a.ws[0];
  const long long total = (long long)n * a.n_pools * a.pieces;
  for (long long u = blockIdx.x; u < total; u += gridDim.x) {
    const int c = (int)(u % a.pieces);
    const long long rest = u / a.pieces;
    const int pool = (int)(rest % a.n_pools), i = (int)(rest / a.n_pools);
    const long long bytes = a.bytes[pool], o = (long long)c * COPY_BYTES + threadIdx.x * 16;
    const char* s = a.pool[pool] + a.ws[4 + i] * bytes;
    char* d = a.pool[pool] + a.ws[4 + a.max_copies + i] * bytes;
    i32x4 x[COPY_VECS];
#pragma unroll
    for (int k = 0; k < COPY_VECS; ++k)
      if (o + k * 4096 < bytes) x[k] = *reinterpret_cast<const i32x4*>(s + o + k * 4096);
#pragma unroll
    for (int k = 0; k < COPY_VECS; ++k)
      if (o + k * 4096 < bytes) *reinterpret_cast<i32x4*>(d + o + k * 4096) = x[k];
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_of(int page_size) { return 31 - __builtin_clz(page_size); }

int hash_entries(int B) {
  int h = 64;
  while (h < 2 * B) h *= 2;
  return h;
}

size_t update_lds(int B, int n_pages) { return 4 * ((size_t)(n_pages + 31) / 32 + 2 * (size_t)hash_entries(B) + 4 * (size_t)B); }

int check_table(const void* table, const void* len, const void* table_out, int B, int slots, int n_pages, int page, const void* ws,
                size_t ws_bytes, size_t need, const char* who) {
  if (!table || !len || !table_out) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  int shift = 0;
  if (int rc = palu::check_pages(static_cast<const int32_t*>(table), n_pages, page, slots, &shift, who)) return rc;
  if (B <= 0) return fail(PALU_EINVAL, "%s: batch must be positive, got %d", who, B);
  if (table == table_out) return fail(PALU_EINVAL, "%s: the new page table must not be the old one's memory", who);
  if (!ws || !al16(ws) || ws_bytes < need)
    return fail(PALU_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes needed (palu_pages_workspace_bytes), got %zu", who, need,
                ws ? ws_bytes : 0);
  return PALU_OK;
}

int check_pools(void* const* pools, const long long* page_bytes, int n_pools, const char* who) {
  if (n_pools < 0 || (n_pools > 0 && (!pools || !page_bytes))) return fail(PALU_EINVAL, "%s: %d pools", who, n_pools);
  for (int i = 0; i < n_pools; ++i)
    if (!pools[i] || !al16(pools[i]) || page_bytes[i] <= 0 || page_bytes[i] % 16)
      return fail(PALU_EINVAL, "%s: pool %d must be 16-byte aligned, its pages a multiple of 16 bytes, got %lld", who, i,
                  page_bytes[i]);
  return PALU_OK;
}

int launched(const char* who, const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s: %s launch: %s", who, what, hipGetErrorString(e));
}

int launch_copies(const PlanArgs& a, void* const* pools, const long long* page_bytes, int n_pools, const char* who, hipStream_t s) {
  for (int p0 = 0; p0 < n_pools; p0 += MAX_POOLS) {
    CopyArgs c;
    c.ws = a.ws;
    c.max_copies = a.max_copies;
    c.n_pools = std::min(MAX_POOLS, n_pools - p0);
    long long most = 0;
    for (int i = 0; i < c.n_pools; ++i) {
      c.pool[i] = static_cast<char*>(pools[p0 + i]);
      c.bytes[i] = page_bytes[p0 + i];
      most = std::max(most, c.bytes[i]);
    }
    c.pieces = (int)((most + COPY_BYTES - 1) / COPY_BYTES);
    const long long units = (long long)a.max_copies * c.n_pools * c.pieces;
    hipLaunchKernelGGL(palu_copy_pages_kernel, dim3((unsigned)std::min<long long>(units, 2048)), dim3(256), 0, s, c);
    if (int rc = launched(who, "copy")) return rc;
  }
  return PALU_OK;
}

}  // namespace

extern "C" int palu_latent_fill_paged(void* cache_pages, const void* rows, long long row_stride, long long group_stride,
                                      const int32_t* cu_seqlens, const int32_t* start_pos, const int32_t* page_table, int n_rows,
                                      int batch, int n_groups, int num_pages, int page_size, int max_pages_per_seq, int width,
                                      int cache_layout, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_latent_fill_paged";
  if (!cache_pages || !rows || !cu_seqlens) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  int shift = 0;
  if (int rc = palu::check_pages(page_table, num_pages, page_size, max_pages_per_seq, &shift, who)) return rc;
  if (n_rows <= 0 || batch <= 0 || n_groups <= 0)
    return fail(PALU_EINVAL, "%s: row, sequence and group counts must be positive, got %d, %d, %d", who, n_rows, batch, n_groups);
  if (cache_layout != PALU_LAYOUT_ROWS && cache_layout != PALU_LAYOUT_TILED && cache_layout != PALU_LAYOUT_TILED_V)
    return fail(PALU_EINVAL, "%s: cache layout must be PALU_LAYOUT_ROWS, _TILED or _TILED_V, got %d", who, cache_layout);
  const int step = cache_layout == PALU_LAYOUT_ROWS ? 8 : 16;
  if (width <= 0 || width % step || width > 512)
    return fail(PALU_EINVAL, "%s: width must be a multiple of %d up to 512, got %d", who, step, width);
  if (row_stride < 0 || row_stride % 8 || group_stride < 0 || group_stride % 8)
    return fail(PALU_EINVAL, "%s: source strides must be non-negative multiples of 8, got %lld and %lld", who, row_stride,
                group_stride);
  if (!al16(cache_pages) || !al16(rows)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  if (n_rows > (1 << 28) || batch > 65535 || n_groups > 65535) return fail(PALU_EUNSUPPORTED, "%s: counts exceed the grid", who);
  FillArgs a{static_cast<__bf16*>(cache_pages), static_cast<const __bf16*>(rows), row_stride, group_stride, cu_seqlens, start_pos,
             page_table, n_rows, batch, n_groups, width, num_pages, shift, max_pages_per_seq, 0};
  a.gpw = std::min(n_groups, std::max(1, 8192 / (32 * width)));   // 4 vectors of 8 a thread
  // A sequence of n rows touches at most n / 32 + 2 blocks, and at most n.
  const dim3 grid((unsigned)std::min<long long>(n_rows, n_rows / 32 + 2LL * batch), (unsigned)((n_groups + a.gpw - 1) / a.gpw));
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, a); };
  if (cache_layout == PALU_LAYOUT_TILED) go(palu_fill_pages_kernel<PALU_LAYOUT_TILED>);
  else if (cache_layout == PALU_LAYOUT_TILED_V) go(palu_fill_pages_kernel<PALU_LAYOUT_TILED_V>);
  else go(palu_fill_pages_kernel<PALU_LAYOUT_ROWS>);
  return launched(who, "fill");
}

extern "C" size_t palu_pages_workspace_bytes(int batch, int num_pages) {
  if (batch <= 0 || num_pages <= 0) return 0;
  // the copies' number, their pages (an update copies at most one page a row, a compaction at most half of all) and a page list
  return 16 + 4 * (2 * (size_t)std::max(batch, num_pages / 2 + 1) + (size_t)num_pages);
}

extern "C" int palu_pages_update(const int32_t* page_table, const int32_t* lengths, const int32_t* parents,
                                 const int32_t* new_lengths, int32_t* page_table_out, int32_t* lengths_out, void* const* pools,
                                 const long long* page_bytes, int n_pools, int batch, int num_pages, int page_size,
                                 int max_pages_per_seq, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_pages_update";
  if (int rc = check_table(page_table, lengths, page_table_out, batch, max_pages_per_seq, num_pages, page_size, workspace,
                           workspace_bytes, palu_pages_workspace_bytes(batch, num_pages), who))
    return rc;
  if (!lengths_out || lengths_out == lengths) return fail(PALU_EINVAL, "%s: lengths_out must be memory of its own", who);
  if (int rc = check_pools(pools, page_bytes, n_pools, who)) return rc;
  if (batch > 4096 || update_lds(batch, num_pages) > PLAN_LDS)
    return fail(PALU_EUNSUPPORTED, "%s: %d rows (at most 4096) over %d pages exceed the plan's LDS", who, batch, num_pages);
  const PlanArgs a{page_table, lengths, parents, new_lengths, page_table_out, lengths_out, batch, max_pages_per_seq, num_pages,
                   page_size, log2_of(page_size), hash_entries(batch), static_cast<int32_t*>(workspace),
                   std::max(batch, num_pages / 2 + 1)};
  const size_t lds = update_lds(batch, num_pages);
  if (lds > (64 << 10)) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(palu_update_pages_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, PLAN_LDS);
    if (e != hipSuccess) return fail(PALU_EHIP, "%s: LDS attribute: %s", who, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(palu_update_pages_kernel, dim3(1), dim3(PLAN_THREADS), lds, stream, a);
  if (int rc = launched(who, "plan")) return rc;
  return launch_copies(a, pools, page_bytes, n_pools, who, stream);
}

extern "C" int palu_pages_compact(const int32_t* page_table, const int32_t* lengths, int32_t* page_table_out, int32_t* n_live,
                                  void* const* pools, const long long* page_bytes, int n_pools, int batch, int num_pages,
                                  int page_size, int max_pages_per_seq, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_pages_compact";
  if (int rc = check_table(page_table, lengths, page_table_out, batch, max_pages_per_seq, num_pages, page_size, workspace,
                           workspace_bytes, palu_pages_workspace_bytes(batch, num_pages), who))
    return rc;
  if (!n_live) return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  if (int rc = check_pools(pools, page_bytes, n_pools, who)) return rc;
  const size_t lds = 4 * ((size_t)(num_pages + 31) / 32);
  if (lds > PLAN_LDS) return fail(PALU_EUNSUPPORTED, "%s: %d pages exceed the plan's LDS", who, num_pages);
  const PlanArgs a{page_table, lengths, nullptr, nullptr, page_table_out, nullptr, batch, max_pages_per_seq, num_pages,
                   page_size, log2_of(page_size), 0, static_cast<int32_t*>(workspace), std::max(batch, num_pages / 2 + 1)};
  if (lds > (64 << 10)) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(palu_compact_pages_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, PLAN_LDS);
    if (e != hipSuccess) return fail(PALU_EHIP, "%s: LDS attribute: %s", who, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(palu_compact_pages_kernel, dim3(1), dim3(PLAN_THREADS), lds, stream, a, n_live);
  if (int rc = launched(who, "plan")) return rc;
  return launch_copies(a, pools, page_bytes, n_pools, who, stream);
}
