// Log probabilities of given tokens, the entropy of the distribution and its top entries, from rows of logits:
//   lp = x_t - m - log Z,   Z = sum exp(x - m),   H = log Z - sum exp(x - m) (x - m) / Z,   m = max x.
// One pass: every lane keeps its own running maximum, sum and weighted sum, rescaled when the maximum rises, and
// every wave the largest entries of what it has read, one per lane and sorted, which an entry joins only if it beats the
// last of them. Among equal values the lower index comes first; NaN counts above every number (as in the greedy
// pick), and makes the log probabilities and the entropy NaN. Bound by the logits' bytes (4096 rows of 128256 bf16, top 1:
// 171 us, 6.1 TB/s); of few rows, which are cut into parts for as many workgroups as the chip holds and joined by a second
// launch, by latency (64 rows fp32, top 20: 13.7 + 5.3 us, 7.2 + 1.7 without a top; one row, top 5: 6.2 + 3.4).
#include "palu_kernel.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int SCORE_TOP = 64;             // entries of a wave's list, one a lane
constexpr int SCORE_WAVES = 4;            // of a workgroup
constexpr int SCORE_WGS = 2048;           // workgroups that the chip holds at once
constexpr int SCORE_PART = 8192;          // logits of a row's part, about, at least: 32 a lane
constexpr int SCORE_PARTS = 32;           // of a row, at most
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct ScoreArgs {
  const void* x;
  long long ld;
  const int64_t* tokens;
  int rows, n, top;
  float* lp;
  float* ent;
  float* top_lp;                          // [rows][top]
  int64_t* top_id;
  int parts;                              // of a row
  char* ws;                               // parts > 1: a record per (row, part), its Stats (16 bytes) and `top` entries
};
// Bytes of a record: whole 16s, so that every Stats lies as its type says.
__host__ __device__ constexpr int record_bytes(int top) { return 16 + 8 * (top + (top & 1)); }

// Entries compare as (value, lower index first): one 64-bit key, value made order-preserving above, complemented index below.
// -0 counts as 0 and every NaN as one value.
__device__ __forceinline__ unsigned order_key(unsigned b) {   // of a float's bits
  const unsigned k = b & 0x80000000u ? (b == 0x80000000u ? b : ~b) : b | 0x80000000u;
  return (b & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu : k;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k == 0xffffffffu ? 0x7fc00000u : k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
typedef unsigned long long u64;
__device__ __forceinline__ u64 entry(unsigned bits, int i) { return (u64)order_key(bits) << 32 | (unsigned)~i; }

__device__ __forceinline__ u64 lane_of(u64 v, int lane) {   // the entry of a uniform lane
  const unsigned lo = __builtin_amdgcn_readlane((unsigned)v, lane), hi = __builtin_amdgcn_readlane((unsigned)(v >> 32), lane);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 lane_before(u64 v) {       // the entry of the lane before (lane 0: none)
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (unsigned)v, 0x138, 0xf, 0xf, false);   // wave_shr 1
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (unsigned)(v >> 32), 0x138, 0xf, 0xf, false);
  return (u64)hi << 32 | lo;
}

struct __attribute__((aligned(16))) Stats {
  float m, z, e;                          // maximum, sum of p = exp(x - m), sum of p log2 p
};
// (log2 p is bounded below where it multiplies: p is 0 there, and -infinity times 0 is NaN.)
__device__ __forceinline__ float log2p(float x, float m) { return __builtin_elementwise_maximum((x - m) * LOG2E, -1000.f); }

// f over all lanes: within rows of 16 by DPP (a shuffle would go through LDS), then the four rows.
template <typename F>
__device__ __forceinline__ float over_lanes(float x, F f) {
  auto dpp = [&](auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = f(x, dpp(std::integral_constant<int, 0xb1>{}));     // lanes 1 apart, 2 apart,
  x = f(x, dpp(std::integral_constant<int, 0x4e>{}));
  x = f(x, dpp(std::integral_constant<int, 0x141>{}));    // the halves of 8, of 16, mirrored
  x = f(x, dpp(std::integral_constant<int, 0x140>{}));
  auto row = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); };
  return f(f(row(0), row(16)), f(row(32), row(48)));
}

// The lanes' statistics as one.
__device__ __forceinline__ Stats join(const Stats& s) {
  const float m = over_lanes(s.m, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
  const float t = log2p(s.m, m == NEG_INF ? 0.f : m), c = __builtin_amdgcn_exp2f(t);
  auto sum = [](float a, float b) { return a + b; };
  return Stats{m, over_lanes(c * s.z, sum), over_lanes(c * fmaf(t, s.z, s.e), sum)};
}

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
  static constexpr int N = 8;
  typedef bf16x8 V;
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  typedef f32x4 V;
};

// The largest value bits t, to 16 bits, that at least `top` of the lanes' `n` keys (R of each, 0: none) reach. BITS at a time:
// two where a wave has its SIMD to itself (the counts of three candidates are independent; the join of 64 rows took 5.1 us in
// place of 5.8), one where waves share it (three counts are more work; 300 rows took 31 us in place of 34).
template <int R, int BITS>
__device__ __forceinline__ unsigned reached_by(const unsigned (&k)[R], int n, int top) {
  unsigned t = 0;
  for (int bit = 32 - BITS; bit >= 16; bit -= BITS) {
    int m[1 << BITS] = {};
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (64 * r < n)
#pragma unroll
        for (int d = 1; d < 1 << BITS; ++d) m[d] += __popcll(__ballot(k[r] >= (t | (unsigned)d << bit)));
    unsigned most = 0;
#pragma unroll
    for (int d = 1; d < 1 << BITS; ++d) most = m[d] >= top ? d : most;
    t |= most << bit;
  }
  return t;
}

// The largest `top` of `n` lists of `top` entries in LDS (0: none; no two others are equal), each with its place:
// use(place, entry). What is left above reached_by is placed by the number of larger ones. At most 64 R entries; `left` and
// `count`: LDS for as many and a counter. Returns how many are left.
template <int R, typename F>
__device__ __forceinline__ int merge_lists(const u64* lists, int n, int top, u64* left, int* count, F use) {
  const int all = n * top, lane = threadIdx.x & 63;
  if (threadIdx.x == 0) *count = 0;
  unsigned t = 0;
  if (all > 128) {                        // (of fewer the search costs more than the places of all)
    unsigned k[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned x = (unsigned)(lists[min(64 * r + lane, all - 1)] >> 32);
      k[r] = 64 * r + lane < all ? x : 0;
    }
    t = reached_by<R, 2>(k, all, top);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < all; i += SCORE_WAVES * 64) {
    const u64 x = lists[i];
    if (x != 0 && (unsigned)(x >> 32) >= t) left[atomicAdd(count, 1)] = x;   // in any order: places go by the entries
  }
  __syncthreads();
  const int m = *count;
  for (int i = threadIdx.x; i < m; i += SCORE_WAVES * 64) {
    const u64 x = left[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < m; ++j) place += left[j] > x;
    if (place < top) use(place, x);
  }
  return m;
}

// The row's results from its whole statistics and the sorted lists of its parts.
template <int R>
__device__ __forceinline__ void finish_row(const ScoreArgs& a, long long row, const Stats& st, float token_logit, const u64* lists,
                                           int n, u64* left, int* count) {
  const float logz = __builtin_amdgcn_logf(st.z) * LN2;    // log2 Z, in natural units
  if (threadIdx.x == 0) {
    const long long t = a.tokens[row];
    a.lp[row] = t < 0 ? 0.f : t >= a.n ? __builtin_nanf("") : (token_logit - st.m) - logz;
    a.ent[row] = logz - st.e / st.z * LN2;
  }
  if (a.top)
    merge_lists<R>(lists, n, a.top, left, count, [&](int place, u64 k) {
      a.top_lp[row * a.top + place] = (key_value((unsigned)(k >> 32)) - st.m) - logz;
      a.top_id[row * a.top + place] = (int64_t)(unsigned)~(unsigned)k;
    });
}

template <typename T>
__global__ __launch_bounds__(SCORE_WAVES * 64) void palu_score_kernel(const ScoreArgs a) {
  constexpr int N = Vec<T>::N, U = 32 / N;                 // a lane's vectors in flight: 32 entries
  typedef typename Vec<T>::V V;
  __shared__ u64 lists[SCORE_WAVES * SCORE_TOP], left[SCORE_WAVES * SCORE_TOP];
  __shared__ Stats stats[SCORE_WAVES];
  __shared__ unsigned maxima[2][SCORE_WAVES * 64];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int part = blockIdx.x % a.parts;
  const long long row = blockIdx.x / a.parts;
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  // Vector v holds entries N v - skew .. + N - 1, so that whole vectors are aligned; the row's ends are read one by one.
  const int skew = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % N);
  const int nv = (a.n + skew + N - 1) / N, share = (nv + a.parts - 1) / a.parts;
  const int v_lo = min(nv, part * share), v_hi = min(nv, v_lo + share);
  float token_logit = 0.f;
  if (tid == 0) {
    const long long t = a.tokens[row];
    if (t >= 0 && t < a.n) token_logit = (float)x[t];
  }
  Stats st{NEG_INF, 0.f, 0.f};
  u64 mine = 0, least = 0;                // entry `lane` of the wave's list (0: none), and the last of its `top`
  float bound = NEG_INF;                  // no entry below it can be among the top
  int turn = 0;
  for (int vc = v_lo; vc < v_hi; vc += SCORE_WAVES * 64 * U, ++turn) {   // uniform: all waves take every turn
    const int v0 = vc + w * 64 * U;
    // Whole vectors first, all loads at once; then the entries of the row's ends.
    V q[U];
    bool ends = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * 64 + lane, e0 = v * N - skew;
      const bool whole = v < v_hi && e0 >= 0 && e0 + N <= a.n;
      ends = ends || (v < v_hi && !whole);
#pragma unroll
      for (int i = 0; i < N; ++i) q[u][i] = (T)NEG_INF;
      if (whole) q[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(x + e0));
    }
    if (__any(ends)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = v0 + u * 64 + lane, e0 = v * N - skew;
        if (v < v_hi && (e0 < 0 || e0 + N > a.n))
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (e0 + i >= 0 && e0 + i < a.n) q[u][i] = x[e0 + i];
      }
    }
    float f[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) f[u][i] = (float)q[u][i];
    float mx = f[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) mx = __builtin_elementwise_maximum(mx, f[u][i]);
    const float m = __builtin_elementwise_maximum(st.m, mx), ref = m == NEG_INF ? 0.f : m;
    const float t0 = log2p(st.m, ref), c0 = __builtin_amdgcn_exp2f(t0);
    st.e = c0 * fmaf(t0, st.z, st.e);
    st.z *= c0;
    st.m = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float t = log2p(f[u][i], ref), p = __builtin_amdgcn_exp2f(t);
        st.z += p;
        st.e = fmaf(t, p, st.e);
      }
    if (a.top == 0) continue;
    if ((turn & (turn + 1)) == 0) {
      // The top-th largest of all lanes' maxima so far bounds the top-th entry from below. Found bit by bit, to 16 bits, at turns
      // 0, 1, 3, 7, .., it leaves about `top` entries a time for the workgroup's lists (each wave by its own entries: 5.6
      // times as many, at 20 of 2048).
      unsigned* const keys = maxima[(31 - __builtin_clz(turn + 1)) & 1];
      keys[tid] = order_key(__float_as_uint(st.m));
      __syncthreads();
      unsigned k4[SCORE_WAVES];
#pragma unroll
      for (int r = 0; r < SCORE_WAVES; ++r) k4[r] = keys[64 * r + lane];
      const unsigned t = reached_by<SCORE_WAVES, 1>(k4, SCORE_WAVES * 64, a.top);
      if (t > order_key(0xff800000u)) bound = __builtin_elementwise_maximum(bound, key_value(t));
    }
    // Values compare as floats, NaN above all: !(x < bound).
    if (!__any(!(mx < bound))) continue;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u64 who = __ballot(!(f[u][i] < bound));
        if (!who) continue;
        // What beats the last of the list joins it, lane by lane; against the risen last the lanes compare again, so that a row
        // of equal values (most of it masked) costs no more than what joins.
        const int v = v0 + u * 64 + lane, idx = v * N - skew + i;
        const u64 c = v < v_hi && idx >= 0 && idx < a.n ? entry(__float_as_uint(f[u][i]), idx) : 0;
        while ((who &= __ballot(c > least))) {
          const u64 x = lane_of(c, __builtin_ctzll(who));
          who &= who - 1;
          // the lanes that hold less move on by one, the first of them takes the entry
          const u64 up = lane_before(mine);
          if (mine < x) mine = lane > 0 && up < x ? up : x;
          least = lane_of(mine, a.top - 1);
        }
      }
    if (least) bound = __builtin_elementwise_maximum(bound, key_value((unsigned)(least >> 32)));
  }
  st = join(st);
  if (lane == 0) stats[w] = st;
  if (lane < a.top) lists[w * a.top + lane] = mine;
  __syncthreads();
  st = join(lane < SCORE_WAVES ? stats[lane] : Stats{NEG_INF, 0.f, 0.f});
  if (a.parts == 1) {
    finish_row<SCORE_WAVES>(a, row, st, token_logit, lists, SCORE_WAVES, left, &count);
    return;
  }
  char* ws = a.ws + (long long)blockIdx.x * record_bytes(a.top);
  if (tid == 0) *reinterpret_cast<Stats*>(ws) = st;
  if (a.top) {
    u64* out = reinterpret_cast<u64*>(ws + 16);
    const int m = merge_lists<SCORE_WAVES>(lists, SCORE_WAVES, a.top, left, &count, [&](int place, u64 k) { out[place] = k; });
    if (m + tid < a.top) out[m + tid] = 0;
  }
}

// The parts of a row, a workgroup to a row.
template <typename T>
__global__ __launch_bounds__(SCORE_WAVES * 64) void palu_score_join_kernel(const ScoreArgs a) {
  extern __shared__ u64 lists[];          // [parts][top], and as much for what is left of them
  __shared__ int count;
  const long long row = blockIdx.x;
  const int record = record_bytes(a.top);
  const char* ws = a.ws + row * a.parts * record;
  float token_logit = 0.f;
  if (threadIdx.x == 0) {
    const long long t = a.tokens[row];
    if (t >= 0 && t < a.n) token_logit = (float)static_cast<const T*>(a.x)[row * a.ld + t];
  }
  const int lane = threadIdx.x & 63;
  Stats st{NEG_INF, 0.f, 0.f};
  if (lane < a.parts) st = *reinterpret_cast<const Stats*>(ws + lane * record);
  u64 x[SCORE_PARTS / SCORE_WAVES];       // all loads at once: each comes from another XCD's writes, by way of memory
#pragma unroll
  for (int i = 0; i < SCORE_PARTS / SCORE_WAVES; ++i) {
    const int p = i * SCORE_WAVES + (threadIdx.x >> 6);
    x[i] = 0;
    if (p < a.parts && lane < a.top) x[i] = reinterpret_cast<const u64*>(ws + p * record + 16)[lane];
  }
#pragma unroll
  for (int i = 0; i < SCORE_PARTS / SCORE_WAVES; ++i) {
    const int p = i * SCORE_WAVES + (threadIdx.x >> 6);
    if (p < a.parts && lane < a.top) lists[p * a.top + lane] = x[i];
  }
  st = join(st);
  __syncthreads();
  u64* left = lists + a.parts * a.top;
  if (a.parts * a.top <= 64 * 8) finish_row<8>(a, row, st, token_logit, lists, a.parts, left, &count);
  else finish_row<SCORE_PARTS>(a, row, st, token_logit, lists, a.parts, left, &count);
}

int score_parts(int rows, int n) {
  return std::max(1, std::min({SCORE_WGS / rows, (n + SCORE_PART - 1) / SCORE_PART, SCORE_PARTS}));
}

template <typename T>
int launch_score(const ScoreArgs& a, const char* who, hipStream_t s) {
  hipLaunchKernelGGL((palu_score_kernel<T>), dim3((unsigned)a.rows * a.parts), dim3(SCORE_WAVES * 64), 0, s, a);
  if (a.parts > 1 && hipPeekAtLastError() == hipSuccess)
    hipLaunchKernelGGL((palu_score_join_kernel<T>), dim3(a.rows), dim3(SCORE_WAVES * 64), 16 * a.parts * a.top, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PALU_OK : fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
}

bool score_dims_ok(int rows, int n, int top) { return rows > 0 && n > 0 && top >= 0 && top <= SCORE_TOP && top <= n; }

}  // namespace

extern "C" size_t palu_token_logprobs_workspace_bytes(int rows, int n, int top) {
  if (!score_dims_ok(rows, n, top)) return 0;
  const int parts = score_parts(rows, n);
  return parts == 1 ? 0 : (size_t)rows * parts * record_bytes(top);
}

extern "C" int palu_token_logprobs(const void* logits, long long ld, int dtype, const int64_t* tokens, int rows, int n, int top,
                                   float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_token_logprobs";
  if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  if (rows <= 0 || n <= 0 || ld < 0) return fail(PALU_EINVAL, "%s: rows and n must be positive, got %d and %d", who, rows, n);
  if (n > (1 << 30) || rows > (1 << 23)) return fail(PALU_EUNSUPPORTED, "%s: %d rows of %d logits", who, rows, n);
  if (dtype != PALU_DTYPE_F32 && dtype != PALU_DTYPE_BF16)
    return fail(PALU_EINVAL, "%s: dtype must be PALU_DTYPE_F32 or PALU_DTYPE_BF16, got %d", who, dtype);
  if (!score_dims_ok(rows, n, top)) return fail(PALU_EINVAL, "%s: top = %d (0 .. %d, at most n)", who, top, SCORE_TOP);
  const size_t need = palu_token_logprobs_workspace_bytes(rows, n, top);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(PALU_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes needed (palu_token_logprobs_workspace_bytes), got %zu",
                who, need, workspace ? workspace_bytes : 0);
  const ScoreArgs a{logits, ld, tokens, rows, n, top, logprob, entropy, top_logprobs, top_ids, score_parts(rows, n),
                    static_cast<char*>(workspace)};
  return dtype == PALU_DTYPE_BF16 ? launch_score<__bf16>(a, who, stream) : launch_score<float>(a, who, stream);
}
