// Log probabilities of given tokens, the entropy of the distribution and its top entries, from rows of logits:
//   lp = x_t - m - log Z,   Z = sum exp(x - m),   H = log Z - sum exp(x - m) (x - m) / Z,   m = max x.
// One pass: every lane keeps its own running maximum, sum and weighted sum, rescaled when the maximum rises, and
// every wave the largest entries of what it has read, one per lane and sorted, which an entry joins only if it beats the
// last of them. Among equal values the lower index comes first; NaN counts above every number (as in the greedy
// pick), and makes the log probabilities and the entropy NaN. Bound by the logits' bytes.
#include "palu_kernel.h"

#include <algorithm>

namespace {

constexpr int SCORE_TOP = 64;             // entries of a wave's list, one a lane
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
};

// Entries compare as (value, lower index first): one 64-bit key, value made order-preserving above, complemented index below.
// -0 counts as 0 and every NaN as one value.
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);             // -0 + 0 = +0
  const unsigned k = b & 0x80000000u ? ~b : b | 0x80000000u;
  return x != x ? 0xffffffffu : k;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k == 0xffffffffu ? 0x7fc00000u : k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
typedef unsigned long long u64;
__device__ __forceinline__ u64 entry(float x, int i) { return (u64)order_key(x) << 32 | (unsigned)~i; }

__device__ __forceinline__ u64 shfl64(u64 v, int lane) {
  const unsigned lo = __shfl((unsigned)v, lane, 64), hi = __shfl((unsigned)(v >> 32), lane, 64);
  return (u64)hi << 32 | lo;
}

struct Stats {
  float m, z, e;                          // maximum, sum of p = exp(x - m), sum of p log2 p
};
// (log2 p is bounded below where it multiplies: p is 0 there, and -infinity times 0 is NaN.)
__device__ __forceinline__ float log2p(float x, float m) { return __builtin_elementwise_maximum((x - m) * LOG2E, -1000.f); }

__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const float m = __builtin_elementwise_maximum(a.m, b.m), ref = m == NEG_INF ? 0.f : m;
  const float ta = log2p(a.m, ref), tb = log2p(b.m, ref);
  const float ca = __builtin_amdgcn_exp2f(ta), cb = __builtin_amdgcn_exp2f(tb);
  return Stats{m, ca * a.z + cb * b.z, ca * fmaf(ta, a.z, a.e) + cb * fmaf(tb, b.z, b.e)};
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

template <typename T, int NW>
__global__ __launch_bounds__(NW * 64) void palu_score_kernel(const ScoreArgs a) {
  constexpr int N = Vec<T>::N, U = 32 / N;                 // a lane's vectors in flight: 32 entries
  typedef typename Vec<T>::V V;
  __shared__ u64 lists[NW * SCORE_TOP];
  __shared__ Stats stats[NW];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  // Vector v holds entries N v - skew .. + N - 1, so that whole vectors are aligned; the row's ends are read one by one.
  const int skew = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % N);
  const int nv = (a.n + skew + N - 1) / N;
  Stats st{NEG_INF, 0.f, 0.f};
  u64 mine = 0;                           // entry `lane` of the wave's list (0: none), and its last entry
  u64 least = 0;
  for (int v0 = w * 64 * U; v0 < nv; v0 += NW * 64 * U) {
    float f[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e0 = (v0 + u * 64 + lane) * N - skew;
      if (e0 >= 0 && e0 + N <= a.n) {
        const V q = __builtin_nontemporal_load(reinterpret_cast<const V*>(x + e0));
#pragma unroll
        for (int i = 0; i < N; ++i) f[u][i] = (float)q[i];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[u][i] = e0 + i >= 0 && e0 + i < a.n ? (float)x[e0 + i] : NEG_INF;
      }
    }
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
    if (a.top && __any(order_key(mx) >= (unsigned)(least >> 32))) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int idx = (v0 + u * 64 + lane) * N - skew + i;
          const u64 k = idx >= 0 && idx < a.n ? entry(f[u][i], idx) : 0;
          u64 who = __ballot(k > least);
          while (who) {
            const int l = __builtin_ctzll(who);
            const u64 c = shfl64(k, l);
            // the lanes that hold less move on by one, the first of them takes the entry
            const u64 up = shfl64(mine, max(lane - 1, 0));
            const u64 up_less = lane > 0 && up < c;
            if (mine < c) mine = up_less ? up : c;
            least = shfl64(mine, a.top - 1);
            who &= who - 1;
            who &= __ballot(k > least);
          }
        }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
    st = join(st, Stats{__shfl_xor(st.m, o, 64), __shfl_xor(st.z, o, 64), __shfl_xor(st.e, o, 64)});
  if (lane == 0) stats[w] = st;
  if (lane < a.top) lists[w * a.top + lane] = mine;
  __syncthreads();
  st = stats[0];
  for (int i = 1; i < NW; ++i) st = join(st, stats[i]);
  const float logz = __builtin_amdgcn_logf(st.z) * LN2;    // log2 Z, in natural units
  if (tid == 0) {
    const long long t = a.tokens[row];
    a.lp[row] = t < 0 ? 0.f : t >= a.n ? __builtin_nanf("") : ((float)x[t] - st.m) - logz;
    a.ent[row] = logz - st.e / st.z * LN2;
  }
  // An entry's place among all lists is the number of larger ones (no two are equal).
  const int all = NW * a.top;
  for (int i = tid; i < all; i += NW * 64) {
    const u64 k = lists[i];
    if (k == 0) continue;
    int place = 0;
    for (int j = 0; j < all; ++j) place += lists[j] > k;
    if (place < a.top) {
      a.top_lp[row * a.top + place] = (key_value((unsigned)(k >> 32)) - st.m) - logz;
      a.top_id[row * a.top + place] = (int64_t)(unsigned)~(unsigned)k;
    }
  }
}

}  // namespace

extern "C" int palu_token_logprobs(const void* logits, long long ld, int dtype, const int64_t* tokens, int rows, int n, int top,
                                   float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_token_logprobs";
  if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return fail(PALU_EINVAL, "%s: a required pointer is null", who);
  if (rows <= 0 || n <= 0 || ld < 0) return fail(PALU_EINVAL, "%s: rows and n must be positive, got %d and %d", who, rows, n);
  if (n > (1 << 30)) return fail(PALU_EUNSUPPORTED, "%s: rows of %d logits", who, n);
  if (dtype != PALU_DTYPE_F32 && dtype != PALU_DTYPE_BF16)
    return fail(PALU_EINVAL, "%s: dtype must be PALU_DTYPE_F32 or PALU_DTYPE_BF16, got %d", who, dtype);
  if (top < 0 || top > SCORE_TOP || top > n) return fail(PALU_EINVAL, "%s: top = %d (0 .. %d, at most n)", who, top, SCORE_TOP);
  const ScoreArgs a{logits, ld, tokens, rows, n, top, logprob, entropy, top_logprobs, top_ids};
  const bool few = rows < 512;            // a row to a CU: its waves share the row
  if (dtype == PALU_DTYPE_BF16) {
    if (few) hipLaunchKernelGGL((palu_score_kernel<__bf16, 16>), dim3(rows), dim3(1024), 0, stream, a);
    else hipLaunchKernelGGL((palu_score_kernel<__bf16, 4>), dim3(rows), dim3(256), 0, stream, a);
  } else {
    if (few) hipLaunchKernelGGL((palu_score_kernel<float, 16>), dim3(rows), dim3(1024), 0, stream, a);
    else hipLaunchKernelGGL((palu_score_kernel<float, 4>), dim3(rows), dim3(256), 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PALU_EHIP, "%s launch: %s", who, hipGetErrorString(e));
  return PALU_OK;
}
