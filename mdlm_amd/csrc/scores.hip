// Token scores of the SUBS rows (diffusion.py:261-277) without the table: the
// log-probability of a given token, the entropy, the log-sum-exp and the k best
// alternatives of every row, and the gradient of the three.
//
// With x the logits of a masked row, the mask token's column excluded, m = max x,
// y = x - m, Z = sum e^y:
//   l_v = y_v - log Z,   H = log Z - (sum e^y y) / Z   (two non-negative terms)
//   d/dx_v = g [v = x0] + sum_j g_j [v = top_j] - (g + sum_j g_j) p_v - gH p_v (l_v + H)
// Both directions read a row once (the alternatives look at a few threads' share
// of it again): bound by HBM.
#include "common.h"

namespace mdlm {

constexpr float SC_L2E = 1.4426950408889634f;
constexpr float SC_LN2 = 0.6931471805599453f;
constexpr float SC_NEG = -1000000.f;      // Diffusion.neg_infinity
constexpr int SC_MAX_K = 64;
// Up to so many rows a workgroup has a CU to itself and its latency counts: 1024 threads, if
// the row has a chunk for each.  Measured, us (256 / 1024 threads, bf16, 50258 columns): 64 rows with
// 8 alternatives 20 / 16, 1024 rows 32 / 44; gradient of 64 rows of 128000 columns 26 / 14.
constexpr int64_t SC_WIDE_ROWS = 256;
constexpr int SC_WIDE_BYTES = 16 * 1024;

// order of the alternatives: larger logit first (NaN above all, -0 = +0), then
// the lower index; unique per column, 0 for none
__device__ __forceinline__ unsigned long long score_key(float x, int v) {
  const unsigned u = __float_as_uint(x + 0.f);
  unsigned o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if (x != x) o = 0xffffffffu;
  return ((unsigned long long)o << 32) | (unsigned)(0x7fffffff - v);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return 0x7fffffff - (int)(unsigned)k; }

__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  return v;
}

// A position that is not masked: log-probability 0 for its own token (and for what is
// no token), -1e6 for every other one; the alternatives are its token and the lowest other ids.
__device__ __forceinline__ void known_row(int64_t r, int64_t tok, const int64_t* x0, float* logp, float* ent, float* lse,
                                          float* top_logp, int64_t* top_ids, int V, int mask, int k, int tid) {
  if (tid == 0) {
    const int64_t tgt = x0[r];
    logp[r] = tgt == tok || tgt < 0 || tgt >= V ? 0.f : SC_NEG;
    ent[r] = 0.f;
    lse[r] = 0.f;
  }
  if (tid < k) {
    int64_t id = tok;
    if (tid > 0) {
      id = tid - 1;
      const int64_t t = (tok >= 0 && tok < V) ? tok : mask;
      const int64_t lo = t < mask ? t : mask, hi = t < mask ? mask : t;
      if (id >= lo) ++id;
      if (hi != lo && id >= hi) ++id;
    }
    top_ids[r * k + tid] = id;
    top_logp[r * k + tid] = tid == 0 ? 0.f : SC_NEG;
  }
}

// A row's elements as 16-byte chunks that start on 16-byte addresses, wherever the
// row starts: `head` elements before the first, n chunks, `tail` elements behind.
template <typename T>
struct RowSpan {
  static constexpr int E = 16 / sizeof(T);
  int head, n, tail;
  int mask_chunk, mask_elem;      // where the mask column is (-1: not in a chunk)
  __device__ RowSpan(const T* p, int V, int mask) {
    head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    head = head < V ? head : V;
    n = (V - head) / E;
    tail = V - head - n * E;
    const int c = mask - head;
    mask_chunk = c >= 0 && c < n * E ? c / E : -1;
    mask_elem = c - mask_chunk * E;
  }
  // element handled alone by thread t < head + tail
  __device__ int single(int t) const { return t < head ? t : n * E + t; }
};
template <typename T, typename F>
__device__ __forceinline__ void unpack16(const uint4& q, F& f);
template <> __device__ __forceinline__ void unpack16<float, float[4]>(const uint4& q, float (&f)[4]) {
  f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
}
template <> __device__ __forceinline__ void unpack16<bf16_t, float[8]>(const uint4& q, float (&f)[8]) {
  const unsigned u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = __uint_as_float(u[k] << 16);
    f[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
  }
}

// Running maximum and sums of one thread, in units of log 2:
//   s = sum 2^t, s1 = sum 2^t t,  t = x log2(e) - m2,  m2 = fp32(m log2(e)).
// m starts at a finite value below every logit that counts, so that no infinity
// meets another; a row with nothing above it goes the slow way.
constexpr float SC_FLOOR = -1e30f;
// m2.  Rounded before any use: the compiler would fold the product into the differences of two m2,
// and what the sums were made with no longer cancels (1.2e-4 in a log-probability at logits of 1e4).
__device__ __forceinline__ float max_log2(float m) {
  float m2 = m * SC_L2E;
  asm("" : "+v"(m2));
  return m2;
}
struct Running {
  float m = SC_FLOOR, m2 = SC_FLOOR * SC_L2E, s = 0.f, s1 = 0.f;
  float next = SC_FLOOR;        // the largest maximum of any other chunk than `best`, which holds m
  int best = -1;
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N], int chunk) {
    float mx = f[0];
#pragma unroll
    for (int k = 1; k < N; ++k) mx = fmaxf(mx, f[k]);
    next = fmaxf(next, fminf(m, mx));
    if (mx > m) {
      best = chunk;
      const float n2 = max_log2(mx), d = m2 - n2, sc = __builtin_amdgcn_exp2f(d);
      s1 = __builtin_fmaf(d, s, s1) * sc;
      s *= sc;
      m = mx; m2 = n2;
    }
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float t = __builtin_fmaf(f[k], SC_L2E, -m2), e = __builtin_amdgcn_exp2f(t);
      a += e;
      b = __builtin_fmaf(e, t, b);
    }
    if (b != b) {               // 0 * inf: a logit of -inf (or of the lowest value) adds nothing
      b = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float t = __builtin_fmaf(f[k], SC_L2E, -m2), e = __builtin_amdgcn_exp2f(t);
        b += e == 0.f ? 0.f : e * t;
      }
    }
    s += a;
    s1 += b;
  }
};

template <int BLOCK>
struct ScoreShared {
  float m[BLOCK / 64], s[BLOCK / 64], s1[BLOCK / 64];
  float group[64];
  float tau;
  int count;
  static constexpr int CAP = 1024;
  unsigned long long cand[CAP];
  unsigned long long best[2][BLOCK / 64];
};

// The sums of a row straight from the definition (a row without a finite logit, or
// with a NaN): maximum first, differences instead of fused products.
template <typename T, int BLOCK>
__device__ void slow_stats(const T* row, int V, int mask, ScoreShared<BLOCK>& sh, float& m, float& s, float& s1) {
  const int tid = threadIdx.x, w = tid >> 6;
  __syncthreads();
  m = -INFINITY;
  for (int v = tid; v < V; v += BLOCK)
    if (v != mask) m = fmaxf(m, elem<T>::load(row + v));
  m = wave_max(m);
  if ((tid & 63) == 0) sh.m[w] = m;
  __syncthreads();
  for (int i = 0; i < BLOCK / 64; ++i) m = fmaxf(m, sh.m[i]);
  s = s1 = 0.f;
  for (int v = tid; v < V; v += BLOCK)
    if (v != mask) {
      const float x = elem<T>::load(row + v);
      const float t = m > -INFINITY ? (x - m) * SC_L2E : x;    // all -inf: nothing to add
      const float e = __builtin_amdgcn_exp2f(t);
      s += e;
      s1 += e == 0.f ? 0.f : e * t;
    }
  s = wave_sum(s); s1 = wave_sum(s1);
  if ((tid & 63) == 0) { sh.s[w] = s; sh.s1[w] = s1; }
  __syncthreads();
  s = s1 = 0.f;
  for (int i = 0; i < BLOCK / 64; ++i) { s += sh.s[i]; s1 += sh.s1[i]; }
}

// The k best columns one after another (candidates that do not fit, or NaN rows).
template <typename T, int BLOCK>
__device__ void slow_top(const T* row, int V, int mask, int k, float m, float lz, ScoreShared<BLOCK>& sh,
                         float* top_logp, int64_t* top_ids) {
  const int tid = threadIdx.x, w = tid >> 6;
  unsigned long long last = ~0ull;
  __syncthreads();
  for (int j = 0; j < k; ++j) {
    unsigned long long b = 0;
    for (int v = tid; v < V; v += BLOCK)
      if (v != mask) {
        const unsigned long long q = score_key(elem<T>::load(row + v), v);
        if (q < last && q > b) b = q;
      }
    b = wave_max_u64(b);
    if ((tid & 63) == 0) sh.best[j & 1][w] = b;
    __syncthreads();
    for (int i = 0; i < BLOCK / 64; ++i) b = sh.best[j & 1][i] > b ? sh.best[j & 1][i] : b;
    last = b;
    if (tid == 0) {
      const int v = key_index(b);
      top_ids[j] = v;
      top_logp[j] = (elem<T>::load(row + v) - m) - lz;
    }
  }
}

// One workgroup per row, one pass over it.
//
// Alternatives: the maxima of 64 groups of threads are at hand after the pass; the
// k-th largest of them, tau, is a lower bound of the k-th best logit (k groups
// reach it).  Only threads whose own maximum reaches tau look again (from the
// caches), at the one chunk that holds it unless another's maximum reaches tau
// too; a handful of columns pass, and each one's rank among them is its place.
// Ranks go by (logit, index) keys: the order in which the atomic hands out list
// places does not show.
//
// Measured on 8192 x 50258 bf16 with 8 alternatives: 157 us, 5.2 TB/s (the card
// copies at 4.6 and sums at 4.0); one row: 8 us, a row's latency.
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void subs_scores_kernel(
    const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ xt, const int64_t* __restrict__ x0,
    float* __restrict__ logp, float* __restrict__ ent, float* __restrict__ lse, float* __restrict__ top_logp,
    int64_t* __restrict__ top_ids, int V, int mask, int k) {
  // chunks in flight per thread: a whole row of the common vocabularies for the wide
  // workgroup, whose latency counts; the narrow ones hide theirs behind each other
  constexpr int E = RowSpan<T>::E, U = BLOCK == 1024 ? 8 : 4;
  __shared__ ScoreShared<BLOCK> sh;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, w = tid >> 6;
  const int64_t tok = xt[r];
  if (tok != mask) { known_row(r, tok, x0, logp, ent, lse, top_logp, top_ids, V, mask, k, tid); return; }
  const T* row = logits + r * ld;
  const RowSpan<T> sp(row, V, mask);
  const uint4* chunks = reinterpret_cast<const uint4*>(row + sp.head);
  const int64_t tgt = x0[r];
  float xtgt = 0.f;
  if (tid == 0) {
    sh.count = 0;
    if (tgt >= 0 && tgt < V) xtgt = elem<T>::load(row + tgt);
  }
  Running run;
  auto add_chunk = [&](const uint4& q, int i) {
    float f[E];
    unpack16<T>(q, f);
    if (i == sp.mask_chunk) {
#pragma unroll
      for (int e = 0; e < E; ++e) if (e == sp.mask_elem) f[e] = -INFINITY;
    }
    run.add(f, i);
  };
  for (int i = tid; i < sp.n; i += U * BLOCK) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) if (i + u * BLOCK < sp.n) q[u] = chunks[i + u * BLOCK];
#pragma unroll
    for (int u = 0; u < U; ++u) if (i + u * BLOCK < sp.n) add_chunk(q[u], i + u * BLOCK);
  }
  const int alone = tid < sp.head + sp.tail ? sp.single(tid) : -1;
  if (alone >= 0 && alone != mask) {
    const float f[1] = {elem<T>::load(row + alone)};
    run.add(f, -1);
  }
  // ---- across the workgroup
  const float own = run.m;
  const float wm = wave_max(own), wm2 = max_log2(wm);
  float s, s1;
  {
    const float d = run.m2 - wm2, sc = __builtin_amdgcn_exp2f(d);
    s = wave_sum(run.s * sc);
    s1 = wave_sum(__builtin_fmaf(d, run.s, run.s1) * sc);
  }
  if ((tid & 63) == 0) { sh.m[w] = wm; sh.s[w] = s; sh.s1[w] = s1; }
  if (k) {
    float gm = own;
#pragma unroll
    for (int o = 1; o < BLOCK / 64; o <<= 1) gm = fmaxf(gm, __shfl_xor(gm, o));
    if (tid % (BLOCK / 64) == 0) sh.group[tid / (BLOCK / 64)] = gm;
  }
  __syncthreads();
  float m = sh.m[0];
#pragma unroll
  for (int j = 1; j < BLOCK / 64; ++j) m = fmaxf(m, sh.m[j]);
  const float m2 = max_log2(m);
  s = s1 = 0.f;
#pragma unroll
  for (int j = 0; j < BLOCK / 64; ++j) {
    const float d = max_log2(sh.m[j]) - m2, sc = __builtin_amdgcn_exp2f(d);
    s1 += __builtin_fmaf(d, sh.s[j], sh.s1[j]) * sc;
    s += sh.s[j] * sc;
  }
  float off = __builtin_fmaf(m, SC_L2E, -m2);        // what the rounding of m2 moved s by
  const bool plain = s > 0.f;                        // workgroup-uniform; false for NaN too
  if (!plain) { slow_stats<T, BLOCK>(row, V, mask, sh, m, s, s1); off = 0.f; }
  // log Z and the entropy are not below 0, but for what the logarithm rounds where one token
  // has all the weight (NaN stays NaN)
  const float l2s = log2f(s);
  float lz = (l2s - off) * SC_LN2;
  if (lz < 0.f) lz = 0.f;
  if (tid == 0) {
    const float h = (l2s - s1 / s) * SC_LN2;
    lse[r] = m + lz;
    ent[r] = h < 0.f ? 0.f : h;
    // a row without a finite logit has no scores, not even the mask token's
    logp[r] = tgt < 0 || tgt >= V ? 0.f
              : m == -INFINITY   ? NAN
              : tgt == mask      ? (xtgt + SC_NEG) - (m + lz)
                                 : (xtgt - m) - lz;
  }
  if (k == 0) return;
  float* tl = top_logp + r * k;
  int64_t* ti = top_ids + r * k;
  int n = 0;
  if (plain) {
    if (w == 0) {
      const float g = sh.group[tid];
      int above = 0;
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
        above += (o > g || (o == g && j < tid)) ? 1 : 0;
      }
      if (above == k - 1) sh.tau = g;
    }
    __syncthreads();
    const float tau = sh.tau;
    if (own >= tau) {
      auto offer = [&](float x, int v) {
        if (x >= tau && v != mask) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < ScoreShared<BLOCK>::CAP) sh.cand[at] = score_key(x, v);
        }
      };
      const bool all = run.next >= tau;
      if (all || run.best < 0) { if (alone >= 0) offer(elem<T>::load(row + alone), alone); }
      const int last = all ? sp.n : run.best + 1;
      for (int c0 = all ? tid : run.best; c0 >= 0 && c0 < last; c0 += 8 * BLOCK) {
        uint4 q[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) if (c0 + u * BLOCK < last) q[u] = chunks[c0 + u * BLOCK];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (c0 + u * BLOCK < last) {
            float f[E];
            unpack16<T>(q[u], f);
#pragma unroll
            for (int e = 0; e < E; ++e) offer(f[e], sp.head + (c0 + u * BLOCK) * E + e);
          }
      }
    }
    __syncthreads();
    n = sh.count;
  }
  if (n < k || n > ScoreShared<BLOCK>::CAP) { slow_top<T, BLOCK>(row, V, mask, k, m, lz, sh, tl, ti); return; }
  for (int c = tid; c < n; c += BLOCK) {
    const unsigned long long key = sh.cand[c];
    int above = 0;
    for (int j = 0; j < n; ++j) above += sh.cand[j] > key ? 1 : 0;
    if (above < k) {
      const int v = key_index(key);
      ti[above] = v;
      tl[above] = (elem<T>::load(row + v) - m) - lz;
    }
  }
}

// The gradient, one workgroup per row, one pass: with t = l / log 2
//   d_v = -p_v (total + gH (l_v + H)) = -2^t (g0 + g1 t)
// and then the columns that take a gradient of their own (the given token, the
// alternatives), each written once with all that it takes.  Measured on 8192 x 50258
// bf16: 326 us, 5.1 TB/s read and written; 1001 x 50257 fp32: 83 us.
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void subs_scores_bwd_kernel(
    const T* logits, int64_t ld, const int64_t* __restrict__ xt, const int64_t* __restrict__ x0,
    const float* __restrict__ lse, const float* __restrict__ ent, const float* __restrict__ g_logp,
    const float* __restrict__ g_ent, const int64_t* __restrict__ top_ids, const float* __restrict__ g_top, int k,
    T* dl, int64_t ldo, int V, int mask) {
  constexpr int E = RowSpan<T>::E, U = BLOCK == 1024 ? 8 : 4;
  __shared__ float sg[SC_MAX_K + 1], sx[SC_MAX_K + 1];
  __shared__ int sid[SC_MAX_K + 1];
  __shared__ float red[2][BLOCK / 64];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const bool live = xt[r] == mask;
  const T* row = logits + r * ld;
  T* out = dl + r * ldo;
  if (live && tid <= k) {
    const int64_t id = tid == 0 ? x0[r] : top_ids[r * k + tid - 1];
    const bool col = id >= 0 && id < V;
    const float g = tid == 0 ? (g_logp ? g_logp[r] : 0.f) : g_top[r * k + tid - 1];
    sg[tid] = col ? g : 0.f;
    sid[tid] = col && id != mask ? (int)id : -1;
    sx[tid] = col ? elem<T>::load(row + id) : 0.f;     // before anything is written: dl may be the logits
  }
  __syncthreads();
  float total = 0.f;
  const float gh = live && g_ent ? g_ent[r] : 0.f;
  bool any = gh != 0.f;
  if (live)
    for (int j = 0; j <= k; ++j) { total += sg[j]; any |= sg[j] != 0.f; }
  const RowSpan<T> sp(out, V, mask);
  uint4* const oc = reinterpret_cast<uint4*>(out + sp.head);
  const int alone = tid < sp.head + sp.tail ? sp.single(tid) : -1;
  if (!any) {   // known, or nothing comes in: zero whatever the logits hold
    for (int i = tid; i < sp.n; i += BLOCK) oc[i] = make_uint4(0, 0, 0, 0);
    if (alone >= 0) elem<T>::store(out + alone, 0.f);
    return;
  }
  // l = (x - m) - lz.  The saved log-sum-exp serves as m (lz = 0) unless it is so
  // large (rows of lowest values, say) that it no longer holds log Z to 2^-17.
  float m = lse[r], lz = 0.f;
  const float H = ent[r];
  if (!(fabsf(m) <= 128.f)) {
    m = -INFINITY;
    for (int v = tid; v < V; v += BLOCK)
      if (v != mask) m = fmaxf(m, elem<T>::load(row + v));
    m = wave_max(m);
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    for (int j = 0; j < BLOCK / 64; ++j) m = fmaxf(m, red[0][j]);
    for (int v = tid; v < V; v += BLOCK)
      if (v != mask) lz += __builtin_amdgcn_exp2f((elem<T>::load(row + v) - m) * SC_L2E);
    lz = wave_sum(lz);
    if ((tid & 63) == 0) red[1][tid >> 6] = lz;
    __syncthreads();
    lz = 0.f;
    for (int j = 0; j < BLOCK / 64; ++j) lz += red[1][j];
    lz = log2f(lz) * SC_LN2;
  }
  const float g0 = total + gh * H, g1 = gh * SC_LN2, l2z = lz * SC_L2E;
  const bool bad = !(fabsf(m) < INFINITY) || !(fabsf(lz) < INFINITY);    // no distribution: NaN
  auto dense = [&](float x) {
    // 2^-200 is 0: a logit of -inf gives 0, not 0 * inf
    const float t = fmaxf(__builtin_fmaf(x - m, SC_L2E, -l2z), -200.f);
    const float p = __builtin_amdgcn_exp2f(t);
    return bad ? NAN : -p * __builtin_fmaf(g1, t, g0);
  };
  auto do_chunk = [&](const uint4& q, int i) {
    float f[E];
    unpack16<T>(q, f);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = dense(f[e]);
    if (i == sp.mask_chunk) {
#pragma unroll
      for (int e = 0; e < E; ++e) if (e == sp.mask_elem) f[e] = 0.f;
    }
    if constexpr (E == 8)
      oc[i] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    else
      oc[i] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  };
  const T* in = row + sp.head;
  auto pass = [&](auto load) {
    for (int i = tid; i < sp.n; i += U * BLOCK) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) if (i + u * BLOCK < sp.n) q[u] = load(i + u * BLOCK);
#pragma unroll
      for (int u = 0; u < U; ++u) if (i + u * BLOCK < sp.n) do_chunk(q[u], i + u * BLOCK);
    }
  };
  if (alone >= 0) elem<T>::store(out + alone, alone == mask ? 0.f : dense(elem<T>::load(row + alone)));
  if (((uintptr_t)in & 15) == 0) {
    pass([&](int i) { return reinterpret_cast<const uint4*>(in)[i]; });
  } else {        // rows of logits and gradient start at different places: loads that are not aligned
    pass([&](int i) { uint4 q; __builtin_memcpy(&q, in + (int64_t)i * E, 16); return q; });
  }
  __syncthreads();
  if (tid <= k && sid[tid] >= 0) {
    const int v = sid[tid];
    float g = 0.f;
    bool first = true;
    for (int j = 0; j <= k; ++j)
      if (sid[j] == v) { g += sg[j]; first &= j >= tid; }
    if (first) elem<T>::store(out + v, dense(sx[tid]) + g);
  }
}

}  // namespace mdlm

using namespace mdlm;

extern "C" int mdlm_subs_scores(const void* logits, int64_t ld, int dtype, const int64_t* xt, const int64_t* x0,
                                float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_ids,
                                int64_t rows, int V, int mask_index, int top_k, void* stream) {
  if (rows == 0) return 0;
  MDLM_CHECK_ARG(logits && xt && x0 && logp && entropy && lse, "subs_scores: null pointer");
  MDLM_CHECK_ARG(rows > 0 && rows < (1ll << 31) && V > 0 && ld >= V, "subs_scores: bad shape");
  MDLM_CHECK_ARG(mask_index >= 0 && mask_index < V, "subs_scores: bad mask index");
  MDLM_CHECK_ARG(top_k >= 0 && top_k <= SC_MAX_K && top_k < V,
                 "subs_scores: top_k=%d must be at most %d and less than V=%d", top_k, SC_MAX_K, V);
  MDLM_CHECK_ARG(top_k == 0 || (top_logp && top_ids), "subs_scores: null pointer (alternatives)");
#define SC_LAUNCH(T, B) \
  subs_scores_kernel<T, B><<<(unsigned)rows, B, 0, (hipStream_t)stream>>>((const T*)logits, ld, xt, x0, logp, entropy, lse, top_logp, top_ids, V, mask_index, top_k)
  const bool wide = rows <= SC_WIDE_ROWS && (int64_t)V * (dtype == MDLM_BF16 ? 2 : 4) >= SC_WIDE_BYTES;
  if (dtype == MDLM_BF16) { if (wide) SC_LAUNCH(bf16_t, 1024); else SC_LAUNCH(bf16_t, 256); }
  else if (dtype == MDLM_F32) { if (wide) SC_LAUNCH(float, 1024); else SC_LAUNCH(float, 256); }
#undef SC_LAUNCH
  else { set_error("subs_scores: bad dtype %d", dtype); return -1; }
  MDLM_LAUNCH_CHECK();
  return 0;
}

extern "C" int mdlm_subs_scores_bwd(const void* logits, int64_t ld, int dtype, const int64_t* xt, const int64_t* x0,
                                    const float* lse, const float* entropy, const float* g_logp,
                                    const float* g_entropy, const int64_t* top_ids, const float* g_top, int top_k,
                                    void* dlogits, int64_t ldo, int64_t rows, int V, int mask_index, void* stream) {
  if (rows == 0) return 0;
  MDLM_CHECK_ARG(logits && xt && x0 && lse && entropy && dlogits, "subs_scores_bwd: null pointer");
  MDLM_CHECK_ARG(rows > 0 && rows < (1ll << 31) && V > 0 && ld >= V && ldo >= V, "subs_scores_bwd: bad shape");
  MDLM_CHECK_ARG(dlogits != logits || ldo == ld || rows == 1, "subs_scores_bwd: in place, but with rows at other places");
  MDLM_CHECK_ARG(mask_index >= 0 && mask_index < V, "subs_scores_bwd: bad mask index");
  MDLM_CHECK_ARG(top_k >= 0 && top_k <= SC_MAX_K && top_k < V,
                 "subs_scores_bwd: top_k=%d must be at most %d and less than V=%d", top_k, SC_MAX_K, V);
  MDLM_CHECK_ARG(top_k == 0 || (top_ids && g_top), "subs_scores_bwd: null pointer (alternatives)");
#define SC_LAUNCH(T, B) \
  subs_scores_bwd_kernel<T, B><<<(unsigned)rows, B, 0, (hipStream_t)stream>>>((const T*)logits, ld, xt, x0, lse, entropy, g_logp, g_entropy, top_ids, g_top, top_k, (T*)dlogits, ldo, V, mask_index)
  const bool wide = rows <= SC_WIDE_ROWS && (int64_t)V * (dtype == MDLM_BF16 ? 2 : 4) >= SC_WIDE_BYTES;
  if (dtype == MDLM_BF16) { if (wide) SC_LAUNCH(bf16_t, 1024); else SC_LAUNCH(bf16_t, 256); }
  else if (dtype == MDLM_F32) { if (wide) SC_LAUNCH(float, 1024); else SC_LAUNCH(float, 256); }
#undef SC_LAUNCH
  else { set_error("subs_scores_bwd: bad dtype %d", dtype); return -1; }
  MDLM_LAUNCH_CHECK();
  return 0;
}
