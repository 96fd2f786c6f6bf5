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

// A position that is not masked: log-probability 0 for its own token, -1e6 for
// every other one; the alternatives are its token and the lowest other ids.
__device__ __forceinline__ void known_row(int64_t r, int64_t tok, const int64_t* x0, float* logp, float* ent, float* lse,
                                          float* top_logp, int64_t* top_ids, int V, int mask, int k, int tid) {
  if (tid == 0) {
    logp[r] = x0[r] == tok ? 0.f : SC_NEG;
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

template <typename T>
__global__ __launch_bounds__(256) void subs_scores_kernel(
    const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ xt, const int64_t* __restrict__ x0,
    float* __restrict__ logp, float* __restrict__ ent, float* __restrict__ lse, float* __restrict__ top_logp,
    int64_t* __restrict__ top_ids, int V, int mask, int k) {
  __shared__ float red[3][4];
  __shared__ unsigned long long best[2][4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, w = tid >> 6;
  const int64_t tok = xt[r];
  if (tok != mask) { known_row(r, tok, x0, logp, ent, lse, top_logp, top_ids, V, mask, k, tid); return; }
  const T* row = logits + r * ld;
  float m = -INFINITY;
  for (int v = tid; v < V; v += 256)
    if (v != mask) m = fmaxf(m, elem<T>::load(row + v));
  m = wave_max(m);
  if ((tid & 63) == 0) red[0][w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float s = 0.f, s1 = 0.f;
  if (m > -INFINITY) {
    for (int v = tid; v < V; v += 256)
      if (v != mask) {
        const float t = (elem<T>::load(row + v) - m) * SC_L2E;
        const float e = __builtin_amdgcn_exp2f(t);
        s += e;
        s1 += e == 0.f ? 0.f : e * t;
      }
  }
  s = wave_sum(s); s1 = wave_sum(s1);
  if ((tid & 63) == 0) { red[1][w] = s; red[2][w] = s1; }
  __syncthreads();
  s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  s1 = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  const float lz = log2f(s) * SC_LN2;
  if (tid == 0) {
    lse[r] = m + lz;
    ent[r] = lz - (s1 / s) * SC_LN2;
    const int64_t t = x0[r];
    float lp = 0.f;                                     // no token there
    if (t >= 0 && t < V) {
      const float x = elem<T>::load(row + t);
      lp = t == mask ? (x + SC_NEG) - (m + lz) : (x - m) - lz;
    }
    logp[r] = lp;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long b = 0;
    for (int v = tid; v < V; v += 256)
      if (v != mask) {
        const unsigned long long q = score_key(elem<T>::load(row + v), v);
        if (q < last && q > b) b = q;
      }
    b = wave_max_u64(b);
    if ((tid & 63) == 0) best[j & 1][w] = b;
    __syncthreads();
    b = best[j & 1][0];
    for (int i = 1; i < 4; ++i) b = best[j & 1][i] > b ? best[j & 1][i] : b;
    last = b;
    if (tid == 0) {
      const int v = key_index(b);
      top_ids[r * k + j] = v;
      top_logp[r * k + j] = (elem<T>::load(row + v) - m) - lz;
    }
  }
}

// One row's incoming gradients: the columns that get one of their own (the given
// token, the alternatives), each column once.
template <typename T>
__global__ __launch_bounds__(256) void subs_scores_bwd_kernel(
    const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ xt, const int64_t* __restrict__ x0,
    const float* __restrict__ lse, const float* __restrict__ ent, const float* __restrict__ g_logp,
    const float* __restrict__ g_ent, const int64_t* __restrict__ top_ids, const float* __restrict__ g_top, int k,
    T* __restrict__ dl, int64_t ldo, int V, int mask) {
  __shared__ float sg[SC_MAX_K + 1];
  __shared__ int sid[SC_MAX_K + 1];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const bool live = xt[r] == mask;
  if (live && tid <= k) {
    const int64_t id = tid == 0 ? x0[r] : top_ids[r * k + tid - 1];
    const bool col = id >= 0 && id < V;
    float g = tid == 0 ? (g_logp ? g_logp[r] : 0.f) : g_top[r * k + tid - 1];
    if (!col) g = 0.f;
    sg[tid] = g;
    sid[tid] = col && id != mask ? (int)id : -1;
  }
  __syncthreads();
  float total = 0.f;
  const float gh = live && g_ent ? g_ent[r] : 0.f;
  bool any = gh != 0.f;
  if (live)
    for (int j = 0; j <= k; ++j) { total += sg[j]; any |= sg[j] != 0.f; }
  T* out = dl + r * ldo;
  if (!any) {   // known, or nothing comes in: zero whatever the logits hold
    for (int v = tid; v < V; v += 256) elem<T>::store(out + v, 0.f);
    return;
  }
  const T* row = logits + r * ld;
  // l = (x - m) - lz.  The saved log-sum-exp serves as m (lz = 0) unless it is so
  // large (rows of lowest values, say) that it no longer holds log Z to 2^-17.
  float m = lse[r], lz = 0.f;
  const float H = ent[r];
  if (!(fabsf(m) <= 128.f)) {
    __shared__ float red[2][4];
    m = -INFINITY;
    for (int v = tid; v < V; v += 256)
      if (v != mask) m = fmaxf(m, elem<T>::load(row + v));
    m = wave_max(m);
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    for (int v = tid; v < V; v += 256)
      if (v != mask) lz += __builtin_amdgcn_exp2f((elem<T>::load(row + v) - m) * SC_L2E);
    lz = wave_sum(lz);
    if ((tid & 63) == 0) red[1][tid >> 6] = lz;
    __syncthreads();
    lz = log2f((red[1][0] + red[1][1]) + (red[1][2] + red[1][3])) * SC_LN2;
  }
  auto dense = [&](int v) {
    const float l = (elem<T>::load(row + v) - m) - lz;
    const float p = __builtin_amdgcn_exp2f(l * SC_L2E);
    return p == 0.f ? 0.f : -p * __builtin_fmaf(gh, l + H, total);
  };
  for (int v = tid; v < V; v += 256) {
    float d = v == mask ? 0.f : dense(v);
    if (v != mask)
      for (int j = 0; j <= k; ++j)
        if (sid[j] == v) d += sg[j];
    elem<T>::store(out + v, d);
  }
}

}  // namespace mdlm

using namespace mdlm;

extern "C" int64_t mdlm_subs_scores_workspace_bytes(int64_t rows, int V, int top_k) {
  if (rows < 0 || V <= 0 || top_k < 0 || top_k > SC_MAX_K) return -1;
  return 0;
}

extern "C" int mdlm_subs_scores(const void* logits, int64_t ld, int dtype, const int64_t* xt, const int64_t* x0,
                                float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_ids,
                                int64_t rows, int V, int mask_index, int top_k, void* ws, void* stream) {
  if (rows == 0) return 0;
  MDLM_CHECK_ARG(logits && xt && x0 && logp && entropy && lse, "subs_scores: null pointer");
  MDLM_CHECK_ARG(rows > 0 && rows < (1ll << 31) && V > 0 && ld >= V, "subs_scores: bad shape");
  MDLM_CHECK_ARG(mask_index >= 0 && mask_index < V, "subs_scores: bad mask index");
  MDLM_CHECK_ARG(top_k >= 0 && top_k <= SC_MAX_K && top_k < V,
                 "subs_scores: top_k=%d must be at most %d and less than V=%d", top_k, SC_MAX_K, V);
  MDLM_CHECK_ARG(top_k == 0 || (top_logp && top_ids), "subs_scores: null pointer (alternatives)");
  (void)ws;
  if (dtype == MDLM_BF16)
    subs_scores_kernel<bf16_t><<<(unsigned)rows, 256, 0, (hipStream_t)stream>>>((const bf16_t*)logits, ld, xt, x0, logp, entropy, lse, top_logp, top_ids, V, mask_index, top_k);
  else if (dtype == MDLM_F32)
    subs_scores_kernel<float><<<(unsigned)rows, 256, 0, (hipStream_t)stream>>>((const float*)logits, ld, xt, x0, logp, entropy, lse, top_logp, top_ids, V, mask_index, top_k);
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
  MDLM_CHECK_ARG(mask_index >= 0 && mask_index < V, "subs_scores_bwd: bad mask index");
  MDLM_CHECK_ARG(top_k >= 0 && top_k <= SC_MAX_K && top_k < V,
                 "subs_scores_bwd: top_k=%d must be at most %d and less than V=%d", top_k, SC_MAX_K, V);
  MDLM_CHECK_ARG(top_k == 0 || (top_ids && g_top), "subs_scores_bwd: null pointer (alternatives)");
  if (dtype == MDLM_BF16)
    subs_scores_bwd_kernel<bf16_t><<<(unsigned)rows, 256, 0, (hipStream_t)stream>>>((const bf16_t*)logits, ld, xt, x0, lse, entropy, g_logp, g_entropy, top_ids, g_top, top_k, (bf16_t*)dlogits, ldo, V, mask_index);
  else if (dtype == MDLM_F32)
    subs_scores_bwd_kernel<float><<<(unsigned)rows, 256, 0, (hipStream_t)stream>>>((const float*)logits, ld, xt, x0, lse, entropy, g_logp, g_entropy, top_ids, g_top, top_k, (float*)dlogits, ldo, V, mask_index);
  else { set_error("subs_scores_bwd: bad dtype %d", dtype); return -1; }
  MDLM_LAUNCH_CHECK();
  return 0;
}
