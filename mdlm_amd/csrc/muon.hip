// Orthogonalised weight update (the optimizer step of the reference is AdamW,
// diffusion.py:449-459, 254-259): Newton-Schulz products on the matrix cores.
//   X_0 = G / (|G|_F + eps),   X <- a X + (b A + c A^2) X,   A = X X^T
// with X held s x l, s = min(rows, cols) (a tall G is worked on transposed).
//
// Arithmetic.  Operands are fp16, sums fp32.  Left as written the polynomial
// cancels (a = 3.44, b = -4.78, c = 2.03 leave 0.7..1.2 near sigma = 1) and one
// rounding of A or B costs ten times its size.  With the square completed,
//   a + b t + c t^2 = c (t + b/2c)^2 + (a - b^2/4c),
// D = A + (b/2c) I is small near convergence and nothing cancels:
//   P = c D D^T + (a - b^2/4c) I,   X <- mu X + (P - mu I) X.
// mu = a in the early steps (small singular values: P is close to a I) and 1 in
// the last two (P is close to I), and the mu X term takes X from TWO fp16 words
// (hi + lo, 22 bits), so that only the small P - mu I sees X rounded to fp16.
// The diagonal of D, its largest part, is also corrected for its rounding:
// d = D_ii - fp16(D_ii) enters D D^T to first order.  Against 64 bits the result is
// 4e-4 .. 1e-3 off (2-norm, relative), less than rounding it to bf16 costs
// (1.7e-3); plain bf16 operands are 1e-2 .. 3e-2 off.
//
// Every matrix is padded with zeros to whole tiles in the workspace, so the
// products have no edges; padding stays zero through every step.
#include "common.h"
#include <math.h>

namespace mdlm {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int NS_TILE = 128;
constexpr int NS_BK = 64;
constexpr int NS_NORM_BLOCKS = 256;   // partial sums of |G|^2 per matrix
// Powers of two that keep the fp16 words away from the subnormal range: entries
// of X are at most about 1.2 and about 1/sqrt(s l) on average, D and P are at
// most a few units.
constexpr float NS_SX = 2048.f;
constexpr float NS_SD = 256.f;

struct NsShape { int s, l, sp, lp; bool tall; };
static inline NsShape ns_shape(int rows, int cols) {
  NsShape q;
  q.tall = rows > cols;
  q.s = q.tall ? cols : rows;
  q.l = q.tall ? rows : cols;
  q.sp = (q.s + NS_TILE - 1) / NS_TILE * NS_TILE;
  q.lp = (q.l + NS_TILE - 1) / NS_TILE * NS_TILE;
  return q;
}

// workspace of n matrices
struct NsWs {
  double* norm;      // n x NS_NORM_BLOCKS partial sums of squares
  float* diag;       // n x sp
  float* o;          // n x sp x lp, the result of the last step
  f16 *h[2], *lo;    // n x sp x lp
  f16 *d, *p;        // n x sp x sp
};
static inline int64_t ns_layout(const NsShape& q, int n, char* base, NsWs* w) {
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t at = off; off += (bytes + 255) / 256 * 256; return base + at; };
  const int64_t x = (int64_t)n * q.sp * q.lp, d = (int64_t)n * q.sp * q.sp;
  NsWs t;
  t.norm = (double*)take((int64_t)n * NS_NORM_BLOCKS * 8);
  t.diag = (float*)take((int64_t)n * q.sp * 4);
  t.o = (float*)take(x * 4);
  t.h[0] = (f16*)take(x * 2);
  t.h[1] = (f16*)take(x * 2);
  t.lo = (f16*)take(x * 2);
  t.d = (f16*)take(d * 2);
  t.p = (f16*)take(d * 2);
  if (w) *w = t;
  return off;
}

// What is orthogonalised: G itself (MOM = false), or the look-ahead of the momentum
// of the clipped gradient.
struct NsSrc {
  const void* g; int64_t ld, bs; int bf16;
  float* m;                 // momentum, the layout of g (null: g alone)
  float momentum;
  const float* sumsq; float max_norm, grad_scale;
};
__device__ __forceinline__ float clip_coef(const NsSrc& a) {
  float coef = a.grad_scale;
  if (a.sumsq && a.max_norm > 0.f) {
    const float total = sqrtf(a.sumsq[0]) * a.grad_scale;
    coef *= fminf(1.f, a.max_norm / (total + 1e-6f));
  }
  return coef;
}
__device__ __forceinline__ float src_load(const NsSrc& a, int64_t i, float coef) {
  float g = a.bf16 ? bf16_to_f32(((const bf16_t*)a.g)[i]) : ((const float*)a.g)[i];
  if (a.m) {
    g *= coef;
    g += a.momentum * (a.m[i] - g);
  }
  return g;
}

// momentum (in place) and the partial sums of squares of what will be orthogonalised,
// in 64 bits: squares of small gradients leave the fp32 range
__global__ __launch_bounds__(256) void ns_norm_kernel(NsSrc a, double* __restrict__ part, int rows, int cols) {
  __shared__ double red[4];
  const int b = blockIdx.y;
  const float coef = a.m ? clip_coef(a) : 1.f;
  double acc = 0.0;
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t at = b * a.bs + r * a.ld;
    for (int c = threadIdx.x; c < cols; c += 256) {
      if (a.m) {
        const float g = ((const float*)a.g)[at + c] * coef, m = a.m[at + c];
        a.m[at + c] = m + (g - m) * (1.f - a.momentum);
      }
      const double u = src_load(a, at + c, coef);
      acc += u * u;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) part[b * NS_NORM_BLOCKS + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void split_f16(float x, f16& h, f16& l) {
  h = (f16)x;
  l = (f16)(x - (float)h);
}

// X_0 = G / (|G| + eps), scaled, as hi + lo; 32 x 32 tiles through LDS so that a tall
// G is read by rows and written by rows
__global__ __launch_bounds__(256) void ns_ingest_kernel(NsSrc a, const double* __restrict__ part, double eps,
                                                        f16* __restrict__ h, f16* __restrict__ lo, int rows, int cols,
                                                        int sp, int lp, int tall) {
  __shared__ float tile[32][33];
  __shared__ float inv_s;
  const int b = blockIdx.z, tid = threadIdx.x;
  if (tid < 64) {
    double t = 0.0;
    for (int i = tid; i < NS_NORM_BLOCKS; i += 64) t += part[b * NS_NORM_BLOCKS + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
    if (tid == 0) inv_s = (float)((double)NS_SX / (sqrt(t) + eps));
  }
  __syncthreads();
  const float inv = inv_s, coef = a.m ? clip_coef(a) : 1.f;
  const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;   // of X
  const int tx = tid & 31, ty = tid >> 5;
  for (int k = ty; k < 32; k += 8) {
    const int r = tall ? j0 + k : i0 + k, c = tall ? i0 + tx : j0 + tx;
    const float v = r < rows && c < cols ? src_load(a, b * a.bs + r * a.ld + c, coef) * inv : 0.f;
    if (tall) tile[tx][k] = v; else tile[k][tx] = v;
  }
  __syncthreads();
  for (int k = ty; k < 32; k += 8) {
    const int64_t at = ((int64_t)b * sp + i0 + k) * lp + j0 + tx;
    split_f16(tile[k][tx], h[at], lo[at]);
  }
}

enum { NS_GRAM = 0, NS_SQUARE = 1, NS_APPLY = 2 };

struct NsGemm {
  const f16* A; int64_t lda, bsa;    // M x K, K contiguous
  const f16* B; int64_t ldb, bsb;    // N x K, K contiguous (APPLY: K x N, N contiguous)
  int K, tiles_m, tiles_n, n;
  f16* out; int64_t ldo, bso;        // D, P or the next X's high words
  f16* lo;                           // APPLY: low words of X, in place
  float* o;                          // APPLY, last step: fp32 result (null: not the last)
  float* diag; int sp;               // rounding of D's diagonal
  float shift, c, mu;                // b/2c; c; see the head of this file
};

#define NS_GLDS16(gptr, lptr) \
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(gptr), \
                                   (__attribute__((address_space(3))) void*)(lptr), 16, 0, 0)

// 128 x 128 tile, 4 waves of 64 x 64, 64-deep slabs double-buffered in LDS by LDS-DMA.
// LDS rows of a K-contiguous operand hold 64 values (128 bytes); the 16-byte chunk
// index is XORed with row & 7 on the source address and on the fragment reads.  The
// N-contiguous operand of APPLY keeps its rows (128 columns, 256 bytes) and is
// read through the transposing LDS read (four rows x 16 columns per 16 lanes);
// its 32-byte blocks are XORed with (row & 3) | (row >> 3 & 1) << 2.
template <int MODE>
__global__ __launch_bounds__(256, 2) void ns_gemm_kernel(NsGemm g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int OP = NS_TILE * NS_BK * 2, STAGE = 2 * OP;   // 16 KiB per operand
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid >> 1, wc = wid & 1;
  const int per_mat = g.tiles_m * g.tiles_n, total = per_mat * g.n;
  // each XCD (workgroup id & 7) gets a contiguous range of tiles
  const int per_xcd = (total + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || idx >= total) return;
  const int b = idx / per_mat, rest = idx - b * per_mat;
  const int tm = rest / g.tiles_n, tn = rest - tm * g.tiles_n;
  const f16* A = g.A + b * g.bsa + (int64_t)tm * NS_TILE * g.lda;
  const f16* B = g.B + b * g.bsb + (MODE == NS_APPLY ? (int64_t)tn * NS_TILE : (int64_t)tn * NS_TILE * g.ldb);

  const int arow = lane >> 3, achunk = ((lane & 7) ^ arow) * 8;
  const f16* a_src = A + (int64_t)(wid * 8 + arow) * g.lda + achunk;
  const f16* b_src;
  if constexpr (MODE == NS_APPLY) {
    const int row = wid * 4 + (lane >> 4), pch = lane & 15;
    const int fx = (row & 3) | (((row >> 3) & 1) << 2);      // + 16 rows: unchanged
    b_src = B + (int64_t)row * g.ldb + (((pch >> 1) ^ fx) * 2 + (pch & 1)) * 8;
  } else {
    b_src = B + (int64_t)(wid * 8 + arow) * g.ldb + achunk;
  }
  auto stage = [&](int buf, int k0) {
    char* const sb = smem + buf * STAGE;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      NS_GLDS16(a_src + (int64_t)(i * 32) * g.lda + k0, sb + (i * 4 + wid) * 1024);
      if constexpr (MODE == NS_APPLY)
        NS_GLDS16(b_src + (int64_t)(k0 + i * 16) * g.ldb, sb + OP + (i * 4 + wid) * 1024);
      else
        NS_GLDS16(b_src + (int64_t)(i * 32) * g.ldb + k0, sb + OP + (i * 4 + wid) * 1024);
    }
  };
  const int fr = lane & 15, fq = lane >> 4;
  int foff[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) foff[ks] = fr * 128 + (((ks * 4 + fq) ^ (lane & 7)) * 16);
  const int a_base = wr * 64 * 128, b_base = OP + wc * 64 * 128;
  unsigned tr_off[4];
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  if constexpr (MODE == NS_APPLY) {
    const int q = fr >> 2, p = lane & 3, fx = q | ((fq & 1) << 2);
#pragma unroll
    for (int n = 0; n < 4; ++n) tr_off[n] = lds0 + OP + (8 * fq + q) * 256 + (((wc * 4 + n) ^ fx) * 32) + p * 8;
  }
  f32x4 acc[4][4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};

  stage(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int KT = g.K / NS_BK;
  for (int kt = 0; kt < KT; ++kt) {
    const int buf = kt & 1;
    if (kt + 1 < KT) stage(buf ^ 1, (kt + 1) * NS_BK);
    const char* sb = smem + buf * STAGE;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f16x8 af[4], bf[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) af[m] = *reinterpret_cast<const f16x8*>(sb + a_base + m * 2048 + foff[ks]);
      if constexpr (MODE == NS_APPLY) {
        // the reads and their wait in one block: the compiler does not count them
        uint2 t[8];
        const unsigned o = buf * STAGE + ks * 32 * 256;
        const unsigned a0 = tr_off[0] + o, a1 = tr_off[1] + o, a2 = tr_off[2] + o, a3 = tr_off[3] + o;
        asm volatile(
          "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:1024\n\t"
          "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:1024\n\t"
          "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:1024\n\t"
          "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:1024\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3]), "=&v"(t[4]), "=&v"(t[5]), "=&v"(t[6]), "=&v"(t[7])
          : "v"(a0), "v"(a1), "v"(a2), "v"(a3) : "memory");
#pragma unroll
        for (int n = 0; n < 4; ++n)
          bf[n] = __builtin_bit_cast(f16x8, make_uint4(t[2 * n].x, t[2 * n].y, t[2 * n + 1].x, t[2 * n + 1].y));
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) bf[n] = *reinterpret_cast<const f16x8*>(sb + b_base + n * 2048 + foff[ks]);
      }
      // swapped operands: a lane holds four consecutive columns of one output row
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[n], af[m], acc[m][n], 0, 0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the next slab has landed
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int i = tm * NS_TILE + wr * 64 + m * 16 + fr;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = tn * NS_TILE + wc * 64 + n * 16 + fq * 4;
      const int64_t at = b * g.bso + (int64_t)i * g.ldo + j;
      f16x4 hv;
      if constexpr (MODE == NS_GRAM) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = acc[m][n][e] * (NS_SD / (NS_SX * NS_SX));
          if (i == j + e) v += g.shift * NS_SD;
          hv[e] = (f16)v;
          if (i == j + e) g.diag[b * g.sp + i] = v - (float)hv[e];
        }
        *reinterpret_cast<f16x4*>(g.out + at) = hv;
      } else if constexpr (MODE == NS_SQUARE) {
        const f16x4 dv = *reinterpret_cast<const f16x4*>(g.A + at);      // D at the output's place
        const float di = g.diag[b * g.sp + i];
        const f32x4 dj = *reinterpret_cast<const f32x4*>(g.diag + b * g.sp + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = (acc[m][n][e] + (di + dj[e]) * (float)dv[e]) * (g.c / NS_SD);
          if (i == j + e) v += g.mu * NS_SD;      // (a - b^2/4c) - mu
          hv[e] = (f16)v;
        }
        *reinterpret_cast<f16x4*>(g.out + at) = hv;
      } else {
        const f16x4 xh = *reinterpret_cast<const f16x4*>(g.B + at), xl = *reinterpret_cast<const f16x4*>(g.lo + at);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = g.mu * ((float)xh[e] + (float)xl[e]) + acc[m][n][e] * (1.f / NS_SD);
        if (g.o) {
          *reinterpret_cast<f32x4*>(g.o + at) = v * (1.f / NS_SX);
        } else {
          f16x4 lv;
#pragma unroll
          for (int e = 0; e < 4; ++e) { f16 hh, ll; split_f16(v[e], hh, ll); hv[e] = hh; lv[e] = ll; }
          *reinterpret_cast<f16x4*>(g.out + at) = hv;
          *reinterpret_cast<f16x4*>(g.lo + at) = lv;
        }
      }
    }
  }
}

// The result in the caller's layout, and what is done with it there.
struct NsOut {
  bf16_t* out;                           // the orthogonalised matrix, or
  float* p; float* ema; bf16_t* w16;     // weights, moving average, bf16 copy
  int64_t ld, bs;
  float step, decay, ema_omd;            // lr * scale; 1 - lr * weight_decay
};
__device__ __forceinline__ void ns_store(const NsOut& w, int64_t at, float o) {
  if (w.out) { w.out[at] = f32_to_bf16(o); return; }
  const float p = w.p[at] * w.decay - w.step * o;
  w.p[at] = p;
  if (w.ema) { const float e = w.ema[at]; w.ema[at] = e - w.ema_omd * (e - p); }
  if (w.w16) w.w16[at] = f32_to_bf16(p);
}
__global__ __launch_bounds__(256) void ns_out_kernel(NsOut w, const float* __restrict__ o, int rows, int cols, int sp,
                                                     int lp, int tall) {
  __shared__ float tile[32][33];
  const int b = blockIdx.z, tid = threadIdx.x, tx = tid & 31, ty = tid >> 5;
  const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;   // of X
  for (int k = ty; k < 32; k += 8) tile[k][tx] = o[((int64_t)b * sp + i0 + k) * lp + j0 + tx];
  __syncthreads();
  for (int k = ty; k < 32; k += 8) {
    const int r = tall ? j0 + k : i0 + k, c = tall ? i0 + tx : j0 + tx;
    if (r < rows && c < cols) ns_store(w, b * w.bs + r * w.ld + c, tall ? tile[tx][k] : tile[k][tx]);
  }
}

static int ns_gemm(int mode, NsGemm g, hipStream_t st) {
  constexpr int LDS = 4 * NS_TILE * NS_BK * 2;
  static bool done[3][MAX_DEVICES] = {};
  const int64_t total = (int64_t)g.tiles_m * g.tiles_n * g.n;
  if (total >= (1ll << 28)) { set_error("orthogonalize: too many tiles"); return -1; }
  const unsigned grid = (unsigned)((total + 7) / 8 * 8);
  int rc;
  if (mode == NS_GRAM) {
    if ((rc = ensure_dynamic_lds(&ns_gemm_kernel<NS_GRAM>, LDS, done[0], "orthogonalize"))) return rc;
    ns_gemm_kernel<NS_GRAM><<<grid, 256, LDS, st>>>(g);
  } else if (mode == NS_SQUARE) {
    if ((rc = ensure_dynamic_lds(&ns_gemm_kernel<NS_SQUARE>, LDS, done[1], "orthogonalize"))) return rc;
    ns_gemm_kernel<NS_SQUARE><<<grid, 256, LDS, st>>>(g);
  } else {
    if ((rc = ensure_dynamic_lds(&ns_gemm_kernel<NS_APPLY>, LDS, done[2], "orthogonalize"))) return rc;
    ns_gemm_kernel<NS_APPLY><<<grid, 256, LDS, st>>>(g);
  }
  MDLM_LAUNCH_CHECK();
  return 0;
}

static int ns_run(const NsSrc& src, const NsOut& dst, int n, int rows, int cols, int steps, double a, double b,
                  double c, double eps, void* ws, hipStream_t st) {
  const NsShape q = ns_shape(rows, cols);
  NsWs w;
  ns_layout(q, n, (char*)ws, &w);
  ns_norm_kernel<<<dim3(NS_NORM_BLOCKS, n), 256, 0, st>>>(src, w.norm, rows, cols);
  MDLM_LAUNCH_CHECK();
  const dim3 grid32(q.lp / 32, q.sp / 32, n);
  ns_ingest_kernel<<<grid32, 256, 0, st>>>(src, w.norm, eps, w.h[0], w.lo, rows, cols, q.sp, q.lp, q.tall);
  MDLM_LAUNCH_CHECK();
  const int64_t bx = (int64_t)q.sp * q.lp, bd = (int64_t)q.sp * q.sp;
  for (int it = 0; it < steps; ++it) {
    const double mu = it + 2 < steps ? a : 1.0;
    f16 *x = w.h[it & 1], *xn = w.h[(it & 1) ^ 1];
    NsGemm g = {};
    g.n = n; g.sp = q.sp; g.diag = w.diag;
    g.A = x; g.lda = q.lp; g.bsa = bx; g.B = x; g.ldb = q.lp; g.bsb = bx; g.K = q.lp;
    g.tiles_m = g.tiles_n = q.sp / NS_TILE;
    g.out = w.d; g.ldo = q.sp; g.bso = bd; g.shift = (float)(b / (2 * c));
    if (int rc = ns_gemm(NS_GRAM, g, st)) return rc;
    g.A = w.d; g.lda = q.sp; g.bsa = bd; g.B = w.d; g.ldb = q.sp; g.bsb = bd; g.K = q.sp;
    g.out = w.p; g.c = (float)c; g.mu = (float)(a - b * b / (4 * c) - mu);
    if (int rc = ns_gemm(NS_SQUARE, g, st)) return rc;
    g.A = w.p; g.B = x; g.ldb = q.lp; g.bsb = bx; g.tiles_n = q.lp / NS_TILE;
    g.out = xn; g.ldo = q.lp; g.bso = bx; g.lo = w.lo; g.mu = (float)mu;
    g.o = it + 1 == steps ? w.o : nullptr;
    if (int rc = ns_gemm(NS_APPLY, g, st)) return rc;
  }
  ns_out_kernel<<<grid32, 256, 0, st>>>(dst, w.o, rows, cols, q.sp, q.lp, q.tall);
  MDLM_LAUNCH_CHECK();
  return 0;
}

// shapes and coefficients that every entry point here shares
static int ns_check(const char* who, int n, int rows, int cols, int64_t ld, int64_t bs, int steps, double a, double b,
                    double c, double eps) {
  MDLM_CHECK_ARG(n > 0 && n < 65536 && rows > 0 && cols > 0 && rows <= (1 << 17) && cols <= (1 << 17),
                 "%s: bad shape", who);
  MDLM_CHECK_ARG((rows < cols ? rows : cols) <= (1 << 15), "%s: the smaller side must be at most 32768", who);
  MDLM_CHECK_ARG(ld >= cols && (n == 1 || bs >= (int64_t)(rows - 1) * ld + cols), "%s: overlapping rows or matrices", who);
  MDLM_CHECK_ARG(steps >= 1 && steps <= 32, "%s: steps=%d is outside 1..32", who, steps);
  MDLM_CHECK_ARG(isfinite(a) && isfinite(b) && isfinite(c) && fabs(a) <= 16 && c != 0.0 && fabs(b / (2 * c)) <= 8 &&
                   fabs(c) <= 16,
                 "%s: coefficients (%g, %g, %g) are outside what the fp16 products hold", who, a, b, c);
  MDLM_CHECK_ARG(eps > 0.0 && isfinite(eps), "%s: eps must be positive", who);
  return 0;
}

}  // namespace mdlm

using namespace mdlm;

extern "C" int64_t mdlm_orthogonalize_workspace_bytes(int n, int rows, int cols) {
  if (n <= 0 || rows <= 0 || cols <= 0 || n >= 65536 || rows > (1 << 17) || cols > (1 << 17)) return -1;
  return ns_layout(ns_shape(rows, cols), n, nullptr, nullptr);
}

extern "C" int mdlm_orthogonalize(const void* g, int64_t ldg, int64_t g_stride, int dtype, void* out_bf16, int64_t ldo,
                                  int64_t out_stride, int n, int rows, int cols, int steps, double a, double b,
                                  double c, double eps, void* ws, void* stream) {
  if (n == 0 || rows == 0 || cols == 0) return 0;
  MDLM_CHECK_ARG(g && out_bf16 && ws, "orthogonalize: null pointer");
  MDLM_CHECK_ARG(dtype == MDLM_F32 || dtype == MDLM_BF16, "orthogonalize: bad dtype %d", dtype);
  if (int rc = ns_check("orthogonalize", n, rows, cols, ldg, g_stride, steps, a, b, c, eps)) return rc;
  if (int rc = ns_check("orthogonalize (out)", n, rows, cols, ldo, out_stride, steps, a, b, c, eps)) return rc;
  MDLM_CHECK_ARG(((uintptr_t)ws & 255) == 0, "orthogonalize: the workspace must be 256-byte aligned");
  NsSrc src = {};
  src.g = g; src.ld = ldg; src.bs = g_stride; src.bf16 = dtype == MDLM_BF16;
  NsOut dst = {};
  dst.out = (bf16_t*)out_bf16; dst.ld = ldo; dst.bs = out_stride;
  return ns_run(src, dst, n, rows, cols, steps, a, b, c, eps, ws, (hipStream_t)stream);
}

extern "C" int mdlm_muon_update(float* p, const float* g, float* m, float* ema, void* w_bf16, int64_t ld,
                                int64_t stride, int n, int rows, int cols, float lr, float momentum,
                                float weight_decay, float update_scale, int steps, double a, double b, double c,
                                double eps, float ema_one_minus_decay, const float* sumsq, float max_norm,
                                float grad_scale, void* ws, void* stream) {
  if (n == 0 || rows == 0 || cols == 0) return 0;
  MDLM_CHECK_ARG(p && g && m && ws, "muon_update: null pointer");
  if (int rc = ns_check("muon_update", n, rows, cols, ld, stride, steps, a, b, c, eps)) return rc;
  MDLM_CHECK_ARG(momentum >= 0.f && momentum < 1.f, "muon_update: momentum %g is outside [0, 1)", momentum);
  MDLM_CHECK_ARG(((uintptr_t)ws & 255) == 0, "muon_update: the workspace must be 256-byte aligned");
  NsSrc src = {};
  src.g = g; src.ld = ld; src.bs = stride; src.m = m; src.momentum = momentum;
  src.sumsq = sumsq; src.max_norm = max_norm; src.grad_scale = grad_scale;
  NsOut dst = {};
  dst.p = p; dst.ema = ema; dst.w16 = (bf16_t*)w_bf16; dst.ld = ld; dst.bs = stride;
  dst.step = lr * update_scale; dst.decay = 1.f - lr * weight_decay; dst.ema_omd = ema_one_minus_decay;
  return ns_run(src, dst, n, rows, cols, steps, a, b, c, eps, ws, (hipStream_t)stream);
}
