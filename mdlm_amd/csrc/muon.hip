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
// The mu X term takes X from two words, fp16 and e4m3 (15 bits together; 8 more bits of the
// second word would take a spectrum of i^-1.5 from 4.2e-4 to 0.9e-4 at 4096 x 8192, less than the result's own
// rounding shows, and it is a third of what the products move), so that only P - mu I sees X
// rounded to fp16.  Without the second word matrices of fast decaying spectra lose: 1.2e-2.
// Early, mu = a: P is a I but for the large singular values, the small ones are still multiplied by
// a, and what P - a I makes of the rounding of X stays with the large ones.  In the last three
// steps mu is each row's own P_ii (fp32), and P's off-diagonal part alone meets fp16.  (mu = 1 there:
// twice the error, three times for low rank and noise.  P_ii in all steps: three times the error
// for few rows of a decaying spectrum, 12 x 192, whose small values take on the roundings of the large.)
// The diagonals of D and P, their largest parts, lose nothing to fp16: d = D_ii - fp16(D_ii)
// enters D D^T to first order, and what fp16 leaves of P_ii - a goes to mu.
//
// Against 64 bits the result of five steps is 1e-4 .. 1.0e-3 off (2-norm, relative; fewer than 64
// rows up to 2e-3, fewer than 8, hardly anything to average over, up to 8e-3 (and bf16's own 2^-8 of
// an element with that: 1.3e-2); 16384 x 32768 with a
// spectrum of i^-1.5 1.3e-3); rounding it to bf16 costs 1.7e-3; plain bf16 operands are 1e-2 .. 3e-2
// off.  The usual coefficients do not converge: a step more makes differences larger, these as
// well as the input's (6 steps up to 1.5e-3, 7 2.0e-3, 10 1.5e-2).
//
// Every matrix is padded with zeros to whole slabs of 64 in the workspace; padding
// stays zero through every step.
#include "common.h"
#include <math.h>

namespace mdlm {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int NS_BK = 64;
constexpr int NS_MAX_SIDE = 32768;    // the smaller one
constexpr int NS_MAX_PARTS = 1024;    // partial sums of |G|^2 per matrix, at most
// Powers of two that keep the fp16 words away from the subnormal range: entries
// of X are at most about 1.2 and about 1/sqrt(s l) on average, D and P are at
// most a few units.
constexpr float NS_SX = 2048.f;
constexpr float NS_SD = 256.f;
// Of the second word, what X loses in the first: at most 1 while the first is below 2^12, |X| < 2.
// e4m3 goes from 2^-9 to 448, so 256 keeps the most of it that large matrices need, whose entries
// are small (average of X_0 at 4096 x 8192: 0.35 with NS_SX).  Off by, with 16 / 256 (spectra of
// i^-1.5): 1024 x 4096 1.8e-3 / 3.3e-4, 4096 x 8192 4.5e-3 / 4.2e-4, 8192 x 16384 7.4e-3 / 7.1e-4.
constexpr float NS_SL = 256.f;
constexpr float NS_LO_MAX = 448.f;    // larger X lose bits of the second word, no more

// Short sides up to this many rows (padded): A in parts of K, then one launch for A^2 and P X.
constexpr int NS_SMALL = 128;
struct NsShape { int s, l, sp, lp, splits; bool tall; };
static inline NsShape ns_shape(int rows, int cols) {
  NsShape q;
  q.tall = rows > cols;
  q.s = q.tall ? cols : rows;
  q.l = q.tall ? rows : cols;
  q.sp = (q.s + NS_BK - 1) / NS_BK * NS_BK;
  q.lp = (q.l + NS_BK - 1) / NS_BK * NS_BK;
  // A part more shortens the chain of slabs (0.2 us each) and is one more to be summed
  // (us per call, with 4, 5, 8 parts: 128 x 4096: 81, 80, 83; with 11, 16, 16: 128 x 32768:
  // 174, 179, 179; with 4, 6, 9: 16 x 6000: 72, 67, 67).  By shape alone: a matrix's result
  // does not depend on how many others it comes with.
  q.splits = 1;
  if (q.sp <= NS_SMALL)
    while (q.splits < 16 && (q.splits + 1) * (q.splits + 1) * (q.sp / 32) <= q.lp / NS_BK) ++q.splits;
  return q;
}

// workspace of n matrices
struct NsWs {
  double* norm;      // n x NS_MAX_PARTS partial sums of squares
  float *diag, *mu;  // n x sp
  f16* h[2];         // n x sp x lp, X's first words
  uint8_t* lo;       // n x sp x lp, its second words
  f16 *d, *p;        // n x sp x sp, or
  float* part;       // n x splits x sp x sp
};
static inline int64_t ns_layout(const NsShape& q, int n, char* base, NsWs* w) {
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t at = off; off += (bytes + 255) / 256 * 256; return base + at; };
  const int64_t x = (int64_t)n * q.sp * q.lp, d = (int64_t)n * q.sp * q.sp;
  NsWs t;
  t.norm = (double*)take((int64_t)n * NS_MAX_PARTS * 8);
  t.diag = (float*)take((int64_t)n * q.sp * 4);
  t.h[0] = (f16*)take(x * 2);
  t.h[1] = (f16*)take(x * 2);
  t.lo = (uint8_t*)take(x);
  t.d = t.p = nullptr;
  t.mu = nullptr;
  t.part = nullptr;
  if (q.sp <= NS_SMALL) {
    t.part = (float*)take(d * q.splits * 4);
  } else {
    t.d = (f16*)take(d * 2);
    t.p = (f16*)take(d * 2);
    t.mu = (float*)take((int64_t)n * q.sp * 4);
  }
  if (w) *w = t;
  return off;
}

// What is orthogonalised: G itself, or the look-ahead of the momentum of the clipped
// gradient.
struct NsSrc {
  const void* g; int64_t ld, bs; int bf16;
  int rows, cols, vec;      // vec: rows start 16-byte aligned
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
// eight columns of row r of matrix b, from column c (a multiple of 8) on; 0 past the last
struct NsRaw { float g[8], m[8]; };
__device__ __forceinline__ void src_fetch8(const NsSrc& a, int b, int r, int c, NsRaw& w) {
  const int64_t at = b * a.bs + r * a.ld + c;
  if (a.vec && c + 8 <= a.cols) {
    if (a.bf16) {
      const uint4 q = *reinterpret_cast<const uint4*>((const bf16_t*)a.g + at);
      const unsigned u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) w.g[e] = __uint_as_float(e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16);
    } else {
      const f32x4 x = *reinterpret_cast<const f32x4*>((const float*)a.g + at);
      const f32x4 y = *reinterpret_cast<const f32x4*>((const float*)a.g + at + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) w.g[e] = e < 4 ? x[e & 3] : y[e & 3];
    }
    if (a.m) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.m + at), y = *reinterpret_cast<const f32x4*>(a.m + at + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) w.m[e] = e < 4 ? x[e & 3] : y[e & 3];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = c + e < a.cols;
      w.g[e] = !in ? 0.f : a.bf16 ? bf16_to_f32(((const bf16_t*)a.g)[at + e]) : ((const float*)a.g)[at + e];
      w.m[e] = in && a.m ? a.m[at + e] : 0.f;
    }
  }
}
// what is orthogonalised, from what was fetched.  STEP: the momentum is moved first (the
// one pass that does so comes before the others).
template <bool STEP>
__device__ __forceinline__ void src_finish8(const NsSrc& a, int b, int r, int c, float coef, NsRaw& w, float (&v)[8]) {
  if (!a.m) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = w.g[e];
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float g = w.g[e] * coef;
    if (STEP) w.m[e] = w.m[e] + (g - w.m[e]) * (1.f - a.momentum);
    v[e] = g + a.momentum * (w.m[e] - g);
  }
  if (STEP) {
    const int64_t at = b * a.bs + r * a.ld + c;
    if (a.vec && c + 8 <= a.cols) {
      *reinterpret_cast<f32x4*>(a.m + at) = (f32x4){w.m[0], w.m[1], w.m[2], w.m[3]};
      *reinterpret_cast<f32x4*>(a.m + at + 4) = (f32x4){w.m[4], w.m[5], w.m[6], w.m[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < a.cols) a.m[at + e] = w.m[e];
    }
  }
}
template <bool STEP>
__device__ __forceinline__ void src_load8(const NsSrc& a, int b, int r, int c, float coef, float (&v)[8]) {
  NsRaw w;
  src_fetch8(a, b, r, c, w);
  src_finish8<STEP>(a, b, r, c, coef, w, v);
}

// momentum (in place) and the partial sums of squares of what will be orthogonalised,
// in 64 bits: squares of small gradients leave the fp32 range
__global__ __launch_bounds__(256) void ns_norm_kernel(NsSrc a, double* __restrict__ part) {
  __shared__ double red[4];
  const int b = blockIdx.y;
  const float coef = a.m ? clip_coef(a) : 1.f;
  const unsigned per_row = (a.cols + 7) / 8, chunks = per_row * a.rows, step = gridDim.x * 256;
  double acc = 0.0;
  // U chunks are fetched before the first is finished: a store in between would hold up the next load
  constexpr int U = 2;
  for (unsigned q0 = blockIdx.x * 256 + threadIdx.x; q0 < chunks; q0 += U * step) {
    NsRaw raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned q = q0 + u * step, r = q / per_row;
      if (q < chunks) src_fetch8(a, b, r, (q - r * per_row) * 8, raw[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned q = q0 + u * step, r = q / per_row;
      if (q >= chunks) continue;
      float v[8];
      src_finish8<true>(a, b, r, (q - r * per_row) * 8, coef, raw[u], v);
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (double)v[e] * (double)v[e];
      acc += s;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)b * NS_MAX_PARTS + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// A value that is split into words, or written twice, as one fp32 number.  Left to itself
// the compiler folds the operation that made it into one of its conversions to fp16 and not
// into the other: where that moves a tie (one element in 2^13) the rest is taken against another
// first word than the stored one, and a whole step of fp16 is lost.
__device__ __forceinline__ float pinned(float x) {
  asm("" : "+v"(x));
  return x;
}
__device__ __forceinline__ uint2 pack_fp8(const float (&x)[8]) {
  float v[8];       // past the largest e4m3 the conversion gives NaN
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_fmed3f(x[e], -NS_LO_MAX, NS_LO_MAX);
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], a, true);
  int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], b, true);
  return make_uint2((unsigned)a, (unsigned)b);
}
__device__ __forceinline__ void unpack_fp8(const uint2& q, float (&v)[8]) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
  const f32x2_t c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// X_0 = G / (|G| + eps), scaled, in two words, 64 x 64 at a time; a tall G goes through LDS,
// so that it is read by rows and written by rows
__global__ __launch_bounds__(256) void ns_ingest_kernel(NsSrc a, const double* __restrict__ part, int parts, double eps,
                                                        f16* __restrict__ h, uint8_t* __restrict__ lo, int sp, int lp,
                                                        int tall) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int b = blockIdx.z, tid = threadIdx.x;
  const float coef = a.m ? clip_coef(a) : 1.f;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;   // of X
  float v[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int q = tid + k * 256, y = q >> 3, x = (q & 7) * 8;
    const int r = (tall ? j0 : i0) + y, c = (tall ? i0 : j0) + x;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
    if (r < a.rows && c < a.cols) src_load8<false>(a, b, r, c, coef, v[k]);
  }
  double t = 0.0;
  for (int i = tid; i < parts; i += 256) t += part[(int64_t)b * NS_MAX_PARTS + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
  if ((tid & 63) == 0) red[tid >> 6] = t;
  __syncthreads();
  // finite, so that an all-zero matrix stays zero whatever eps (NaN stays NaN)
  const double scale = (double)NS_SX / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + eps);
  const float inv = scale > 3.4e38 ? 3.4e38f : (float)scale;
  if (tall) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int q = tid + k * 256, y = q >> 3, x = (q & 7) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[x + e][y] = v[k][e];
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int q = tid + k * 256, y = q >> 3, x = (q & 7) * 8;
    f16x8 hv;
    float lv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = pinned((tall ? tile[y][x + e] : v[k][e]) * inv);
      hv[e] = (f16)f;
      lv[e] = (f - (float)hv[e]) * NS_SL;
    }
    const int64_t at = ((int64_t)b * sp + i0 + y) * lp + j0 + x;
    *reinterpret_cast<f16x8*>(h + at) = hv;
    *reinterpret_cast<uint2*>(lo + at) = pack_fp8(lv);
  }
}

// The result in the caller's layout, and what is done with it there.
struct NsOut {
  bf16_t* out;                           // the orthogonalised matrix, or
  float* p; float* ema; bf16_t* w16;     // weights, moving average, bf16 copy
  int64_t ld, bs;
  int rows, cols;
  float step, decay, ema_omd;            // lr * scale; 1 - lr * weight_decay
  int vec;                               // rows start 16-byte aligned
};
__device__ __forceinline__ void ns_store1(const NsOut& w, int64_t at, float o) {
  if (w.out) { w.out[at] = f32_to_bf16(o); return; }
  const float p = w.p[at] * w.decay - w.step * o;
  w.p[at] = p;
  if (w.ema) { const float e = w.ema[at]; w.ema[at] = e - w.ema_omd * (e - p); }
  if (w.w16) w.w16[at] = f32_to_bf16(p);
}
// eight columns of row r, from column c (a multiple of 8) on
__device__ __forceinline__ void ns_store8(const NsOut& w, int b, int r, int c, const float (&v)[8]) {
  if (r >= w.rows) return;
  const int64_t at = b * w.bs + r * w.ld + c;
  if (!w.vec || c + 8 > w.cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < w.cols) ns_store1(w, at + e, v[e]);
    return;
  }
  float p[8];
  if (w.out) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = v[e];
  } else {
    f32x4 q[2], m[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) q[h] = *reinterpret_cast<const f32x4*>(w.p + at + 4 * h);
    if (w.ema) {
#pragma unroll
      for (int h = 0; h < 2; ++h) m[h] = *reinterpret_cast<const f32x4*>(w.ema + at + 4 * h);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e >> 2][e & 3] = p[e] = q[e >> 2][e & 3] * w.decay - w.step * v[e];
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<f32x4*>(w.p + at + 4 * h) = q[h];
    if (w.ema) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f32x4*>(w.ema + at + 4 * h) = m[h] - w.ema_omd * (m[h] - q[h]);
    }
    if (!w.w16) return;
  }
  *reinterpret_cast<uint4*>((w.out ? w.out : w.w16) + at) =
    make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7]));
}

enum { NS_GRAM = 0, NS_SQUARE = 1, NS_APPLY = 2 };

struct NsGemm {
  const f16* A; int64_t lda, bsa;    // M x K, K contiguous
  const f16* B; int64_t ldb, bsb;    // N x K, K contiguous (APPLY: K x N, N contiguous)
  int K, M, N, n;                    // of one matrix, whole tiles; n matrices
  f16* out; int64_t ldo, bso;        // D, P or the next X's high words
  uint8_t* lo;                       // APPLY: X's second words, in place
  float* diag; int sp;               // rounding of D's diagonal
  float* row_mu;                     // what a row of X's two words is multiplied by
  float* part; int splits;           // GRAM: sums of so many parts of K go here as they are (null: D is made of one)
  float shift, c, mu, p0;            // see the head of this file; p0 = a - b^2/4c - mu
  int own;                           // P's diagonal goes to row_mu whole, not its rounding alone
  int last, tall;                    // APPLY: the result goes to dst
  NsOut dst;
};

#define NS_GLDS16(gptr, lptr) \
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(gptr), \
                                   (__attribute__((address_space(3))) void*)(lptr), 16, 0, 0)

// All but the last `slabs` slabs in flight have landed, for this wave and then for
// the workgroup; this wave's own LDS reads are done too.
template <int L, int MAX>
__device__ __forceinline__ void slab_wait(int slabs) {
  if constexpr (MAX > 0) {
    if (slabs < MAX) { slab_wait<L, MAX - 1>(slabs); return; }
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(MAX * L) : "memory");
}

// T x T tile of WM x WN waves, slabs of 64 in an LDS ring of NST by LDS-DMA.
// LDS rows of a K-contiguous operand hold 64 values (128 bytes); the 16-byte chunk
// index is XORed with row & 7 on the source address and on the fragment reads.  The
// N-contiguous operand of APPLY keeps its rows (T columns) and is read through the
// transposing LDS read (four rows x 16 columns per 16 lanes); its 32-byte blocks
// are XORed so that the eight rows that half a wave reads fall into different banks.
// (APPLY has tiles of 64, 128 and 256.)  Tiles may reach past M and N: rows and columns
// are clamped on load, not stored.
template <int MODE, int T, int WM, int WN, int NST>
struct NsTile {
  static constexpr int OP = T * NS_BK * 2, STAGE = 2 * OP, RING = NST * STAGE;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int TM = T / WM, TN = T / WN, FM = TM / 16, FN = TN / 16;   // wave tile, fragments
  static constexpr int L = T * 8 / (64 * WAVES);        // LDS-DMA instructions per operand, wave and slab
  static constexpr int ER = T > 192 ? T / 2 : T;        // rows of one pass of the epilogue
  static constexpr int PITCH = T + 4, EPI = ER * PITCH; // floats
  static constexpr int LDS = RING > 4 * EPI ? RING : 4 * EPI;
  static __device__ __forceinline__ int block_xor(int row) {
    static_assert(MODE != NS_APPLY || FN == 2 || FN == 4, "transposing reads below");
    return T % 128 == 0 ? (row & 3) | (((row >> 3) & 1) << 2) : ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
  }

  static constexpr int CH = T / 8, NC = (ER * CH + THREADS - 1) / THREADS;     // epilogue: chunks per row, per thread
  // What an output needs from memory (chunks of 8 of a row) is fetched before the loop
  // where registers allow (64-tiles: few of them run and each waits for its own
  // latency), else before the sums are turned round.
  static constexpr bool EARLY = T == 64;
  struct Fetched {
    f16x8 x[NC]; uint2 lo[NC]; bool ok[NC];
    float di[EARLY || MODE == NS_APPLY ? NC : 1];      // of the row: rounding of D's diagonal, or mu
    f32x4 dj[EARLY ? NC : 1][2];
  };
  static __device__ __forceinline__ void fetch_mu(const NsGemm& g, int b, int ip, Fetched& f) {
    if constexpr (MODE == NS_APPLY) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (f.ok[c]) f.di[c] = g.row_mu[b * g.sp + ip + (threadIdx.x + c * THREADS) / CH];
    }
  }
  // One element of P's diagonal, P_ii - mu times NS_SD: what goes into P as fp16, and the
  // rest, to which X's two words are multiplied.
  static __device__ __forceinline__ float split_diag(const NsGemm& g, float q, float& row_mu) {
    q = pinned(q);
    const float in_p = g.own ? 0.f : (float)(f16)q;
    row_mu = __builtin_fmaf(q - in_p, 1.f / NS_SD, g.mu);
    return in_p;
  }
  static __device__ __forceinline__ void fetch(const NsGemm& g, int b, int i0, int ip, int j0, Fetched& f) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int q = threadIdx.x + c * THREADS, i = ip + q / CH, j = j0 + q % CH * 8;
      f.ok[c] = q < ER * CH && i < g.M && j < g.N;
      if (MODE != NS_GRAM && f.ok[c]) {
        const int64_t at = b * g.bso + (int64_t)i * g.ldo + j;
        f.x[c] = *reinterpret_cast<const f16x8*>((MODE == NS_SQUARE ? g.A : g.B) + at);
        if (MODE == NS_APPLY) f.lo[c] = *reinterpret_cast<const uint2*>(g.lo + at);
        if (MODE == NS_SQUARE && EARLY) {
          f.di[c] = g.diag[b * g.sp + i];
          f.dj[c][0] = *reinterpret_cast<const f32x4*>(g.diag + b * g.sp + j);
          f.dj[c][1] = *reinterpret_cast<const f32x4*>(g.diag + b * g.sp + j + 4);
        }
      }
    }
  }

  // The transposing reads of an N-contiguous slab at `slab`: where this lane's are, and
  // the fragments of one slab, `o` bytes further.
  static __device__ __forceinline__ void tr_setup(char* slab, int wc, int lane, unsigned (&tr)[FN]) {
    const int fr = lane & 15, fq = lane >> 4;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)slab;
    const int row = 8 * fq + (fr >> 2);       // + 4, + 32: the same XOR term
#pragma unroll
    for (int n = 0; n < FN; ++n)
      tr[n] = lds0 + row * (2 * T) + (((wc * FN + n) ^ block_xor(row)) * 32) + (lane & 3) * 8;
  }
  static __device__ __forceinline__ void read_tr(const unsigned (&tr)[FN], unsigned o, f16x8 (&bf)[2][FN]) {
    // the reads and their wait in one block: the compiler does not count them
    uint2 t[2][FN][2];
#define TR4(d0, d1, d2, d3, a)                                                              \
  "ds_read_b64_tr_b16 %" #d0 ", %" #a "\n\tds_read_b64_tr_b16 %" #d1 ", %" #a " offset:%c[o4]\n\t" \
  "ds_read_b64_tr_b16 %" #d2 ", %" #a " offset:%c[o32]\n\tds_read_b64_tr_b16 %" #d3 ", %" #a " offset:%c[o36]\n\t"
#define TRO(n) "=&v"(t[0][n][0]), "=&v"(t[0][n][1]), "=&v"(t[1][n][0]), "=&v"(t[1][n][1])
#define TRC [o4] "n"(4 * 2 * T), [o32] "n"(32 * 2 * T), [o36] "n"(36 * 2 * T)
    if constexpr (FN == 4)
      asm volatile(TR4(0, 1, 2, 3, 16) TR4(4, 5, 6, 7, 17) TR4(8, 9, 10, 11, 18) TR4(12, 13, 14, 15, 19)
                   "s_waitcnt lgkmcnt(0)"
                   : TRO(0), TRO(1), TRO(2), TRO(3)
                   : "v"(tr[0] + o), "v"(tr[1] + o), "v"(tr[2] + o), "v"(tr[3] + o), TRC : "memory");
    else
      asm volatile(TR4(0, 1, 2, 3, 8) TR4(4, 5, 6, 7, 9) "s_waitcnt lgkmcnt(0)"
                   : TRO(0), TRO(1)
                   : "v"(tr[0] + o), "v"(tr[1] + o), TRC : "memory");
#undef TR4
#undef TRO
#undef TRC
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int n = 0; n < FN; ++n)
        bf[ks][n] = __builtin_bit_cast(f16x8, make_uint4(t[ks][n][0].x, t[ks][n][0].y, t[ks][n][1].x, t[ks][n][1].y));
  }

  // The epilogue: the sums through LDS, so that global rows are read and written whole.
  static __device__ __forceinline__ void finish(const NsGemm& g, int b, int tm, int tn, int k_part, const Fetched& early,
                                                const f32x4 (&acc)[FM][FN], char* smem) {
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid / WN, wc = wid % WN, fr = lane & 15, fq = lane >> 4;
    const int i0 = tm * T, j0 = tn * T;
    float* const tile = reinterpret_cast<float*>(smem);
    // the other side of a symmetric product, or a tall matrix's own orientation
    const bool turn = MODE == NS_APPLY ? g.last && g.tall : tm != tn;
#pragma unroll
    for (int part = 0; part < T / ER; ++part) {
      const int ip = i0 + part * ER;
      Fetched late;
      if (!EARLY) { fetch(g, b, i0, ip, j0, late); fetch_mu(g, b, ip, late); }
      const Fetched& f = EARLY ? early : late;
      __syncthreads();
      if (T == ER || wr * TM / ER == part) {
        float* const own = tile + (wr * TM - part * ER) * PITCH;
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
          for (int n = 0; n < FN; ++n)
            *reinterpret_cast<f32x4*>(own + (m * 16 + fr) * PITCH + wc * TN + n * 16 + fq * 4) = acc[m][n];
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!f.ok[c]) continue;
        const int q = tid + c * THREADS, r = q / CH, pc = q % CH * 8, i = ip + r, j = j0 + pc;
        const int64_t at = b * g.bso + (int64_t)i * g.ldo + j;
        f32x4* const t4 = reinterpret_cast<f32x4*>(tile + r * PITCH + pc);
        const f32x4 v0 = t4[0], v1 = t4[1];
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < 4 ? v0[e & 3] : v1[e & 3];
        const int on_diag = i - j;                 // 0..7: element of the chunk on the diagonal
        if (MODE == NS_GRAM && g.part) {
          float* const to = g.part + (((int64_t)b * g.splits + k_part) * g.sp + i) * g.sp + j;
          *reinterpret_cast<f32x4*>(to) = v0;
          *reinterpret_cast<f32x4*>(to + 4) = v1;
          continue;
        }
        if constexpr (MODE == NS_GRAM) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= NS_SD / (NS_SX * NS_SX);
          if (on_diag >= 0 && on_diag < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e == on_diag) {
                x[e] = pinned(x[e] + g.shift * NS_SD);
                g.diag[b * g.sp + i] = x[e] - (float)(f16)x[e];
              }
          }
        } else if constexpr (MODE == NS_SQUARE) {
          const float di = EARLY ? f.di[EARLY ? c : 0] : g.diag[b * g.sp + i];
          const f32x4 d0 = EARLY ? f.dj[EARLY ? c : 0][0] : *reinterpret_cast<const f32x4*>(g.diag + b * g.sp + j);
          const f32x4 d1 = EARLY ? f.dj[EARLY ? c : 0][1] : *reinterpret_cast<const f32x4*>(g.diag + b * g.sp + j + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = (x[e] + (di + (e < 4 ? d0[e & 3] : d1[e & 3])) * (float)f.x[c][e]) * (g.c / NS_SD);
          if (on_diag >= 0 && on_diag < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e == on_diag) {
                float m;
                x[e] = split_diag(g, x[e] + g.p0 * NS_SD, m);
                g.row_mu[b * g.sp + i] = m;
              }
          }
        } else {
          const float sc = g.last ? 1.f / NS_SX : 1.f;
          float l8[8];
          unpack_fp8(f.lo[c], l8);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = (f.di[c] * __builtin_fmaf(l8[e], 1.f / NS_SL, (float)f.x[c][e]) + x[e] * (1.f / NS_SD)) * sc;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = pinned(x[e]);
        if (turn) { t4[0] = (f32x4){x[0], x[1], x[2], x[3]}; t4[1] = (f32x4){x[4], x[5], x[6], x[7]}; }
        if (MODE == NS_APPLY && g.last) {
          if (!turn) ns_store8(g.dst, b, i, j, x);
          continue;
        }
        f16x8 hv;
#pragma unroll
        for (int e = 0; e < 8; ++e) hv[e] = (f16)x[e];
        *reinterpret_cast<f16x8*>(g.out + at) = hv;
        if constexpr (MODE == NS_APPLY) {
          float lv[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) lv[e] = (x[e] - (float)hv[e]) * NS_SL;
          *reinterpret_cast<uint2*>(g.lo + at) = pack_fp8(lv);
        }
      }
      if (turn && !(MODE == NS_GRAM && g.part)) {      // 16 columns x 4 chunks of 8 rows per wave and pass
        __syncthreads();
        constexpr int UNITS = (T / 16) * (ER / 32);
#pragma unroll 4
        for (int q = wid; q < UNITS; q += WAVES) {
          const int jj = (q % (T / 16)) * 16 + fr, ii = (q / (T / 16)) * 32 + fq * 8;
          const int i = ip + ii, j = j0 + jj;
          if (i >= g.M || j >= g.N) continue;
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = tile[(ii + e) * PITCH + jj];
          if constexpr (MODE == NS_APPLY) {
            ns_store8(g.dst, b, j, i, x);
          } else {
            f16x8 hv;
#pragma unroll
            for (int e = 0; e < 8; ++e) hv[e] = (f16)x[e];
            *reinterpret_cast<f16x8*>(g.out + b * g.bso + (int64_t)j * g.ldo + i) = hv;
          }
        }
      }
    }
  }

  static __device__ __forceinline__ void run(const NsGemm& g, int b, int tm, int tn, int part, char* smem) {
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid / WN, wc = wid % WN, fr = lane & 15, fq = lane >> 4;
    const int i0 = tm * T, j0 = tn * T;
    // the slabs of this part (GRAM may be split over K)
    const int KT0 = MODE == NS_GRAM ? part * (g.K / NS_BK) / g.splits : 0;
    const int KT = (MODE == NS_GRAM ? (part + 1) * (g.K / NS_BK) / g.splits : g.K / NS_BK) - KT0;
    const f16* A = g.A + b * g.bsa + KT0 * NS_BK;
    const f16* B = g.B + b * g.bsb + KT0 * NS_BK;
    unsigned aoff[L], boff[L];       // of this lane's 16 bytes of each instruction
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int row = (i * WAVES + wid) * 8 + (lane >> 3), ch = ((lane & 7) ^ (row & 7)) * 8;
      const int ai = i0 + row < g.M ? i0 + row : g.M - 1;
      aoff[i] = (unsigned)((ai - i0) * (int)g.lda + ch);
      if constexpr (MODE == NS_APPLY) {
        const int q = (i * WAVES + wid) * 64 + lane, k = q / (T / 8), pch = q % (T / 8);
        int j = j0 + (((pch >> 1) ^ block_xor(k)) * 2 + (pch & 1)) * 8;
        j = j < g.N ? j : g.N - 8;
        boff[i] = (unsigned)(k * (int)g.ldb + (j - j0));
      } else {
        const int bj = j0 + row < g.N ? j0 + row : g.N - 1;
        boff[i] = (unsigned)((bj - j0) * (int)g.ldb + ch);
      }
    }
    A += (int64_t)i0 * g.lda;
    B += MODE == NS_APPLY ? (int64_t)j0 : (int64_t)j0 * g.ldb;
    auto stage = [&](int st, int k0) {
      char* const sb = smem + st * STAGE;
      const f16* a = A + k0;
      const f16* bb = B + (MODE == NS_APPLY ? (int64_t)k0 * g.ldb : (int64_t)k0);
#pragma unroll
      for (int i = 0; i < L; ++i) {
        NS_GLDS16(a + aoff[i], sb + (i * WAVES + wid) * 1024);
        NS_GLDS16(bb + boff[i], sb + OP + (i * WAVES + wid) * 1024);
      }
    };
    int foff[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) foff[ks] = fr * 128 + (((ks * 4 + fq) ^ (lane & 7)) * 16);
    const int a_base = wr * TM * 128, b_base = OP + wc * TN * 128;
    unsigned tr[FN];
    if constexpr (MODE == NS_APPLY) tr_setup(smem + OP, wc, lane, tr);
    Fetched early;
    if (EARLY) { fetch(g, b, i0, i0, j0, early); fetch_mu(g, b, i0, early); }
    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};

    auto read_a = [&](const char* sb, int ks, f16x8 (&f)[FM]) {
#pragma unroll
      for (int m = 0; m < FM; ++m) f[m] = *reinterpret_cast<const f16x8*>(sb + a_base + m * 2048 + foff[ks]);
    };
    auto read_b = [&](const char* sb, int ks, f16x8 (&f)[FN]) {
#pragma unroll
      for (int n = 0; n < FN; ++n) f[n] = *reinterpret_cast<const f16x8*>(sb + b_base + n * 2048 + foff[ks]);
    };
    // swapped operands: a lane holds four consecutive columns of one output row
    auto mma = [&](const f16x8 (&fa)[FM], const f16x8 (&fb)[FN]) {
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[n], fa[m], acc[m][n], 0, 0, 0);
    };
    if constexpr (MODE != NS_APPLY) {
#pragma unroll
      for (int i = 0; i < NST; ++i)
        if (i < KT) stage(i, i * NS_BK);
      slab_wait<2 * L, NST - 1>(KT - 1);
      f16x8 a0[FM], b0[FN], a1[FM], b1[FN];
      read_a(smem, 0, a0);
      read_b(smem, 0, b0);
      int st = 0, kt = 0;
      // a round: the second half's fragments are read under the first half's products,
      // the next slab's first half and its DMA under the second half's (left to itself
      // the compiler puts all reads and one wait in front: 10 - 20 % slower)
      for (; kt + NST < KT; ++kt) {
        const char* sb = smem + st * STAGE;
        read_a(sb, 1, a1);
        read_b(sb, 1, b1);
        mma(a0, b0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
        for (int i = 0; i < FM + FN; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NST - 2) * 2 * L) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        stage(st, (kt + NST) * NS_BK);
        st = st + 1 == NST ? 0 : st + 1;
        sb = smem + st * STAGE;
        read_a(sb, 0, a0);
        read_b(sb, 0, b0);
        mma(a1, b1);
#pragma unroll
        for (int i = 0; i < FM + FN; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      for (; kt < KT; ++kt) {          // the last NST slabs: nothing left to fetch
        read_a(smem + st * STAGE, 1, a1);
        read_b(smem + st * STAGE, 1, b1);
        mma(a0, b0);
        st = st + 1 == NST ? 0 : st + 1;
        if (kt + 1 < KT) {
          slab_wait<2 * L, NST - 2>(KT - 2 - kt);
          read_a(smem + st * STAGE, 0, a0);
          read_b(smem + st * STAGE, 0, b0);
        }
        mma(a1, b1);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NST - 1; ++i)
        if (i < KT) stage(i, i * NS_BK);
      int st = 0, st_in = NST - 1;      // ring slots read and filled next
      for (int kt = 0; kt < KT; ++kt) {
        slab_wait<2 * L, NST - 2>(KT - 1 - kt);
        if (kt + NST - 1 < KT) stage(st_in, (kt + NST - 1) * NS_BK);
        const char* sb = smem + st * STAGE;
        f16x8 af[2][FM], bf[2][FN];
        read_a(sb, 0, af[0]);
        read_a(sb, 1, af[1]);
        read_tr(tr, st * STAGE, bf);
        mma(af[0], bf[0]);
        mma(af[1], bf[1]);
        st = st + 1 == NST ? 0 : st + 1;
        st_in = st_in + 1 == NST ? 0 : st_in + 1;
      }
    }

    finish(g, b, tm, tn, part, early, acc, smem);
  }
};

// Tiles of GRAM and SQUARE: the lower triangle of a symmetric result (t = 0: (0,0),
// then (1,0), (1,1), ..).
__device__ __forceinline__ void triangle(int t, int& tm, int& tn) {
  tm = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while (tm * (tm + 1) / 2 > t) --tm;
  while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
  tn = t - tm * (tm + 1) / 2;
}

template <int MODE, int T, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN, T <= 128 ? 2 : WM * WN / 4) void ns_gemm_kernel(NsGemm g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tiles_m = (g.M + T - 1) / T, tiles_n = (g.N + T - 1) / T;
  const int per_mat = MODE == NS_APPLY ? tiles_m * tiles_n : tiles_m * (tiles_m + 1) / 2;
  const int splits = MODE == NS_GRAM ? g.splits : 1, total = per_mat * splits * g.n;
  // each XCD (workgroup id & 7) gets a contiguous range of tiles
  const int per_xcd = (total + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || idx >= total) return;
  const int u = idx / per_mat, t = idx - u * per_mat, b = u / splits, part = u - b * splits;
  int tm, tn;
  if (MODE == NS_APPLY) { tn = t / tiles_m; tm = t - tn * tiles_m; }     // X's columns are read once per XCD
  else triangle(t, tm, tn);
  NsTile<MODE, T, WM, WN, NST>::run(g, b, tm, tn, part, smem);
}

// SQUARE and APPLY of matrices whose short side fits into 128 rows, in one launch: a
// launch costs 4 us there, the products next to nothing (us per call, three launches per
// step / two: 2 x 384 x 128: 67 / 60, 128 x 4096: 124 / 81, 16 x 6000: 141 / 67,
// 300 x 100 x 140: 202 / 174, 64 x 128 x 2048: 200 / 204; before P's diagonal went to mu, which costs
// 1 .. 4 %: 63, 83, 70, 181, 200 now).  Every workgroup sums D from the
// parts that GRAM left, makes 64 rows of P in LDS and multiplies `group` 64 x 64 tiles of X
// by them, the next one's X on its way meanwhile.  LDS rows as in NsTile.
template <int S>
__global__ __launch_bounds__(256) void ns_step_kernel(NsGemm g, int group) {
  using Tile = NsTile<NS_APPLY, 64, 2, 2, 4>;
  constexpr int KS = S / 64, DSLAB = S * 128, SLAB = 64 * 128;
  // D; later the epilogue's tile and X's second buffer
  constexpr int DBYTES = KS * DSLAB > 4 * Tile::EPI + KS * SLAB ? KS * DSLAB : 4 * Tile::EPI + KS * SLAB;
  __shared__ __attribute__((aligned(16))) char dm[DBYTES];
  __shared__ __attribute__((aligned(16))) char xs[KS * SLAB];
  __shared__ __attribute__((aligned(16))) char ps[KS * SLAB];
  __shared__ __attribute__((aligned(16))) float diag[S];
  __shared__ float row_mu[64];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid >> 1, wc = wid & 1, fr = lane & 15, fq = lane >> 4;
  const int tiles_n = g.N / 64, per_mat = KS * ((tiles_n + group - 1) / group), total = per_mat * g.n, per_xcd = (total + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || idx >= total) return;
  const int b = idx / per_mat, t = idx - b * per_mat, grp = t / KS, tm = t - grp * KS;
  const int i0 = tm * 64, tn0 = grp * group, tn1 = tn0 + group < tiles_n ? tn0 + group : tiles_n;
  const f16* X = g.B + b * g.bsb;
  auto stage = [&](int tn, char* to) {
#pragma unroll
    for (int kt = 0; kt < KS; ++kt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = (i * 4 + wid) * 64 + lane, k = q >> 3, pch = q & 7;
        const int j = (((pch >> 1) ^ Tile::block_xor(k)) * 2 + (pch & 1)) * 8;
        NS_GLDS16(X + (int64_t)(kt * 64 + k) * g.ldb + tn * 64 + j, to + kt * SLAB + (i * 4 + wid) * 1024);
      }
  };
  typename Tile::Fetched own;
  Tile::fetch(g, b, i0, i0, tn0 * 64, own);
  stage(tn0, xs);
  // ---- D: the lower triangle's tiles (0,0), (1,0), (1,1), two chunks of 8 per thread and tile
  constexpr int C = KS * (KS + 1);
  f32x4 v[C][2];
#pragma unroll
  for (int c = 0; c < C; ++c) v[c][0] = v[c][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < g.splits; ++p) {
    const float* part = g.part + ((int64_t)b * g.splits + p) * (S * S);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int q = tid + (c & 1) * 256, i = (c > 1 ? 64 : 0) + (q >> 3), j = (c > 3 ? 64 : 0) + (q & 7) * 8;
      v[c][0] += *reinterpret_cast<const f32x4*>(part + i * S + j);
      v[c][1] += *reinterpret_cast<const f32x4*>(part + i * S + j + 4);
    }
  }
  auto at = [](int row, int col, int slab) { return (col >> 6) * slab + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) * 16) + (col & 7) * 2; };
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int q = tid + (c & 1) * 256, i = (c > 1 ? 64 : 0) + (q >> 3), j = (c > 3 ? 64 : 0) + (q & 7) * 8;
    f16x8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = v[c][e >> 2][e & 3] * (NS_SD / (NS_SX * NS_SX));
      if (i == j + e) x += g.shift * NS_SD;
      x = pinned(x);
      h[e] = (f16)x;
      if (i == j + e) diag[i] = x - (float)h[e];
    }
    *reinterpret_cast<f16x8*>(dm + at(i, j, DSLAB)) = h;
    if (c == 2 || c == 3) {       // the other side
#pragma unroll
      for (int e = 0; e < 8; ++e) *reinterpret_cast<f16*>(dm + at(j + e, i, DSLAB)) = h[e];
    }
  }
  slab_wait<0, 0>(0);
  // ---- P, 64 rows of it
  constexpr int FN = S / 32;
  {
    f32x4 acc[2][FN];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 2 * KS; ++ks) {
      f16x8 fa[2], fb[FN];
      const int col = ks * 32 + fq * 8;
#pragma unroll
      for (int m = 0; m < 2; ++m) fa[m] = *reinterpret_cast<const f16x8*>(dm + at(i0 + wr * 32 + m * 16 + fr, col, DSLAB));
#pragma unroll
      for (int n = 0; n < FN; ++n) fb[n] = *reinterpret_cast<const f16x8*>(dm + at(wc * (S / 2) + n * 16 + fr, col, DSLAB));
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[n], fa[m], acc[m][n], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const int r = wr * 32 + m * 16 + fr, i = i0 + r, j = wc * (S / 2) + n * 16 + fq * 4;
        const f16x4 d = *reinterpret_cast<const f16x4*>(dm + at(i, j, DSLAB));
        const float di = diag[i];
        const f32x4 dj = *reinterpret_cast<const f32x4*>(diag + j);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (acc[m][n][e] + (di + dj[e]) * (float)d[e]) * (g.c / NS_SD);
        if (i0 + wr * 32 + m * 16 == wc * (S / 2) + n * 16) {      // one branch per wave
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i == j + e) x[e] = Tile::split_diag(g, x[e] + g.p0 * NS_SD, row_mu[r]);
        }
        const f16x4 h = {(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3]};
        *reinterpret_cast<f16x4*>(ps + at(r, j, SLAB)) = h;
      }
  }
  // ---- P X
  for (int tn = tn0; tn < tn1; ++tn) {
    // this tile's X has landed and the other buffer is free (first time: P is there, D done with)
    slab_wait<0, 0>(0);
    char* const cur = (tn - tn0) & 1 ? dm + 4 * Tile::EPI : xs;
    typename Tile::Fetched next;
    if (tn + 1 < tn1) {
      Tile::fetch(g, b, i0, i0, (tn + 1) * 64, next);
      stage(tn + 1, (tn - tn0) & 1 ? xs : dm + 4 * Tile::EPI);
    }
    f32x4 acc[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    unsigned tr[2];
    Tile::tr_setup(cur, wc, lane, tr);
#pragma unroll
    for (int kt = 0; kt < KS; ++kt) {
      f16x8 bf[2][2];
      Tile::read_tr(tr, kt * SLAB, bf);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const f16x8 fa = *reinterpret_cast<const f16x8*>(ps + at(wr * 32 + m * 16 + fr, kt * 64 + ks * 32 + fq * 8, SLAB));
#pragma unroll
          for (int n = 0; n < 2; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[ks][n], fa, acc[m][n], 0, 0, 0);
        }
    }
#pragma unroll
    for (int c = 0; c < Tile::NC; ++c) own.di[c] = row_mu[(tid + c * Tile::THREADS) / Tile::CH];
    Tile::finish(g, b, tm, tn, 0, own, acc, dm);
    own = next;
  }
}
static int ns_step(const NsGemm& g, int cus, hipStream_t st) {
  // as many tiles per workgroup as leave two workgroups per CU (what LDS has room for); us per
  // call with one tile each / four workgroups per CU / two / one: 64 x 128 x 2048:
  // 405 / 228 / 204 / 234, 4 x 128 x 8192: 177 / 167 / 131 / 131
  const int tiles_n = g.N / 64;
  int64_t group = ((int64_t)(g.M / 64) * tiles_n * g.n + 2 * cus - 1) / (2 * cus);
  if (group > tiles_n) group = tiles_n;
  const int64_t total = (int64_t)(g.M / 64) * ((tiles_n + group - 1) / group) * g.n;
  if (total >= (1ll << 28)) { set_error("orthogonalize: too many tiles"); return -1; }
  const unsigned grid = (unsigned)((total + 7) / 8 * 8);
  if (g.M == 64) ns_step_kernel<64><<<grid, 256, 0, st>>>(g, (int)group);
  else ns_step_kernel<128><<<grid, 256, 0, st>>>(g, (int)group);
  MDLM_LAUNCH_CHECK();
  return 0;
}

static int64_t ns_tiles(int mode, const NsGemm& g, int T) {
  const int64_t tm = (g.M + T - 1) / T, tn = (g.N + T - 1) / T;
  return (mode == NS_APPLY ? tm * tn : tm * (tm + 1) / 2 * (mode == NS_GRAM ? g.splits : 1)) * g.n;
}
template <int MODE, int T, int WM, int WN, int NST>
static int ns_launch(const NsGemm& g, hipStream_t st) {
  constexpr int LDS = NsTile<MODE, T, WM, WN, NST>::LDS;
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static bool done[MAX_DEVICES] = {};
  if (int rc = ensure_dynamic_lds(&ns_gemm_kernel<MODE, T, WM, WN, NST>, LDS, done, "orthogonalize")) return rc;
  const int64_t total = ns_tiles(MODE, g, T);
  if (total >= (1ll << 28)) { set_error("orthogonalize: too many tiles"); return -1; }
  ns_gemm_kernel<MODE, T, WM, WN, NST><<<(unsigned)((total + 7) / 8 * 8), 64 * WM * WN, LDS, st>>>(g);
  MDLM_LAUNCH_CHECK();
  return 0;
}
// Which tile.  Up to 256 tiles of 128 x 128 (one per CU) the smaller 64 x 64 ones fill the
// chip better; their ring is deep (4 slabs) while a CU holds at most two of them and
// shallow (2 slabs, five workgroups per CU) beyond.  Measured, us per product:
//   A of 768 x 768:            64: 6.2 / 8.9 (deep / shallow)   128: 13
//   A of 1024 x 4096:          64: 16 / 30                      128: 41
//   A of 2048 x 2048:          64: 22 / 19                      128: 25
// For the symmetric products 96 x 96 tiles are in between, where all of them are resident
// at once (two workgroups per CU) and not too few to fill it (64 shallow / 96 / 128):
//   A of 12 x 768 x 2304: 31 / 28 / 30   A of 6 x 768 x 2304: 20 / 18 / 28   A of 2 x 2048 x 8192: 140 / 86 / 106
// With more, the rounds of tiles that a CU goes through, times what a slab of one
// costs with the chip full (us, measured on 4096 x 4096: 128: 0.59 in pairs, 192:
// 1.16, 256: 1.5; P X: 128: 0.54, 256: 2.0):
//   A of 4096 x 8192:          128: 196   192: 139   256: 179
//   A of 24 x 1024 x 4096:     128: 139   192: 140   256: 121
//   P X of 24 x 1024 x 4096:   128: 353   256: 303
//   P X of 12 x 768 x 2304:    128: 52    256: 68
template <int MODE>
static int ns_gemm(const NsGemm& g, int cus, hipStream_t st) {
  const int64_t t128 = ns_tiles(MODE, g, 128);
  if constexpr (MODE != NS_APPLY) {
    const int64_t t96 = ns_tiles(MODE, g, 96);
    if (t96 * 5 >= cus * 4 && t96 <= 2 * cus) return ns_launch<MODE, 96, 2, 2, 3>(g, st);
  }
  if (t128 <= cus)
    return ns_tiles(MODE, g, 64) <= 2 * cus ? ns_launch<MODE, 64, 2, 2, 4>(g, st) : ns_launch<MODE, 64, 2, 2, 2>(g, st);
  auto rounds = [&](int T, int slots) { return (double)((ns_tiles(MODE, g, T) + slots - 1) / slots); };
  const double c128 = rounds(128, 2 * cus) * 2 * (MODE == NS_APPLY ? 0.54 : 0.59);
  const double c256 = rounds(256, cus) * (MODE == NS_APPLY ? 2.0 : 1.5);
  if constexpr (MODE != NS_APPLY) {
    const double c192 = rounds(192, cus) * 1.16;
    if (c192 < c128 && c192 <= c256) return ns_launch<MODE, 192, 2, 4, 3>(g, st);
  }
  return c256 < c128 ? ns_launch<MODE, 256, 2, 4, 2>(g, st) : ns_launch<MODE, 128, 2, 2, 2>(g, st);
}

static inline double ns_mu(int it, int steps, double a) {
  return it + 3 < steps ? a : 1.0;
}
// Whether X, D and P - mu I stay in the range of fp16 with their scales, whatever the matrix:
// an entry is at most the largest singular value, X_0's are in [0, 1], and each step maps [0, s]
// by s p(s^2), p(t) = a + b t + c t^2, which has its extremes at the ends and where its derivative is 0.
static bool ns_in_range(int steps, double a, double b, double c) {
  const double most_x = 65504 / NS_SX * 0.97, most_p = 65504 / NS_SD * 0.97;      // less what roundings add
  double s = 1.0;
  for (int it = 0; it < steps; ++it) {
    const double t = s * s, mu = ns_mu(it, steps, a), shift = b / (2 * c);
    auto p = [&](double u) { return a + u * (b + c * u); };
    double dp = fmax(fabs(a - mu), fabs(p(t) - mu));
    if (-shift > 0 && -shift < t) dp = fmax(dp, fabs(p(-shift) - mu));
    if (!(fmax(fabs(shift), fmax(fabs(t + shift), t)) < most_p) || !(dp < most_p)) return false;
    double next = fabs(s * p(t));
    const double disc = 9 * b * b - 20 * a * c;
    if (disc >= 0)
      for (double u : {(-3 * b + sqrt(disc)) / (10 * c), (-3 * b - sqrt(disc)) / (10 * c)})
        if (u > 0 && u < t) next = fmax(next, fabs(sqrt(u) * p(u)));
    s = next;
    if (it + 1 < steps && !(s < most_x)) return false;
  }
  return true;
}
static int ns_run(NsSrc src, NsOut dst, int n, int rows, int cols, int steps, double a, double b, double c,
                  double eps, void* ws, hipStream_t st) {
  const int dev = current_device();
  if (dev < 0) return -1;
  const int cus = device_cus(dev);
  const NsShape q = ns_shape(rows, cols);
  NsWs w;
  ns_layout(q, n, (char*)ws, &w);
  dst.rows = rows; dst.cols = cols;
  dst.vec = (dst.ld | dst.bs) % 8 == 0 &&
            (((uintptr_t)dst.out | (uintptr_t)dst.p | (uintptr_t)dst.ema | (uintptr_t)dst.w16) & 15) == 0;
  src.rows = rows; src.cols = cols;
  src.vec = (src.ld | src.bs) % 8 == 0 && (((uintptr_t)src.g | (uintptr_t)src.m) & 15) == 0;
  // some 2048 workgroups over all matrices, eight columns per thread and turn
  const int64_t want = ((int64_t)rows * ((cols + 7) / 8) + 255) / 256, most = 2048 / n > 1 ? 2048 / n : 1;
  int parts = (int)(want < most ? want : most);
  if (parts > NS_MAX_PARTS) parts = NS_MAX_PARTS;
  ns_norm_kernel<<<dim3(parts, n), 256, 0, st>>>(src, w.norm);
  MDLM_LAUNCH_CHECK();
  ns_ingest_kernel<<<dim3(q.lp / 64, q.sp / 64, n), 256, 0, st>>>(src, w.norm, parts, eps, w.h[0], w.lo, q.sp, q.lp, q.tall);
  MDLM_LAUNCH_CHECK();
  const int64_t bx = (int64_t)q.sp * q.lp, bd = (int64_t)q.sp * q.sp;
  for (int it = 0; it < steps; ++it) {
    const double mu = ns_mu(it, steps, a);
    f16 *x = w.h[it & 1], *xn = w.h[(it & 1) ^ 1];
    NsGemm g = {};
    g.n = n; g.sp = q.sp; g.diag = w.diag; g.row_mu = w.mu; g.part = w.part; g.splits = q.splits;
    g.mu = (float)mu; g.p0 = (float)(a - b * b / (4 * c) - mu); g.own = it + 3 >= steps;
    g.A = x; g.lda = q.lp; g.bsa = bx; g.B = x; g.ldb = q.lp; g.bsb = bx; g.K = q.lp;
    g.M = g.N = q.sp;
    g.out = w.d; g.ldo = q.sp; g.bso = bd; g.shift = (float)(b / (2 * c));
    if (int rc = w.part ? ns_launch<NS_GRAM, 64, 2, 2, 4>(g, st) : ns_gemm<NS_GRAM>(g, cus, st)) return rc;
    g.A = w.d; g.lda = q.sp; g.bsa = bd; g.B = w.d; g.ldb = q.sp; g.bsb = bd; g.K = q.sp;
    g.out = w.p; g.c = (float)c;
    if (!w.part)
      if (int rc = ns_gemm<NS_SQUARE>(g, cus, st)) return rc;
    g.A = w.p; g.B = x; g.ldb = q.lp; g.bsb = bx; g.N = q.lp;
    g.out = xn; g.ldo = q.lp; g.bso = bx; g.lo = w.lo;
    g.last = it + 1 == steps; g.tall = q.tall; g.dst = dst;
    if (int rc = w.part ? ns_step(g, cus, st) : ns_gemm<NS_APPLY>(g, cus, st)) return rc;
  }
  return 0;
}

// shapes and coefficients that every entry point here shares
static int ns_check(const char* who, int n, int rows, int cols, int64_t ld, int64_t bs, int steps, double a, double b,
                    double c, double eps) {
  MDLM_CHECK_ARG(n > 0 && n < 65536 && rows > 0 && cols > 0 && rows <= (1 << 17) && cols <= (1 << 17),
                 "%s: bad shape", who);
  MDLM_CHECK_ARG((rows < cols ? rows : cols) <= NS_MAX_SIDE, "%s: the smaller side must be at most %d", who, NS_MAX_SIDE);
  // one matrix behind the other, or side by side within a row
  MDLM_CHECK_ARG(ld >= cols && (n == 1 || bs >= (int64_t)(rows - 1) * ld + cols ||
                                (bs >= cols && ld >= (int64_t)(n - 1) * bs + cols)),
                 "%s: overlapping rows or matrices", who);
  MDLM_CHECK_ARG(steps >= 1 && steps <= 32, "%s: steps=%d is outside 1..32", who, steps);
  // the completed square's constant is what rounding D costs: 2.8 for the usual coefficients
  MDLM_CHECK_ARG(isfinite(a) && isfinite(b) && isfinite(c) && fabs(a) <= 16 && c != 0.0 && fabs(c) <= 32 &&
                   fabs(b * b / (4 * c)) <= 16,
                 "%s: coefficients (%g, %g, %g) are outside what the fp16 products hold", who, a, b, c);
  MDLM_CHECK_ARG(ns_in_range(steps, a, b, c),
                 "%s: coefficients (%g, %g, %g) can leave the range of the fp16 products in %d steps", who, a, b, c, steps);
  MDLM_CHECK_ARG(eps > 0.0 && isfinite(eps), "%s: eps must be positive", who);
  return 0;
}

}  // namespace mdlm

using namespace mdlm;

extern "C" int64_t mdlm_orthogonalize_workspace_bytes(int n, int rows, int cols) {
  if (n <= 0 || rows <= 0 || cols <= 0 || n >= 65536 || rows > (1 << 17) || cols > (1 << 17) ||
      (rows < cols ? rows : cols) > NS_MAX_SIDE)
    return -1;
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
  MDLM_CHECK_ARG(p != g && p != m && g != m && ema != p && ema != m && (!ema || ema != g) && w_bf16 != (void*)p &&
                   w_bf16 != (void*)m && (!w_bf16 || (w_bf16 != (void*)ema && w_bf16 != (const void*)g)),
                 "muon_update: the buffers must be different ones");
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
