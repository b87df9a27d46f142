// Newton-Schulz orthogonalisation: X = G / (|G|_F + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T (G taken p x q, p <= q).
//
// Three products a step, all of the form sum_k P[i][k] Q[j][k] (nls_tile.h): A = X X^T and B = b A + c A A^T are symmetric - the tiles on and below
// the diagonal are computed and written twice - and B X reads the transposed copy of X that the step before wrote beside X.
//
// Every matrix between the products is held as a pair of fp16, hi + lo: 22 significant bits, scaled by a power of two that follows from a bound on
// the singular values (polynomial extrema, from the norm on), so that entries stay below 2^15 and neither half leaves fp16's range.  A product of
// pairs is hi hi + lo hi + hi lo (the dropped lo lo is below 2^-22 of a term), three matrix instructions at 16 x the rate of the fp32 one.
#pragma once
#include <cmath>

#include "nls_tile.h"

namespace lb {

constexpr int NS_MAX_STEPS = 32;
constexpr int NS_PARTS = 256;  // partial sums of squares a matrix

// X_t, A_t, B_t are held times 2^ex, 2^ea, 2^eb (of their step); what a product's sum w becomes the next held matrix with:
struct NsFactors {
  float gram;            // A: gram w
  float lin, quad;       // B: lin A + quad w
  float keep, add;       // next X: keep X + add w
};
struct NsScales {  // one per matrix
  double first;    // G to held X_0; NaN when the norm is not finite: the whole result is then NaN
  int last;        // the result is held X times 2^last
  NsFactors f[NS_MAX_STEPS];
};
// A step's polynomial a s + b s^3 + c s^5 and where it and b z + c z^2 have their extrema (host: ns_coefficients)
struct NsStep {
  double a, b, c;
  double xs[2], xv[2];   // s > 0 and the absolute value there
  double zs, zv;
};
struct NsCoef {
  NsStep s[NS_MAX_STEPS];
};

// A matrix of fp16 pairs: granules of 32 elements, 64 bytes hi then 64 bytes lo; rows padded with zeros to 64 elements.
__host__ __device__ inline size_t pair_ld(long k) { return (size_t)((k + 63) / 64 * 64) * 4; }
__device__ __forceinline__ size_t pair_at(size_t row, size_t k, size_t ld) { return row * ld + (k >> 5) * 128 + (k & 31) * 2; }

struct NsMatrix {
  const void* g;
  long p, q;                       // p <= q
  long row_stride, col_stride, batch_stride;  // in elements
};

template <class T>
__global__ __launch_bounds__(256) void k_ns_norm(NsMatrix w, double* parts) {
  const T* g = (const T*)w.g + blockIdx.y * w.batch_stride;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  double s = 0.0;
  // lanes along the direction whose neighbours are neighbours in memory
  const bool along_q = w.col_stride <= w.row_stride;
  const long outer = along_q ? w.p : w.q, inner = along_q ? w.q : w.p;
  const long os = along_q ? w.row_stride : w.col_stride, is = along_q ? w.col_stride : w.row_stride;
  for (long o = (long)blockIdx.x * 4 + y; o < outer; o += (long)gridDim.x * 4)
    for (long i = x; i < inner; i += 64) {
      const double v = (double)to_f32(g[o * os + i * is]);
      s += v * v;
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  __shared__ double part[4];
  if (x == 0) part[y] = s;
  __syncthreads();
  if (threadIdx.x == 0) parts[(size_t)blockIdx.y * NS_PARTS + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

inline void ns_step(double a, double b, double c, NsStep* o) {
  *o = NsStep{a, b, c, {INFINITY, INFINITY}, {0.0, 0.0}, INFINITY, 0.0};
  auto at = [&](int k, double z) {  // z = s^2
    if (!(z > 0.0) || !std::isfinite(z)) return;
    o->xs[k] = std::sqrt(z);
    o->xv[k] = std::fabs(o->xs[k] * (a + z * (b + c * z)));
  };
  const double d = 9.0 * b * b - 20.0 * a * c;
  if (c != 0.0 && d >= 0.0) {
    at(0, (-3.0 * b - std::sqrt(d)) / (10.0 * c));
    at(1, (-3.0 * b + std::sqrt(d)) / (10.0 * c));
  } else if (c == 0.0 && b != 0.0) {
    at(0, -a / (3.0 * b));
  }
  if (c != 0.0 && -b / (2.0 * c) > 0.0) {
    o->zs = -b / (2.0 * c);
    o->zv = std::fabs(o->zs * (b + c * o->zs));
  }
}
__host__ __device__ inline double ns_peak_x(const NsStep& s, double u) {  // max |a s + b s^3 + c s^5| on [0, u]
  double top = fabs(u * (s.a + u * u * (s.b + s.c * u * u)));
  if (s.xs[0] < u) top = fmax(top, s.xv[0]);
  if (s.xs[1] < u) top = fmax(top, s.xv[1]);
  return top;
}
__host__ __device__ inline double ns_peak_b(const NsStep& s, double u) {  // max |b z + c z^2| on [0, u^2]
  const double z = u * u, top = fabs(z * (s.b + s.c * z));
  return s.zs < z ? fmax(top, s.zv) : top;
}
// 15 - e with |v| < 2^e: what is bounded by v is held below 2^15 (fp16 ends at 65504: a factor of two for the roundings)
__device__ __forceinline__ int ns_exponent(double v) {
  const int e = (int)((__double_as_longlong(v) >> 52) & 2047);  // v in [2^(e - 1023), 2^(e - 1022))
  return e == 0 || e == 2047 ? 0 : 15 - (e - 1022);
}
// 2^e.  Past the ends of float32 the nearest power in it: a product that needs a smaller one has no share in a sum beside a term below 2^15.
__device__ __forceinline__ float ns_pow2(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }

// squares: |G|_F^2.  Bounds on the singular values of X_t, from |X_0| <= |X_0|_F on, choose the powers of two.
__device__ __forceinline__ void ns_scales(double squares, double eps, const NsCoef& cf, int steps, NsScales& z) {
  const double norm = sqrt(squares);
  const bool fine = norm < 1e300;
  const double inv = fine ? (norm + eps > 0.0 ? 1.0 / (norm + eps) : 0.0) : __longlong_as_double(0x7ff8000000000000ll);
  double u = fine ? norm * inv * (1.0 + 1e-3) : 1.0;
  int ex = ns_exponent(u);
  z.first = ldexp(inv, ex);
  for (int t = 0; t < steps; ++t) {
    const NsStep& s = cf.s[t];
    const int ea = ns_exponent(u * u), eb = ns_exponent(ns_peak_b(s, u));
    u = ns_peak_x(s, u) * (1.0 + 1e-3);
    const int en = ns_exponent(u);
    NsFactors& f = z.f[t];
    f.gram = ns_pow2(ea - 2 * ex);
    f.lin = (float)s.b * ns_pow2(eb - ea);
    f.quad = (float)s.c * ns_pow2(eb - 2 * ea);
    f.keep = (float)s.a * ns_pow2(en - ex);
    f.add = ns_pow2(en - eb - ex);
    ex = en;
  }
  z.last = -ex;
}

__global__ __launch_bounds__(64) void k_ns_scales(const double* parts, int count, double eps, NsCoef cf, int steps, NsScales* out) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 64) s += parts[(size_t)blockIdx.x * NS_PARTS + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (threadIdx.x == 0) ns_scales(s, eps, cf, steps, out[blockIdx.x]);
}

__device__ __forceinline__ void split(float v, _Float16* hi, _Float16* lo) {
  *hi = (_Float16)v;
  *lo = (_Float16)(v - (float)*hi);
}

// G -> X_0 (p rows) and its transpose (q rows), zero-padded.  One 64 x 64 tile a workgroup.
template <class T>
__global__ __launch_bounds__(256) void k_ns_pack(NsMatrix w, const NsScales* scales, char* x, char* xt, size_t batch_bytes) {
  __shared__ float tile[64][65];
  const T* g = (const T*)w.g + blockIdx.z * w.batch_stride;
  x += blockIdx.z * batch_bytes;
  xt += blockIdx.z * batch_bytes;
  const NsScales& z = scales[blockIdx.z];
  const double f = z.first;
  const long p0 = (long)blockIdx.y * 64, q0 = (long)blockIdx.x * 64;
  const bool along_q = w.col_stride <= w.row_stride;
  const int l = threadIdx.x & 63, r = threadIdx.x >> 6;
  for (int o = r; o < 64; o += 4) {
    const int pi = along_q ? o : l, qi = along_q ? l : o;
    float v = 0.0f;
    if (p0 + pi < w.p && q0 + qi < w.q) v = (float)((double)to_f32(g[(p0 + pi) * w.row_stride + (q0 + qi) * w.col_stride]) * f);
    tile[pi][qi] = v;
  }
  __syncthreads();
  const size_t ldx = pair_ld(w.q), ldt = pair_ld(w.p);
  const int row = threadIdx.x >> 2, part = (threadIdx.x & 3) * 16;
  for (int turn = 0; turn < 2; ++turn) {
    char* base = turn ? xt + pair_at(q0 + row, p0 + part, ldt) : x + pair_at(p0 + row, q0 + part, ldx);
    if (turn ? q0 + row >= w.q : p0 + row >= w.p) continue;
    f16x8 hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      _Float16 h, o;
      split(turn ? tile[part + e][row] : tile[row][part + e], &h, &o);
      hi[e >> 3][e & 7] = h;
      lo[e >> 3][e & 7] = o;
    }
    *(f16x8*)base = hi[0];
    *(f16x8*)(base + 16) = hi[1];
    *(f16x8*)(base + 64) = lo[0];
    *(f16x8*)(base + 80) = lo[1];
  }
}

enum NsKind { NS_GRAM, NS_POLY, NS_STEP, NS_LAST };

struct NsArgs {
  const char *P, *Q;      // operands of the product (pairs)
  const char* E;          // the matrix the epilogue adds, natural orientation (POLY: A, STEP / LAST: X)
  char *D, *DT;           // result and its transpose (pairs); symmetric products write both halves of D
  void* out;              // LAST: the caller's matrix
  const NsScales* scales;
  size_t batch_bytes;     // from a matrix of the batch to the next, workspace
  size_t out_stride;      // elements, out
  int I, J, K;
  int ti, tj, strip;
  int t;                  // step
  int transposed;         // LAST: out is stored q x p
};

__device__ __forceinline__ void store_pairs(char* at, const float (&v)[8]) {  // eight neighbours of a row of pairs
  f16x8 h, o;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    _Float16 hi, lo;
    split(v[e], &hi, &lo);
    h[e] = hi;
    o[e] = lo;
  }
  *(f16x8*)at = h;
  *(f16x8*)(at + 64) = o;
}

template <int KIND, class T, class TL, int MODE, int BI, int BJ>
__global__ __launch_bounds__(TL::THREADS) void k_ns_product(NsArgs g) {
  extern __shared__ char lds[];
  constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
  int bi, bj;
  if (SYM) {  // tiles bj <= bi, row by row
    const int t = die_order(blockIdx.x, g.ti * (g.ti + 1) / 2);
    bi = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
    while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
    while (bi * (bi + 1) / 2 > t) --bi;
    bj = t - bi * (bi + 1) / 2;
  } else {
    strip_order(die_order(blockIdx.x, g.ti * g.tj), g.ti, g.tj, g.strip, &bi, &bj);
  }
  const int i0 = bi * BI, j0 = bj * BJ;
  const size_t off = blockIdx.z * g.batch_bytes;
  const size_t ldk = pair_ld(g.K), ldi = pair_ld(g.I), ldj = pair_ld(g.J);
  TL t;
  const int per = MODE == MODE_F16 ? 64 : 32;
  t.run(Operand{g.P + off, (unsigned)ldk, g.I}, i0, Operand{g.Q + off, (unsigned)ldk, g.J}, j0, 0, (g.K + per - 1) / per, 128, lds);
  const NsScales& z = g.scales[blockIdx.z];
  const NsFactors f = z.f[g.t];
  const int last = z.last;
  const char* E = g.E + off;
  char* D = g.D + off;
  char* DT = SYM ? D : g.DT + off;
  T* out = (T*)g.out + blockIdx.z * g.out_stride;
  const bool natural = KIND != NS_LAST || !g.transposed, turned = KIND == NS_LAST ? g.transposed != 0 : SYM ? bi != bj : true;
  // Chunks of the tile through LDS: the result in the product's own orientation (rows j, eight neighbours i a thread), then, from the values left
  // there, its transpose (rows i, eight neighbours j).
  constexpr int ACROSS = BI / 8, ROWS = TL::THREADS / ACROSS;
  const int iw = threadIdx.x % ACROSS * 8, i = i0 + iw;
  constexpr int DOWN = TL::CHUNK / 8;
  const int iv = threadIdx.x / DOWN, rv = threadIdx.x % DOWN * 8;
#pragma unroll
  for (int c = 0; c < TL::CHUNKS; ++c) {
    __syncthreads();
    t.spill(c, lds);
    __syncthreads();
    for (int r = threadIdx.x / ACROSS; r < TL::CHUNK; r += ROWS) {
      const int j = j0 + TL::column(c, r);
      float v[8];
      chunk_sums<TL>(lds, r, iw, v);
      f16x8 eh = {}, el = {};
      const bool there = j < g.J && (size_t)i * 4 < ldi;  // (rows are padded: whole groups of eight, zeros behind the end)
      if (KIND != NS_GRAM && there) {
        const char* at = E + pair_at(j, i, ldi);
        eh = *(const f16x8*)at;
        el = *(const f16x8*)(at + 64);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = (float)eh[e] + (float)el[e];
        float w = v[e];
        if (KIND == NS_GRAM) w = f.gram * w;
        if (KIND == NS_POLY) w = f.lin * x + f.quad * w;
        if (KIND == NS_STEP) w = f.keep * x + f.add * w;
        if (KIND == NS_LAST) w = ldexpf(f.keep * x + f.add * w, last);
        v[e] = i + e < g.I && j < g.J ? w : 0.0f;
      }
      if (turned)
#pragma unroll
        for (int e = 0; e < 8; ++e) ((float*)lds)[r * TL::PITCH + iw + e] = v[e];
      if (KIND != NS_LAST) {
        if (there) store_pairs(D + pair_at(j, i, ldi), v);
      } else if (natural && j < g.J && i < g.I) {
        store8(out + (size_t)j * g.I + i, v, g.I - i, i + 8 <= g.I && g.I % (16 / (int)sizeof(T)) == 0);
      }
    }
    if (turned) {
      __syncthreads();
      for (int ii = iv; ii < BI; ii += TL::THREADS / DOWN) {
        const int irow = i0 + ii, j = j0 + TL::column(c, rv);
        if (irow >= g.I) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ((const float*)lds)[(rv + e) * TL::PITCH + ii];
        if (KIND != NS_LAST) {
          if ((size_t)j * 4 < ldj) store_pairs(DT + pair_at(irow, j, ldj), v);
        } else if (j < g.J) {
          store8(out + (size_t)irow * g.J + j, v, g.J - j, j + 8 <= g.J && g.J % (16 / (int)sizeof(T)) == 0);
        }
      }
    }
  }
}

// ---- small matrices ---------------------------------------------------------------------------------------------------------------------------
// One workgroup does all steps of a matrix of up to 32 PB x 256 CB (padded to blocks of 32).  X stays in registers in float32, in the places the matrix
// instruction leaves its results in: lane l has column l % 32 of a block, registers r the rows 8 (r / 4) + 4 (l / 32) + r % 4.  Wave w has the column
// blocks w, w + 8, ...
//   A = X X^T contracts over columns, which lie across lanes: X goes through LDS once a step, as rows of fp16 (hi and lo planes).
//   B X contracts over rows, which lie along registers: registers 8 s .. 8 s + 7 of a block ARE a fragment of the 32 x 32 x 16 instruction if k runs in the
//   order 16 s + {4 h, 4 h + 1, .., 4 h + 3, 8 + 4 h, ..} for lane half h - so B is laid out in LDS with its columns in that order and X is never moved.
// Rows of LDS planes are 16 bytes longer than their numbers: eight neighbouring rows start in different banks.
// A step is a chain of three short products; what bounds it is latency (barriers, LDS round trips), not a rate.
// What a general path costs instead is three launches a step.
template <int PB, int CB>
struct NsSmall {
  static constexpr int P = 32 * PB, Q = 256 * CB;
  static constexpr int BLOCKS = PB * PB;
  static constexpr int OWN = (BLOCKS + 7) / 8;              // blocks of A a wave has
  static constexpr int KS = BLOCKS >= 8 ? 1 : PB == 2 ? 2 : 8;  // waves that share a block's columns
  static constexpr int PITCH_A = P * 2 + 16;
  // LDS for the columns that are there
  __host__ __device__ static int pitch_x(int q) { return (q + 31) / 32 * 64 + 16; }
  __host__ __device__ static int lds(int q) {
    const int x = 2 * P * pitch_x(q), a = 2 * P * PITCH_A, parts = KS > 1 ? 8 * 4096 : 0;
    const int m = x > a ? x : a;
    return m > parts ? m : parts;
  }
};

template <class T, int PB, int CB>
__global__ __launch_bounds__(512) void k_ns_small(NsMatrix m, NsCoef cf, int steps, int exact, double eps, T* out, int tall) {
  using S = NsSmall<PB, CB>;
  extern __shared__ char lds[];
  __shared__ NsScales z;
  __shared__ double part[8];
  const int l = (int)(threadIdx.x & 63), w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int h = l >> 5, c32 = l & 31;
  const int p = (int)m.p, q = (int)m.q;
  const int cols = (q + 31) / 32;  // column blocks
  const T* g = (const T*)m.g + blockIdx.x * m.batch_stride;
  float x[CB][PB][16];
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int j = (w + 8 * c) * 32 + c32;
    // (32-bit offsets within the matrix: the host sees to it)
    const unsigned at = (unsigned)(4 * h * (int)m.row_stride + j * (int)m.col_stride) * (unsigned)sizeof(T);
#pragma unroll
    for (int a = 0; a < PB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int iu = 32 * a + 8 * (r >> 2) + (r & 3);
        const char* row = (const char*)(g + iu * m.row_stride);
        x[c][a][r] = (iu + 4 * h < p && j < q) ? to_f32(*(const T*)(row + at)) : 0.0f;
      }
  }
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int a = 0; a < PB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += (double)x[c][a][r] * (double)x[c][a][r];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (l == 0) part[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < 8; ++i) s += part[i];
    ns_scales(s, eps, cf, steps, z);
  }
  __syncthreads();
  {
    const double f = z.first;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int a = 0; a < PB; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[c][a][r] = (float)((double)x[c][a][r] * f);
  }
  const int pitch = S::pitch_x(q);
  for (int t = 0; t < steps; ++t) {
    const bool pairs = t >= steps - exact;
    const NsFactors f = z.f[t];
    // X to LDS, hi plane then lo plane
#pragma unroll
    for (int c = 0; c < CB; ++c)
      if (w + 8 * c < cols) {
#pragma unroll
        for (int a = 0; a < PB; ++a)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            char* at = lds + (32 * a + 8 * (r >> 2) + 4 * h + (r & 3)) * pitch + ((w + 8 * c) * 32 + c32) * 2;
            _Float16 hi, lo;
            split(x[c][a][r], &hi, &lo);
            *(_Float16*)at = hi;
            if (pairs) *(_Float16*)(at + S::P * pitch) = lo;
          }
      }
    __syncthreads();
    // A: block (bi, bj) of wave w % blocks, KS waves share its columns
    f32x16 acc[S::OWN];
#pragma unroll
    for (int o = 0; o < S::OWN; ++o) {
      acc[o] = f32x16{};
      const int blk = S::KS > 1 ? w % S::BLOCKS : w + 8 * o;
      if (blk < S::BLOCKS) {
        const char* pi = lds + (blk / PB * 32 + c32) * pitch + h * 16;
        const char* pj = lds + (blk % PB * 32 + c32) * pitch + h * 16;
        for (int k = S::KS > 1 ? w / S::BLOCKS : 0; k < 2 * cols; k += S::KS) {
          const f16x8 ih = *(const f16x8*)(pi + k * 32), jh = *(const f16x8*)(pj + k * 32);
          acc[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jh, acc[o], 0, 0, 0);
          if (pairs) {
            const f16x8 il = *(const f16x8*)(pi + S::P * pitch + k * 32), jl = *(const f16x8*)(pj + S::P * pitch + k * 32);
            acc[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(il, jh, acc[o], 0, 0, 0);
            acc[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jl, acc[o], 0, 0, 0);
          }
        }
      }
    }
    __syncthreads();
    if constexpr (S::KS > 1) {
      float* mine = (float*)lds + w * 1024 + l;
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[r * 64] = acc[0][r];
      __syncthreads();
      if (w < S::BLOCKS) {
#pragma unroll
        for (int o = 1; o < S::KS; ++o)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[0][r] += mine[o * S::BLOCKS * 1024 + r * 64];
      }
      __syncthreads();
    }
    // A as pairs; it is symmetric, so the lane's column is a row and its four neighbouring rows are four neighbours in it
#pragma unroll
    for (int o = 0; o < S::OWN; ++o) {
      const int blk = w + 8 * o;
      if (blk < S::BLOCKS) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[o][r] *= f.gram;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          char* at = lds + (blk % PB * 32 + c32) * S::PITCH_A + (blk / PB * 32 + 2 * r + 4 * h) * 2;
          f16x4 hi, lo;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16 u, v;
            split(acc[o][r + e], &u, &v);
            hi[e] = u;
            lo[e] = v;
          }
          *(f16x4*)at = hi;
          if (pairs) *(f16x4*)(at + S::P * S::PITCH_A) = lo;
        }
      }
    }
    __syncthreads();
    // B = b A + c A A
    f32x16 poly[S::OWN];
#pragma unroll
    for (int o = 0; o < S::OWN; ++o) {
      poly[o] = f32x16{};
      const int blk = w + 8 * o;
      if (blk < S::BLOCKS) {
        const char* pi = lds + (blk / PB * 32 + c32) * S::PITCH_A + h * 16;
        const char* pj = lds + (blk % PB * 32 + c32) * S::PITCH_A + h * 16;
#pragma unroll 2
        for (int k = 0; k < 2 * PB; ++k) {
          const f16x8 ih = *(const f16x8*)(pi + k * 32), jh = *(const f16x8*)(pj + k * 32);
          poly[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jh, poly[o], 0, 0, 0);
          if (pairs) {
            const f16x8 il = *(const f16x8*)(pi + S::P * S::PITCH_A + k * 32), jl = *(const f16x8*)(pj + S::P * S::PITCH_A + k * 32);
            poly[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(il, jh, poly[o], 0, 0, 0);
            poly[o] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih, jl, poly[o], 0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) poly[o][r] = f.lin * acc[o][r] + f.quad * poly[o][r];
      }
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < S::OWN; ++o) {
      const int blk = w + 8 * o;
      if (blk < S::BLOCKS) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          // row (column of the block) c32, k = 8 (r / 4) + 4 h + e, at the place 16 (r / 8) + 8 h + 4 (r / 4 % 2) + e
          char* at = lds + (blk % PB * 32 + c32) * S::PITCH_A + (blk / PB * 32 + 16 * (r >> 3) + 8 * h + 4 * ((r >> 2) & 1)) * 2;
          f16x4 hi, lo;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16 u, v;
            split(poly[o][r + e], &u, &v);
            hi[e] = u;
            lo[e] = v;
          }
          *(f16x4*)at = hi;
          if (pairs) *(f16x4*)(at + S::P * S::PITCH_A) = lo;
        }
      }
    }
    __syncthreads();
    // X <- a X + B X
#pragma unroll
    for (int c = 0; c < CB; ++c)
      if (w + 8 * c < cols) {
        f16x8 xh[2 * PB], xl[2 * PB];
#pragma unroll
        for (int k = 0; k < 2 * PB; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            _Float16 u, v;
            split(x[c][k >> 1][8 * (k & 1) + e], &u, &v);
            xh[k][e] = u;
            xl[k][e] = v;
          }
#pragma unroll
        for (int a = 0; a < PB; ++a) {
          const char* pi = lds + (32 * a + c32) * S::PITCH_A + h * 16;
          f32x16 s = f32x16{};
#pragma unroll
          for (int k = 0; k < 2 * PB; ++k) {
            const f16x8 bh = *(const f16x8*)(pi + k * 32);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh, xh[k], s, 0, 0, 0);
            if (pairs) {
              const f16x8 bl = *(const f16x8*)(pi + S::P * S::PITCH_A + k * 32);
              s = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl, xh[k], s, 0, 0, 0);
              s = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh, xl[k], s, 0, 0, 0);
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) x[c][a][r] = f.keep * x[c][a][r] + f.add * s[r];
          __builtin_amdgcn_sched_barrier(0);  // (one row block's fragments of B at a time: registers)
        }
      }
    __syncthreads();
  }
  T* y = out + blockIdx.x * (size_t)p * q;
  const int last = z.last, rs = tall ? 1 : q, cs = tall ? p : 1;
#pragma unroll
  for (int c = 0; c < CB; ++c) {
    const int j = (w + 8 * c) * 32 + c32;
    const unsigned at = (unsigned)(4 * h * rs + j * cs) * (unsigned)sizeof(T);
#pragma unroll
    for (int a = 0; a < PB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int iu = 32 * a + 8 * (r >> 2) + (r & 3);
        char* row = (char*)(y + iu * rs);
        if (iu + 4 * h < p && j < q) *(T*)(row + at) = (T)ldexpf(x[c][a][r], last);
      }
  }
}

}  // namespace lb
