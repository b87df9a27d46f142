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

// Matrices are held times a power of two.  What a step's sums w are multiplied with to become the next held matrix:
struct NsFactors {
  float gram;               // A = X X^T: gram w
  float unit, lin, quad;    // B = lin A + quad w;  P = unit 1 + lin A + quad w in a chain (below)
  float keep, add;          // next X: keep X + add w
  float half, next, chain;  // a chain: R = P A: half w;  A <- P R: next w;  Q <- P Q: chain w
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
  double grow;           // max |a + b z + c z^2| for the singular values the step can meet when |X_0| <= 1
};
struct NsCoef {
  NsStep s[NS_MAX_STEPS];
  NsFactors f[NS_MAX_STEPS];  // for matrices whose norm is not small beside eps: |X_0|_F near 1
  int first, last;            // their powers: X_0 is held times 2^first, the result times 2^-last
  unsigned ends;              // bit t: a chain of steps ends with step t
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

// u: bound on the singular values that enter the step
inline void ns_step(double a, double b, double c, double u, NsStep* o) {
  *o = NsStep{a, b, c, {INFINITY, INFINITY}, {0.0, 0.0}, INFINITY, 0.0, 0.0};
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
  const double z = u * u;
  o->grow = std::max(std::fabs(a), std::fabs(a + z * (b + c * z)));
  if (o->zs < z) o->grow = std::max(o->grow, std::fabs(a + o->zs * (b + c * o->zs)));
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
__host__ __device__ inline int ns_exponent(double v) {
  const int e = (int)((__builtin_bit_cast(long long, v) >> 52) & 2047);  // v in [2^(e - 1023), 2^(e - 1022))
  return e == 0 || e == 2047 ? 0 : 15 - (e - 1022);
}
// 2^e.  Past the ends of float32 the nearest power in it: a product that needs a smaller one has no share in a sum beside a term below 2^15.
__host__ __device__ inline float ns_pow2(int e) { return __builtin_bit_cast(float, ((e < -126 ? -126 : e > 127 ? 127 : e) + 127) << 23); }

// The factors of all steps from a bound u on the singular values of X_0 = 2^-first held X_0; returns -last of NsScales.
constexpr int NS_UNIT = 14;  // a chain starts with Q = 1 held as 2^14
__host__ __device__ inline int ns_factors(double u, const NsStep* steps, unsigned ends, int count, NsFactors* out) {
  double chain = 1.0;
  int ex = ns_exponent(u), eq = NS_UNIT;
  for (int t = 0; t < count; ++t) {
    const NsStep& s = steps[t];
    const bool begin = t == 0 || (ends >> (t - 1) & 1), end = ends >> t & 1, alone = begin && end;
    if (begin) {
      eq = NS_UNIT;
      chain = 1.0;
    }
    const double un = ns_peak_x(s, u) * (1.0 + 1e-3);
    chain *= s.grow * (1.0 + 1e-3);
    const int ea = ns_exponent(u * u), en = ns_exponent(un), ean = ns_exponent(un * un);
    const int eb = ns_exponent(alone ? ns_peak_b(s, u) : s.grow), er = ns_exponent(s.grow * u * u), eqn = ns_exponent(chain);
    NsFactors f;
    f.gram = ns_pow2(ea - 2 * ex);
    f.unit = (float)s.a * ns_pow2(eb);
    f.lin = (float)s.b * ns_pow2(eb - ea);
    f.quad = (float)s.c * ns_pow2(eb - 2 * ea);
    f.half = ns_pow2(er - eb - ea);
    f.next = ns_pow2(ean - eb - er);
    f.chain = ns_pow2(eqn - eb - eq);
    f.keep = alone ? (float)s.a * ns_pow2(en - ex) : 0.0f;
    f.add = ns_pow2(en - ex - (alone ? eb : eqn));
    out[t] = f;
    eq = eqn;
    if (end) ex = en;
    u = un;
  }
  return ex;
}
// squares: |G|_F^2.  Bounds on the singular values of X_t, from |X_0| <= |X_0|_F on, choose the powers of two; where |X_0|_F is near 1 (the norm is
// large beside eps) they are known before (ns_fetch has them in place already), else they are worked out here.
__device__ __forceinline__ void ns_scales(double squares, double eps, const NsCoef& cf, int steps, NsScales& z) {
  const double norm = sqrt(squares);
  const bool fine = norm < 1e300;
  const double inv = fine ? (norm + eps > 0.0 ? 1.0 / (norm + eps) : 0.0) : __longlong_as_double(0x7ff8000000000000ll);
  const double u = norm * inv;
  int first = cf.first, last = cf.last;
  if (u < 0.25) {
    const double v = u * (1.0 + 1e-3);
    first = ns_exponent(v);
    last = -ns_factors(v, cf.s, cf.ends, steps, z.f);
  }
  z.first = ldexp(inv, first);
  z.last = last;
}

// The steps' tables from the kernel's arguments, all at once: read one by one they are a chain of misses.  A barrier has to follow.
__device__ __forceinline__ void ns_fetch(const NsCoef& cf, int steps, NsCoef* to, NsFactors* f) {
  for (int i = threadIdx.x; i < steps * (int)(sizeof(NsStep) / 4); i += blockDim.x) ((int*)to->s)[i] = ((const int*)cf.s)[i];
  for (int i = threadIdx.x; i < steps * (int)(sizeof(NsFactors) / 4); i += blockDim.x) ((int*)f)[i] = ((const int*)cf.f)[i];
  if (threadIdx.x == 0) {
    to->ends = cf.ends;
    to->first = cf.first;
    to->last = cf.last;
  }
}
__global__ __launch_bounds__(64) void k_ns_scales(const double* parts, int count, double eps, NsCoef cf, int steps, NsScales* out) {
  __shared__ NsCoef mine;
  ns_fetch(cf, steps, &mine, out[blockIdx.x].f);
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 64) s += parts[(size_t)blockIdx.x * NS_PARTS + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  __syncthreads();
  if (threadIdx.x == 0) ns_scales(s, eps, mine, steps, out[blockIdx.x]);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split(float v, float u, f16x2* hi, f16x2* lo) {  // (two at a time: one conversion instruction)
  *hi = __builtin_convertvector(f32x2{v, u}, f16x2);
  *lo = __builtin_convertvector(f32x2{v - (float)(*hi)[0], u - (float)(*hi)[1]}, f16x2);
}
template <class V>
__device__ __forceinline__ void split8(const V& v, int at, f16x8* hi, f16x8* lo) {  // v[at .. at + 7]
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f16x2 h, o;
    split(v[at + e], v[at + e + 1], &h, &o);
    (*hi)[e] = h[0];
    (*hi)[e + 1] = h[1];
    (*lo)[e] = o[0];
    (*lo)[e + 1] = o[1];
  }
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
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = turn ? tile[part + e][row] : tile[row][part + e];
    split8(v, 0, &hi[0], &lo[0]);
    split8(v, 8, &hi[1], &lo[1]);
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
  split8(v, 0, &h, &o);
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

// ---- up to 128 rows -----------------------------------------------------------------------------------------------------------------------------
// Everything p x p fits one workgroup; X is dealt out to the waves by columns and stays in registers in float32, in the places the matrix instruction
// leaves its results in: a wave has column blocks of 32, lane l the column l % 32, registers r of row block a the rows 32 a + 8 (r / 4) + 4 (l / 32) + r % 4.
//   S X for symmetric S contracts over rows, which lie along registers: registers 8 s .. 8 s + 7 of a block ARE a fragment of the 32 x 32 x 16 instruction
//   if k runs in the order 16 s + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} for lane half h.  So S lies in LDS with its columns in that order (an "image",
//   hi and lo planes) and X never moves (ns_times).
//   A = X X^T contracts over columns, which lie across lanes: X goes through LDS as rows (ns_gram).
// Rows of LDS planes are 16 bytes longer than their numbers: eight neighbouring rows start in different banks.
//
// Chains: with P_t = a + b A_t + c A_t A_t the iterates are X_t+1 = P_t X_t and A_t+1 = P_t A_t P_t, so steps t .. t' can be done on p x p matrices
// alone, Q <- P Q, and X is multiplied once, by Q.  What it costs is accuracy: A's roundings are relative to its LARGEST eigenvalue, and Q amplifies
// what they do to small ones by the square of the polynomials' slope.  Measured against 64 bits (five standard steps, Gaussian, 1 / k and exponential
// spectra, low rank + noise; 64 .. 512 rows): relative error of the result up to 4e-4 in one chain, 2e-5 in chains of 3 + 2, 9e-6 without (as
// float32 products: 9e-6).  So bfloat16 results (rounding 1.7e-3) take chains of growth up to 500, float16 (2e-4) up to 45, float32 none.
// Bound by latency for one small matrix (a chain's step is three dependent products and two barriers), by the matrix cores for batches.
template <int PB, int CB = 1>
struct NsRows {
  static constexpr int P = 32 * PB;
  static constexpr int PITCH = P * 2 + 16, IMAGE = 2 * P * PITCH;
  static constexpr int KS = 8 / PB < 4 ? 8 / PB : 4;          // most waves that share a column block of A
  // Adding shares up costs about as much as 2 .. 4 of the K steps it saves: measured, from these lengths on it pays.
  __device__ static int shares(int cols) { return min(KS, max(1, cols / (PB <= 2 ? 4 : PB == 3 ? 3 : 2))); }
  static constexpr int PARTS = (KS - 1) * PB * PB * 4096;     // what they add up through LDS
  static constexpr int PITCH_X = CB * 512 + 16, X = 2 * P * PITCH_X;  // rows of X (a constant pitch: their addresses are then offsets of one)
  static constexpr int LDS = X > 2 * IMAGE ? (X > PARTS ? X : PARTS) : (2 * IMAGE > PARTS ? 2 * IMAGE : PARTS);
};
template <int PB>
using NsCols = float[PB][16];  // a column block of a p-row matrix

// y = S x, S an image.  One fragment of x at a time is split and met by all row blocks: PB (for one block: three) independent accumulators.
template <int PB>
__device__ __forceinline__ void ns_times(const char* image, const NsCols<PB>& x, NsCols<PB>& y) {
  using S = NsRows<PB>;
  const int l = lane_id();
  const char* at = image + (l & 31) * S::PITCH + (l >> 5) * 16;
  constexpr int APART = PB == 1 ? 3 : 1;
  f32x16 acc[PB * APART];
#pragma unroll
  for (int a = 0; a < PB * APART; ++a) acc[a] = f32x16{};
#pragma unroll
  for (int k = 0; k < 2 * PB; ++k) {
    f16x8 xh, xl, bh[PB], bl[PB];
#pragma unroll
    for (int a = 0; a < PB; ++a) {
      bh[a] = *(const f16x8*)(at + a * 32 * S::PITCH + k * 32);
      bl[a] = *(const f16x8*)(at + (a * 32 + S::P) * S::PITCH + k * 32);
    }
    split8(x[k >> 1], 8 * (k & 1), &xh, &xl);
#pragma unroll
    for (int a = 0; a < PB; ++a) acc[a * APART] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[a], xh, acc[a * APART], 0, 0, 0);
#pragma unroll
    for (int a = 0; a < PB; ++a) acc[a * APART + APART / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl[a], xh, acc[a * APART + APART / 2], 0, 0, 0);
#pragma unroll
    for (int a = 0; a < PB; ++a) acc[a * APART + APART - 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[a], xl, acc[a * APART + APART - 1], 0, 0, 0);
    if (PB > 1) {  // one step's fragments at a time: all of them would not fit the registers
#pragma unroll
      for (int a = 0; a < PB; ++a) asm volatile("" : "+v"(acc[a]));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int a = 0; a < PB; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) y[a][r] = APART == 1 ? acc[a][r] : (acc[a * APART + 1][r] + acc[a * APART + APART - 1][r]) + acc[a * APART][r];
}
// A column block to rows of LDS (hi plane, lo plane `plane` bytes on): the lane's column is at byte `at`, rows are `pitch` apart.  Neighbouring lanes swap
// halves of two rows, so that each writes two neighbours of one.
template <int PB>
__device__ __forceinline__ void ns_scatter(char* lds, int pitch, int plane, int at, const NsCols<PB>& x) {
  const int l = lane_id(), h = l >> 5;
  const bool odd = l & 1;
  char* base = lds + (4 * h + odd) * pitch + at - 2 * odd;
  const unsigned pick = odd ? 0x03020706u : 0x05040100u;  // bytes of (mine, the neighbour's): even lanes the lower halves, odd lanes the upper ones
#pragma unroll
  for (int a = 0; a < PB; ++a)
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      f16x2 hi, lo;
      split(x[a][r], x[a][r + 1], &hi, &lo);
      char* to = base + (32 * a + 8 * (r >> 2) + (r & 3)) * pitch;
      const unsigned mh = __builtin_bit_cast(unsigned, hi), ml = __builtin_bit_cast(unsigned, lo);
      const unsigned nh = (unsigned)__builtin_amdgcn_mov_dpp((int)mh, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2
      const unsigned nl = (unsigned)__builtin_amdgcn_mov_dpp((int)ml, 0xb1, 0xf, 0xf, true);
      *(unsigned*)to = __builtin_amdgcn_perm(nh, mh, pick);
      *(unsigned*)(to + plane) = __builtin_amdgcn_perm(nl, ml, pick);
      if (r % 8 == 6) __builtin_amdgcn_sched_barrier(0);
    }
}
// Column block b of a p x p matrix into an image.  (Row i of the image is row i: the matrices of a chain are symmetric but for their roundings, and an
// image of the transpose would make those grow - the products of a chain commute only as long as all are polynomials of the SAME A.)
template <int PB>
__device__ __forceinline__ void ns_put(char* image, int b, const NsCols<PB>& x) {
  using S = NsRows<PB>;
  const int c = lane_id() & 31;
  ns_scatter<PB>(image, S::PITCH, S::P * S::PITCH, 64 * b + 32 * (c >> 4) + 16 * ((c >> 2) & 1) + 8 * ((c >> 3) & 1) + 2 * (c & 3), x);
}
// Column block number c of X to rows
template <int PB, int CB>
__device__ __forceinline__ void ns_rows(char* lds, int c, const NsCols<PB>& x) {
  using S = NsRows<PB, CB>;
  ns_scatter<PB>(lds, S::PITCH_X, S::P * S::PITCH_X, 64 * c + 2 * (lane_id() & 31), x);
}
// Column block w % PB of X X^T from the rows in LDS, wave w's share w / PB of the K range (added up by ns_gather)
template <int PB, int CB>
__device__ __forceinline__ void ns_gram(const char* lds, int cols, NsCols<PB>& m) {
  using S = NsRows<PB, CB>;
  constexpr int pitch = S::PITCH_X;
  const int w = wave_id(), l = lane_id();
  f32x16 acc[PB];
#pragma unroll
  for (int a = 0; a < PB; ++a) acc[a] = f32x16{};
  const int shares = S::shares(cols);
  if (w < PB * shares) {
    const char* at = lds + (l & 31) * pitch + (l >> 5) * 16;
    const int j = w % PB * 32;
    for (int k = w / PB; k < 2 * cols; k += shares) {
      const f16x8 jh = *(const f16x8*)(at + j * pitch + k * 32), jl = *(const f16x8*)(at + (j + S::P) * pitch + k * 32);
      f16x8 ih[PB], il[PB];
#pragma unroll
      for (int a = 0; a < PB; ++a) {
        ih[a] = *(const f16x8*)(at + 32 * a * pitch + k * 32);
        il[a] = *(const f16x8*)(at + (32 * a + S::P) * pitch + k * 32);
      }
#pragma unroll
      for (int a = 0; a < PB; ++a) acc[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih[a], jh, acc[a], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < PB; ++a) acc[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(il[a], jh, acc[a], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < PB; ++a) acc[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ih[a], jl, acc[a], 0, 0, 0);
    }
  }
#pragma unroll
  for (int a = 0; a < PB; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) m[a][r] = acc[a][r];
}
// Adds the shares up: afterwards waves 0 .. PB - 1 have the column blocks.  The first barrier is for the rows, which have been read.
template <int PB>
__device__ __forceinline__ void ns_gather(char* lds, int cols, NsCols<PB>& m) {
  using S = NsRows<PB>;
  const int w = wave_id(), l = lane_id();
  const int shares = S::shares(cols);
  __syncthreads();
  if (shares == 1) return;
  if (w >= PB && w < PB * shares) {
    float* mine = (float*)lds + (w - PB) * PB * 1024 + l;
#pragma unroll
    for (int a = 0; a < PB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(a * 16 + r) * 64] = m[a][r];
  }
  __syncthreads();
  if (w < PB) {
    for (int o = 1; o < shares; ++o) {
      const float* its = (const float*)lds + (o * PB + w - PB) * PB * 1024 + l;
#pragma unroll
      for (int a = 0; a < PB; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[a][r] += its[(a * 16 + r) * 64];
    }
  }
  __syncthreads();
}
// From A (waves 0 .. PB - 1: its column blocks, as summed) the image that X is multiplied with: B of a single step, or Q of the chain t .. end.
// Images at lds and lds + IMAGE; returns the one that holds it; a barrier has passed.
template <int PB>
__device__ __forceinline__ char* ns_chain(char* lds, NsCols<PB>& m, const NsScales& z, int t, int end) {
  using S = NsRows<PB>;
  const int w = wave_id(), l = lane_id();
  const bool a_wave = w < PB, q_wave = w >= 4 && w < 4 + PB;
  char *ia = lds, *ip = lds + S::IMAGE;
  const float gram = z.f[t].gram;
#pragma unroll
  for (int a = 0; a < PB; ++a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) m[a][r] = q_wave ? 0.0f : gram * m[a][r];
    if (a == w - 4)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + 4 * (l >> 5) + (r & 3) == (l & 31)) m[a][r] = (float)(1 << NS_UNIT);
  }
  const bool alone = t == end;
  for (;; ++t) {
    const NsFactors f = z.f[t];
    if (a_wave) ns_put<PB>(ia, w, m);
    __syncthreads();
    if (a_wave) {
      NsCols<PB> p;
      ns_times<PB>(ia, m, p);
#pragma unroll
      for (int a = 0; a < PB; ++a) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[a][r] = f.lin * m[a][r] + f.quad * p[a][r];
        if (!alone && a == w)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + 4 * (l >> 5) + (r & 3) == (l & 31)) p[a][r] += f.unit;
      }
      ns_put<PB>(ip, w, p);
    }
    __syncthreads();
    if (alone) return ip;
    const bool on = a_wave && t != end;
    if (on || q_wave) {  // R = P A, Q <- P Q
      NsCols<PB> y;
      ns_times<PB>(ip, m, y);
      const float by = a_wave ? f.half : f.chain;
#pragma unroll
      for (int a = 0; a < PB; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[a][r] = by * y[a][r];
    }
    if (t == end) break;
    if (on) {
      NsCols<PB> y;
      ns_times<PB>(ip, m, y);
#pragma unroll
      for (int a = 0; a < PB; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[a][r] = f.next * y[a][r];
    }
  }
  if (q_wave) ns_put<PB>(ia, w - 4, m);
  __syncthreads();
  return ia;
}
// Column block number c of G times f.  (32-bit offsets within the matrix: the host sees to it.)
template <class T, int PB>
__device__ __forceinline__ void ns_load(const T* g, const NsMatrix& m, long j0, int c, NsCols<PB>& x) {
  const int l = lane_id(), h = l >> 5;
  const long j = j0 + 32 * c + (l & 31);
  const char* col = (const char*)(g + (j0 + 32 * c) * m.col_stride);
  const unsigned rs = (unsigned)m.row_stride * (unsigned)sizeof(T);
  const int rows = j < m.q ? (int)m.p - 4 * h : 0;
  // rows past the end are read from the last one, columns past it from the first, and count as zeros: all loads are under way together
  const unsigned side = (j < m.q ? l & 31 : 0) * (unsigned)m.col_stride * (unsigned)sizeof(T);
  const unsigned end = ((unsigned)m.p - 1) * rs + side;
  unsigned at = 4 * h * rs + side;
  const char* from = m.q > j0 + 32 * c ? col : (const char*)g;
  T v[PB][16];
#pragma unroll
  for (int a = 0; a < PB; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      v[a][r] = *(const T*)(from + min(at, end));
      at += (r & 3) == 3 ? 5 * rs : rs;  // rows 0 1 2 3, 8 9 10 11, ..
    }
#pragma unroll
  for (int a = 0; a < PB; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[a][r] = 32 * a + 8 * (r >> 2) + (r & 3) < rows ? to_f32(v[a][r]) : 0.0f;
}
template <class T, int PB>
__device__ __forceinline__ void ns_store(T* out, const NsMatrix& m, long j0, int c, const NsCols<PB>& x, int last, bool tall) {
  const int l = lane_id(), h = l >> 5;
  const long j = j0 + 32 * c + (l & 31);
  const long rs = tall ? 1 : m.q, cs = tall ? m.p : 1;
  char* col = (char*)(out + (j0 + 32 * c) * cs);
  const unsigned step = (unsigned)rs * (unsigned)sizeof(T);
  int rows = j < m.q ? (int)m.p - 4 * h : 0;
  asm volatile("" : "+v"(rows));  // (compare again: the 16 PB masks of the load are not worth keeping in scalar registers until here)
  unsigned at = 4 * h * step + (l & 31) * (unsigned)cs * (unsigned)sizeof(T);
#pragma unroll
  for (int a = 0; a < PB; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (32 * a + 8 * (r >> 2) + (r & 3) < rows) *(T*)(col + at) = (T)ldexpf(x[a][r], last);
      at += (r & 3) == 3 ? 5 * step : step;
    }
}

// One workgroup does a whole matrix of up to 32 PB x 256 CB.
template <class T, int PB, int CB>
__global__ __launch_bounds__(512) void k_ns_small(NsMatrix m, NsCoef cf, int steps, double eps, T* out, int tall) {
  extern __shared__ char lds[];
  __shared__ NsScales z;
  __shared__ NsCoef mine;
  __shared__ double part[8];
  const int l = lane_id(), w = wave_id();
  ns_fetch(cf, steps, &mine, z.f);
  const int cols = (int)((m.q + 31) / 32);
  const T* g = (const T*)m.g + blockIdx.x * m.batch_stride;
  NsCols<PB> x[CB];
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < CB; ++c) ns_load<T, PB>(g, m, 0, w + 8 * c, x[c]);
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int a = 0; a < PB; ++a) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += (double)x[c][a][r] * (double)x[c][a][r];
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (l == 0) part[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < 8; ++i) s += part[i];
    ns_scales(s, eps, mine, steps, z);
  }
  __syncthreads();
  const double first = z.first;
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int a = 0; a < PB; ++a) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[c][a][r] = (float)((double)x[c][a][r] * first);
      __builtin_amdgcn_sched_barrier(0);
    }
  for (int t = 0; t < steps;) {
    int end = t;
    while (!(mine.ends >> end & 1)) ++end;
#pragma unroll
    for (int c = 0; c < CB; ++c)
      if (w + 8 * c < cols) ns_rows<PB, CB>(lds, w + 8 * c, x[c]);
    __syncthreads();
    NsCols<PB> a;
    ns_gram<PB, CB>(lds, cols, a);
    ns_gather<PB>(lds, cols, a);
    const char* image = ns_chain<PB>(lds, a, z, t, end);
    const float keep = z.f[end].keep, add = z.f[end].add;
#pragma unroll
    for (int c = 0; c < CB; ++c)
      if (w + 8 * c < cols) {
        NsCols<PB> y;
        ns_times<PB>(image, x[c], y);
#pragma unroll
        for (int b = 0; b < PB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[c][b][r] = keep * x[c][b][r] + add * y[b][r];
      }
    t = end + 1;
    if (t < steps) __syncthreads();
  }
  T* y = out + blockIdx.x * (size_t)(m.p * m.q);
#pragma unroll
  for (int c = 0; c < CB; ++c) ns_store<T, PB>(y, m, 0, w + 8 * c, x[c], z.last, tall);
}

}  // namespace lb
