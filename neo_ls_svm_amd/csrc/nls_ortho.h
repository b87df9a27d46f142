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
constexpr int NS_PARTS = 1024;  // partial sums of squares a matrix, at most

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

// A matrix of fp16 pairs: rows padded with zeros to 64 elements, 4 bytes an element; for every 32 elements the hi halves, then the lo halves.
__host__ __device__ inline size_t pair_ld(long k) { return (size_t)((k + 63) / 64 * 64) * 4; }
__device__ __forceinline__ size_t pair_at(size_t row, size_t k, size_t ld) { return row * ld + (k >> 5) * 128 + (k & 31) * 2; }
constexpr int PAIR_LO = 64;  // bytes from a hi half to its lo half

struct NsMatrix {
  const void* g;
  long p, q;                       // p <= q
  long row_stride, col_stride, batch_stride;  // in elements
};

// Sums of squares, a part a workgroup.  Sixteen bytes a thread and turn along the direction whose neighbours are neighbours in memory, from any element
// on; bound by memory (4096 x 4096 float32 was 103 us with one element a thread and 256 workgroups).
template <class T>
__global__ __launch_bounds__(256) void k_ns_norm(NsMatrix w, double* parts) {
  constexpr int N = 16 / (int)sizeof(T);
  typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  const T* g = (const T*)w.g + blockIdx.y * w.batch_stride;
  double s[2] = {0.0, 0.0};
  const bool along_q = w.col_stride <= w.row_stride;
  const long outer = along_q ? w.p : w.q, inner = along_q ? w.q : w.p;
  const long os = along_q ? w.row_stride : w.col_stride, is = along_q ? w.col_stride : w.row_stride;
  // 64 threads along a row, four rows at a time
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (long o = (long)blockIdx.x * 4 + y; o < outer; o += (long)gridDim.x * 4) {
    const T* row = g + o * os;
    long i = x * N;
    if (is == 1)
#pragma unroll 4
      for (; i + N <= inner; i += 64 * N) {
        const V v = *(const V*)(row + i);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const double d = (double)to_f32(v[e]);
          s[e & 1] += d * d;
        }
      }
    for (; i < inner; i += 64 * N)
      for (int e = 0; e < N && i + e < inner; ++e) {
        const double d = (double)to_f32(row[(i + e) * is]);
        s[e & 1] += d * d;
      }
  }
  double sum = s[0] + s[1];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  __shared__ double part[4];
  if (x == 0) part[y] = sum;
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
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split(float v, float u, f16x2* hi, f16x2* lo) {  // (two at a time: one conversion instruction)
  *hi = __builtin_convertvector(f32x2{v, u}, f16x2);
  *lo = __builtin_convertvector(f32x2{v - (float)(*hi)[0], u - (float)(*hi)[1]}, f16x2);
}
__device__ __forceinline__ void split8(const float* v, f16x8* hi, f16x8* lo) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f16x2 h, o;
    split(v[e], v[e + 1], &h, &o);
    (*hi)[e] = h[0];
    (*hi)[e + 1] = h[1];
    (*lo)[e] = o[0];
    (*lo)[e + 1] = o[1];
  }
}

// G -> X_0 (p rows) and its transpose (q rows), zero-padded.  One 64 x 64 tile a workgroup; each adds the parts of the norm up for itself while its
// elements are on the way (a launch of its own for that took 4 us), the first of a matrix leaves the factors for the products.
template <class T>
__global__ __launch_bounds__(256) void k_ns_pack(NsMatrix w, const double* parts, int count, double eps, NsCoef cf, int steps, NsScales* scales, char* x,
                                                 char* xt, size_t batch_bytes) {
  __shared__ float tile[64][65];
  __shared__ NsCoef mine;
  __shared__ NsScales z;
  __shared__ double part[4];
  const T* g = (const T*)w.g + blockIdx.z * w.batch_stride;
  x += blockIdx.z * batch_bytes;
  xt += blockIdx.z * batch_bytes;
  const long p0 = (long)blockIdx.y * 64, q0 = (long)blockIdx.x * 64;
  const bool along_q = w.col_stride <= w.row_stride;
  const int l = threadIdx.x & 63, r = threadIdx.x >> 6;
  T v[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int o = r + 4 * u, pi = along_q ? o : l, qi = along_q ? l : o;
    v[u] = p0 + pi < w.p && q0 + qi < w.q ? g[(p0 + pi) * w.row_stride + (q0 + qi) * w.col_stride] : (T)0.0f;
  }
  ns_fetch(cf, steps, &mine, z.f);
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 256) s += parts[(size_t)blockIdx.z * NS_PARTS + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (l == 0) part[r] = s;
  __syncthreads();
  if (threadIdx.x == 0) ns_scales((part[0] + part[1]) + (part[2] + part[3]), eps, mine, steps, z);
  __syncthreads();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < (int)(sizeof(NsScales) / 4); i += 256) ((int*)(scales + blockIdx.z))[i] = ((const int*)&z)[i];
  const double f = z.first;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int o = r + 4 * u;
    tile[along_q ? o : l][along_q ? l : o] = (float)((double)to_f32(v[u]) * f);
  }
  __syncthreads();
  const size_t ldx = pair_ld(w.q), ldt = pair_ld(w.p);
  const int row = threadIdx.x >> 2, from = (threadIdx.x & 3) * 16;
  for (int turn = 0; turn < 2; ++turn) {
    char* base = turn ? xt + pair_at(q0 + row, p0 + from, ldt) : x + pair_at(p0 + row, q0 + from, ldx);
    if (turn ? q0 + row >= w.q : p0 + row >= w.p) continue;
    f16x8 hi[2], lo[2];
    float e[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) e[k] = turn ? tile[from + k][row] : tile[row][from + k];
    split8(e, &hi[0], &lo[0]);
    split8(e + 8, &hi[1], &lo[1]);
    *(f16x8*)base = hi[0];
    *(f16x8*)(base + 16) = hi[1];
    *(f16x8*)(base + PAIR_LO) = lo[0];
    *(f16x8*)(base + PAIR_LO + 16) = lo[1];
  }
}

enum NsKind { NS_GRAM, NS_POLY, NS_STEP, NS_LAST };

struct NsArgs {
  const char *P, *Q;      // operands of the product
  const char* E;          // the matrix the epilogue adds, natural orientation (POLY: A, STEP / LAST: X)
  char *D, *DT;           // result and its transpose; symmetric products write both halves of D
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
  split8(v, &h, &o);
  *(f16x8*)at = h;
  *(f16x8*)(at + PAIR_LO) = o;
}

template <int KIND, class T, class TL, int BI, int BJ>
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
  const NsScales& z = g.scales[blockIdx.z];
  const NsFactors f = z.f[g.t];
  const int last = z.last;
  const char* E = g.E + off;
  // A chunk's groups of eight elements, TURNS a thread: row r, words iw .. iw + 7
  constexpr int ACROSS = TL::W / 8, TURNS = TL::ROWS * ACROSS / TL::TEAM;
  static_assert(TURNS * TL::TEAM == TL::ROWS * ACROSS, "chunks must divide over the threads");
  auto place = [&](int u, int* r, int* iw) {
    const bool straight = TL::TEAM % ACROSS == 0;  // (iw is the same in all turns)
    const int at = straight ? TL::who() : TL::who() + u * TL::TEAM;
    *r = at / ACROSS + (straight ? u * (TL::TEAM / ACROSS) : 0);
    *iw = at % ACROSS * 8;
  };
  auto addend = [&](int i, int j, f16x8* h, f16x8* o) {  // eight elements of E; rows are padded: whole groups of eight, zeros behind the end
    *h = *o = f16x8{};
    if (j < g.J && (size_t)i * 4 < ldi) {
      const char* at = E + pair_at(j, i, ldi);
      *h = *(const f16x8*)at;
      *o = *(const f16x8*)(at + PAIR_LO);
    }
  };
  // What the epilogue adds is fetched in batches: for tiles of one chunk before the product, else before the chunk goes to LDS, four turns at a time.
  // (A fetch a turn, each waited for, was 5 .. 10 us of a product.)
  constexpr bool EARLY = KIND != NS_GRAM && TL::CHUNKS == 1;
  constexpr int BATCH = TURNS % 4 == 0 ? 4 : TURNS % 3 == 0 ? 3 : TURNS;
  f16x8 eh[BATCH], el[BATCH];
  auto batch = [&](int c, int u0) {
    if (KIND == NS_GRAM) return;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      int r, iw;
      place(u0 + u, &r, &iw);
      addend(i0 + TL::row0() + iw, j0 + TL::column0(c) + r, &eh[u], &el[u]);
    }
  };
  if constexpr (EARLY) batch(0, 0);
  TL t;
  t.run(Operand{g.P + off, (unsigned)ldk, g.I}, i0, Operand{g.Q + off, (unsigned)ldk, g.J}, j0, (g.K + 31) / 32, 128, lds);
  char* D = g.D + off;
  char* DT = SYM ? D : g.DT + off;
  T* out = (T*)g.out + blockIdx.z * g.out_stride;
  const bool natural = KIND != NS_LAST || !g.transposed, turned = KIND == NS_LAST ? g.transposed != 0 : SYM ? bi != bj : true;
  // Chunks of the tile through LDS: the result in the product's own orientation (rows j, eight neighbours i a thread), then, from the values left
  // there, its transpose (rows i, eight neighbours j).
  constexpr int DOWN = TL::ROWS / 8;
  char* mine = TL::part(lds);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < TL::CHUNKS; ++c) {
    if constexpr (!EARLY) batch(c, 0);
    t.spill(c, mine);
#pragma unroll 1
    for (int u0 = 0; u0 < TURNS; u0 += BATCH) {
    if (u0) batch(c, u0);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      int r, iw;
      place(u0 + u, &r, &iw);
      const int i = i0 + TL::row0() + iw, j = j0 + TL::column0(c) + r;
      float v[8];
      chunk_sums<TL, 8>(mine, r, iw, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = KIND == NS_GRAM ? 0.0f : (float)eh[u][e] + (float)el[u][e];
        float w = v[e];
        if (KIND == NS_GRAM) w = f.gram * w;
        if (KIND == NS_POLY) w = f.lin * x + f.quad * w;
        if (KIND == NS_STEP) w = f.keep * x + f.add * w;
        if (KIND == NS_LAST) w = ldexpf(f.keep * x + f.add * w, last);
        v[e] = i + e < g.I && j < g.J ? w : 0.0f;
      }
      if (turned)
#pragma unroll
        for (int e = 0; e < 8; e += 4) *(f32x4*)((float*)mine + r * TL::PITCH + iw + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
      if (KIND != NS_LAST) {
        if (j < g.J && (size_t)i * 4 < ldi) store_pairs(D + pair_at(j, i, ldi), v);
      } else if (natural && j < g.J && i < g.I) {
        store_some<T, 8>(out + (size_t)j * g.I + i, v, g.I - i);
      }
    }
    }
    if (turned) {
      TL::settle();
      for (int at = TL::who(); at < TL::W * DOWN; at += TL::TEAM) {
        const int ii = at / DOWN, rv = at % DOWN * 8;
        const int irow = i0 + TL::row0() + ii, j = j0 + TL::column0(c) + rv;
        if (irow >= g.I) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ((const float*)mine)[(rv + e) * TL::PITCH + ii];
        if (KIND != NS_LAST) {
          if ((size_t)j * 4 < ldj) store_pairs(DT + pair_at(irow, j, ldj), v);
        } else if (j < g.J) {
          store_some<T, 8>(out + (size_t)irow * g.J + j, v, g.J - j);
        }
      }
    }
  }
}

// ---- up to 128 rows -----------------------------------------------------------------------------------------------------------------------------
// Everything p x p fits one workgroup of eight waves; X is dealt out to the waves by columns and stays in registers in float32, in the places the matrix
// instruction leaves its results in: a wave has column blocks of 16, lane l the column l % 16, register r of row block a the row 16 a + 4 (l / 16) + r.
//   S X for a p x p matrix S contracts over rows, which lie along registers: the registers of two neighbouring row blocks ARE a fragment of the
//   16 x 16 x 32 instruction if k runs in the order {4 g .. 4 g + 3, 16 + 4 g .. 16 + 4 g + 3} for quarter g of the lanes.  So S lies in LDS with its columns
//   in that order (an "image", hi and lo planes) and X never moves (ns_times).
//   A = X X^T contracts over columns, which lie across lanes: X goes through LDS as rows (ns_rows, ns_gram).
// Rows of LDS planes are 16 bytes longer than their numbers: eight neighbouring rows start in different banks.
//
// Chains: with P_t = a + b A_t + c A_t A_t the iterates are X_t+1 = P_t X_t and A_t+1 = P_t A_t P_t, so steps t .. t' can be done on p x p matrices
// alone, Q <- P Q, and X is multiplied once, by Q.  What it costs is accuracy: A's roundings, 2^-23 of its LARGEST eigenvalue, grow with the square of what a
// chain lets small singular values grow by.  A chain may be so long that this stays below a sixteenth of half a step of the result: growth up to 45 for
// bfloat16 (three standard steps), 16 for float16 (two), none for float32.  (Worst of one to four strong directions over noise of 1e-1 .. 3e-4, up to 16
// standard and 32 cubic steps, 16 .. 128 rows, in units of the result's own rounding: growth 500 in bfloat16 3.8, 45 in float16 0.4; as
// above 0.1 and 0.2.  64 x 512 bfloat16 34.5 us against 27.9 in one chain, 64 x 8192 47 / 35; float16 40 / 34 and 58 / 47 in 3 + 2; float32 52 and 80.)
// Bound by latency and by vector instructions (roundings to pairs) for few matrices: a step is a chain of dependent products, LDS round trips and
// barriers.  Five float32 steps of a 64 x 64 matrix take 20 us, of a 128 x 128 one 54 us; column blocks of 32 and the 32 x 32 x 16 instruction read half
// as much LDS but keep half as many waves busy (26 and 63 us).  Two column blocks at a time beside all of X are more than 256 registers for 64 x 512 (66
// of them spill, 54 us in float32), 128 x 256 (42, 84 us) and 64 x 256 (32).
template <int PB, bool F>
struct NsRows {
  static constexpr int P = 32 * PB, RB = 2 * PB;              // rows, row blocks
  // F: the result is float32.  Up to 32 rows its products are of float32 itself, 16 x 16 x 4 a time: few rows are where 22 bits show beside plain float32
  // (4 x 304, six steps: error 3.4e-6 against 0.8e-6, so 0.9e-6).  The price: 23 x 761 42 us against 37.  More rows: pairs, with lo lo where a matrix of
  // the chain is multiplied (58 x 2574: 2.2e-6, plain float32 1.4e-6; so 1.9e-6; 32 of 64 x 128 28 us against 27).
  static constexpr bool FULL = F && PB == 1;
  static constexpr int PITCH = P * (FULL ? 4 : 2) + 16, IMAGE = (FULL ? 1 : 2) * P * PITCH;
  static constexpr bool BOTH = PB > 2;                        // A's and Q's column blocks on the same waves, else A on the first four, Q on the others
  static constexpr int KS = 8 / RB;                           // most waves that share a column block of A
  static constexpr int PARTS = KS > 1 ? (KS - 1) * P * P * 4 : 0;
  // Adding shares up costs about as much as the K steps it saves for short rows.  blocks: column blocks of X
  __device__ static int shares(int blocks) { return KS == 1 ? 1 : min(KS, max(1, blocks / 8)); }
};
template <int PB, int CB, bool F>
struct NsLds {  // X of 128 CB columns as rows (a constant pitch: their addresses are offsets of one another), or two images, or the shares
  using S = NsRows<PB, F>;
  static constexpr int PITCH = CB * (S::FULL ? 512 : 256) + 16, X = (S::FULL ? 1 : 2) * S::P * PITCH;
  static constexpr int IMAGES = X > 2 * S::IMAGE ? X : 2 * S::IMAGE;
  static constexpr int BYTES = IMAGES > S::PARTS ? IMAGES : S::PARTS;
};
template <class T, int PB>
constexpr bool ns_full() {
  return sizeof(T) == 4;
}
template <int PB>
using NsCols = float[2 * PB][4];  // a column block of a p-row matrix

// y = S x for N column blocks, S an image (rb: its row blocks of 16 that are not zeros): every wave reads all of S, so blocks done together share what bounds it, the reads of LDS.  One fragment of x
// at a time is split and met by all row blocks.
template <int PB, bool F, int N>
__device__ __forceinline__ void ns_times(const char* image, int rb, const NsCols<PB>* const (&x)[N], NsCols<PB>* const (&y)[N]) {
  using S = NsRows<PB, F>;
  const int l = lane_id();
  const char* at = image + (l & 15) * S::PITCH + (l >> 4) * 16;
  constexpr int APART = N == 1 && PB <= 2 ? 2 : 1;  // few accumulators: the small products in ones of their own
  f32x4 acc[N][APART][S::RB];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 0; o < APART; ++o)
#pragma unroll
      for (int a = 0; a < S::RB; ++a) acc[n][o][a] = f32x4{};
  if constexpr (S::FULL) {  // register r of row block k is the rows 16 k + 4 (l / 16) + r: an operand as it is
#pragma unroll
    for (int k = 0; k < S::RB; ++k)
#pragma unroll
      for (int a = 0; a < S::RB; ++a) {
        if (k >= rb || a >= rb) continue;
        const f32x4 b = *(const f32x4*)(at + a * 16 * S::PITCH + k * 64);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < N; ++n) acc[n][r % APART][a] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[r], (*x[n])[k][r], acc[n][r % APART][a], 0, 0, 0);
      }
  }
#pragma unroll
  for (int k = 0; k < (S::FULL ? 0 : PB); ++k) {
    f16x8 xh[N], xl[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const NsCols<PB>& c = *x[n];
      const float v[8] = {c[2 * k][0], c[2 * k][1], c[2 * k][2], c[2 * k][3], c[2 * k + 1][0], c[2 * k + 1][1], c[2 * k + 1][2], c[2 * k + 1][3]};
      split8(v, &xh[n], &xl[n]);
    }
#pragma unroll
    for (int a = 0; a < S::RB; ++a) {
      const f16x8 bh = *(const f16x8*)(at + a * 16 * S::PITCH + k * 64), bl = *(const f16x8*)(at + (a * 16 + S::P) * S::PITCH + k * 64);
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n][0][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh, xh[n], acc[n][0][a], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n][APART - 1][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl, xh[n], acc[n][APART - 1][a], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n][APART - 1][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh, xl[n], acc[n][APART - 1][a], 0, 0, 0);
      if (F)
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n][APART - 1][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl, xl[n], acc[n][APART - 1][a], 0, 0, 0);
      if (PB > 2 && a % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    if (PB > 1) {  // one step's fragments at a time: all of them would not fit the registers
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int o = 0; o < APART; ++o)
#pragma unroll
          for (int a = 0; a < S::RB; ++a) asm volatile("" : "+v"(acc[n][o][a]));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int a = 0; a < S::RB; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) (*y[n])[a][r] = APART == 1 ? acc[n][0][a][r] : acc[n][0][a][r] + acc[n][APART - 1][a][r];
}
template <int PB, bool F>
__device__ __forceinline__ void ns_times(const char* image, int rb, const NsCols<PB>& x, NsCols<PB>& y) {
  const NsCols<PB>* const from[1] = {&x};
  NsCols<PB>* const to[1] = {&y};
  ns_times<PB, F, 1>(image, rb, from, to);
}
// A column block to rows of LDS (hi plane, lo plane `plane` bytes on): the lane's column is at byte `at`, rows are `pitch` apart.  Neighbouring lanes swap
// halves of two rows, so that each writes two neighbours of one.
template <int PB>
__device__ __forceinline__ void ns_scatter(char* lds, int pitch, int plane, int at, const NsCols<PB>& x) {
  const int l = lane_id();
  const bool odd = l & 1;
  char* base = lds + (4 * (l >> 4) + odd) * pitch + at - 2 * odd;
  const unsigned pick = odd ? 0x03020706u : 0x05040100u;  // bytes of (mine, the neighbour's): even lanes the lower halves, odd lanes the upper ones
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      f16x2 hi, lo;
      split(x[a][r], x[a][r + 1], &hi, &lo);
      char* to = base + (16 * a + r) * pitch;
      const unsigned mh = __builtin_bit_cast(unsigned, hi), ml = __builtin_bit_cast(unsigned, lo);
      const unsigned nh = (unsigned)__builtin_amdgcn_mov_dpp((int)mh, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2
      const unsigned nl = (unsigned)__builtin_amdgcn_mov_dpp((int)ml, 0xb1, 0xf, 0xf, true);
      *(unsigned*)to = __builtin_amdgcn_perm(nh, mh, pick);
      *(unsigned*)(to + plane) = __builtin_amdgcn_perm(nl, ml, pick);
    }
}
// .. to rows of float32, from column c on
template <int PB>
__device__ __forceinline__ void ns_lay(char* lds, int pitch, int c, const NsCols<PB>& x) {
  const int l = lane_id();
  char* base = lds + 4 * (l >> 4) * pitch + (c + (l & 15)) * 4;
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) *(float*)(base + (16 * a + r) * pitch) = x[a][r];
}
// Column block b of a p x p matrix into an image.  (Row i of the image is row i: the matrices of a chain are symmetric but for their roundings, and an
// image of the transpose would make those grow - the products of a chain commute only as long as all are polynomials of the SAME A.)
template <int PB, bool F>
__device__ __forceinline__ void ns_put(char* image, int b, const NsCols<PB>& x) {
  using S = NsRows<PB, F>;
  const int c = lane_id() & 15;
  if constexpr (NsRows<PB, F>::FULL)
    ns_lay<PB>(image, S::PITCH, 16 * b, x);
  else
    ns_scatter<PB>(image, S::PITCH, S::P * S::PITCH, 64 * (b >> 1) + 16 * (c >> 2) + 8 * (b & 1) + 2 * (c & 3), x);
}
// Column block number c of X to rows
template <int PB, int CB, bool F>
__device__ __forceinline__ void ns_rows(char* lds, int c, const NsCols<PB>& x) {
  using L = NsLds<PB, CB, F>;
  if constexpr (NsRows<PB, F>::FULL)
    ns_lay<PB>(lds, L::PITCH, 16 * c, x);
  else
    ns_scatter<PB>(lds, L::PITCH, NsRows<PB, F>::P * L::PITCH, 32 * c + 2 * (lane_id() & 15), x);
}
// Column block w % RB of X X^T from the rows in LDS, wave w's share w / RB of the K range, then the shares added up: waves 0 .. RB - 1 have the result.
// blocks: an even number of column blocks of X.  All rows have been read when this returns (a barrier).
template <int PB, int CB, bool F>
__device__ __forceinline__ void ns_gram(char* lds, int rb, int blocks, NsCols<PB>& m) {
  using S = NsRows<PB, F>;
  constexpr int pitch = NsLds<PB, CB, F>::PITCH;
  const int w = wave_id(), l = lane_id(), shares = S::shares(blocks);
  constexpr int APART = PB <= 2 ? 2 : 1;
  f32x4 acc[APART][S::RB];
#pragma unroll
  for (int o = 0; o < APART; ++o)
#pragma unroll
    for (int a = 0; a < S::RB; ++a) acc[o][a] = f32x4{};
  if (w < S::RB * shares && w % S::RB < rb) {
    const char* at = lds + (l & 15) * pitch + (l >> 4) * 16;
    const int j = w % S::RB * 16;
    if constexpr (S::FULL) {
      for (int k = w / S::RB; 2 * k < blocks; k += shares)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 jv = *(const f32x4*)(at + j * pitch + k * 128 + h * 64);
#pragma unroll
          for (int a = 0; a < S::RB; ++a) {
            if (a >= rb) continue;
            const f32x4 iv = *(const f32x4*)(at + 16 * a * pitch + k * 128 + h * 64);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r % APART][a] = __builtin_amdgcn_mfma_f32_16x16x4f32(iv[r], jv[r], acc[r % APART][a], 0, 0, 0);
          }
        }
    }
    for (int k = w / S::RB; !S::FULL && 2 * k < blocks; k += shares) {
      const f16x8 jh = *(const f16x8*)(at + j * pitch + k * 64), jl = *(const f16x8*)(at + (j + S::P) * pitch + k * 64);
#pragma unroll
      for (int a = 0; a < S::RB; ++a) {
        const f16x8 ih = *(const f16x8*)(at + 16 * a * pitch + k * 64), il = *(const f16x8*)(at + (16 * a + S::P) * pitch + k * 64);
        acc[0][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ih, jh, acc[0][a], 0, 0, 0);
        acc[APART - 1][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(il, jh, acc[APART - 1][a], 0, 0, 0);
        acc[APART - 1][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ih, jl, acc[APART - 1][a], 0, 0, 0);
        if (PB > 2 && a % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
#pragma unroll
  for (int a = 0; a < S::RB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) m[a][r] = APART == 1 ? acc[0][a][r] : acc[0][a][r] + acc[APART - 1][a][r];
  __syncthreads();
  if (shares == 1) return;
  if (w >= S::RB && w < S::RB * shares) {
    f32x4* mine = (f32x4*)lds + (w - S::RB) * S::RB * 64 + l;
#pragma unroll
    for (int a = 0; a < S::RB; ++a) mine[a * 64] = f32x4{m[a][0], m[a][1], m[a][2], m[a][3]};
  }
  __syncthreads();
  if (w < S::RB) {
    for (int o = 1; o < shares; ++o) {
      const f32x4* its = (const f32x4*)lds + (o * S::RB + w - S::RB) * S::RB * 64 + l;
#pragma unroll
      for (int a = 0; a < S::RB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) m[a][r] += its[a * 64][r];
    }
  }
  __syncthreads();
}
// m[row][column] += v where they are equal; b: the column block
template <int PB>
__device__ __forceinline__ void ns_diagonal(int b, float v, NsCols<PB>& m) {
  const int l = lane_id();
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
    if (a == b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * (l >> 4) + r == (l & 15)) m[a][r] += v;
}
template <int PB>
__device__ __forceinline__ void ns_scale(float v, NsCols<PB>& m) {
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) m[a][r] *= v;
}
// From A (waves 0 .. RB - 1: its column blocks, as summed) the image that X is multiplied with: B of a single step, or Q of the chain t .. end.
// Images at lds and lds + IMAGE; returns the one that holds it; a barrier has passed.
template <int PB, bool F>
__device__ __forceinline__ char* ns_chain(char* lds, int rb, NsCols<PB>& m, const NsScales& z, int t, int end) {
  using S = NsRows<PB, F>;
  const int w = wave_id(), first_q = S::BOTH ? 0 : 4;
  const bool a_wave = w < S::RB, q_wave = w >= first_q && w < first_q + S::RB;
  char *ia = lds, *ip = lds + S::IMAGE;
  NsCols<PB> own;  // Q's column block, where the wave has A's too
  NsCols<PB>& q = S::BOTH ? own : m;
  ns_scale<PB>(z.f[t].gram, m);
  const bool alone = t == end;
  if (!alone && q_wave) {
#pragma unroll
    for (int a = 0; a < S::RB; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) q[a][r] = 0.0f;
    ns_diagonal<PB>(w - first_q, (float)(1 << NS_UNIT), q);
  }
  for (;; ++t) {
    const NsFactors f = z.f[t];
    if (a_wave) ns_put<PB, F>(ia, w, m);
    __syncthreads();
    if (a_wave) {
      NsCols<PB> p;
      ns_times<PB, F>(ia, rb, m, p);
#pragma unroll
      for (int a = 0; a < S::RB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[a][r] = f.lin * m[a][r] + f.quad * p[a][r];
      if (!alone) ns_diagonal<PB>(w, f.unit, p);
      ns_put<PB, F>(ip, w, p);
    }
    __syncthreads();
    if (alone) return ip;
    // Q <- P Q; R = P A, A <- P R
    if (S::BOTH && a_wave && t != end) {
      NsCols<PB> r, y;
      const NsCols<PB>* const from[2] = {&m, &q};
      NsCols<PB>* const to[2] = {&r, &y};
      ns_times<PB, F, 2>(ip, rb, from, to);
      ns_scale<PB>(f.half, r);
#pragma unroll
      for (int a = 0; a < S::RB; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) q[a][e] = f.chain * y[a][e];
      ns_times<PB, F>(ip, rb, r, m);
      ns_scale<PB>(f.next, m);
      continue;
    }
    if (q_wave) {
      NsCols<PB> y;
      ns_times<PB, F>(ip, rb, q, y);
#pragma unroll
      for (int a = 0; a < S::RB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) q[a][r] = f.chain * y[a][r];
    }
    if (t == end) break;
    if (!S::BOTH && a_wave) {
      NsCols<PB> r;
      ns_times<PB, F>(ip, rb, m, r);
      ns_scale<PB>(f.half, r);
      ns_times<PB, F>(ip, rb, r, m);
      ns_scale<PB>(f.next, m);
    }
  }
  if (q_wave) ns_put<PB, F>(ia, w - first_q, q);
  __syncthreads();
  return ia;
}
// Column block number c of G, from column j0 on.  (32-bit offsets within the matrix: the host sees to it.)
// Rows past the end are read from the last one, columns past it from the first, and count as zeros: all loads are under way together.
template <class T, int PB>
__device__ __forceinline__ void ns_load(const T* g, const NsMatrix& m, long j0, int c, NsCols<PB>& x) {
  const int l = lane_id();
  const long jb = j0 + 16 * c, j = jb + (l & 15);
  const char* from = (const char*)(jb < m.q ? g + jb * m.col_stride : g);
  const unsigned rs = (unsigned)m.row_stride * (unsigned)sizeof(T);
  const unsigned side = (j < m.q ? l & 15 : 0) * (unsigned)m.col_stride * (unsigned)sizeof(T);
  const int rows = j < m.q ? (int)m.p - 4 * (l >> 4) : 0;
  const unsigned end = ((unsigned)m.p - 1) * rs + side;
  unsigned at = 4 * (l >> 4) * rs + side;
  T v[2 * PB][4];
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[a][r] = *(const T*)(from + min(at, end));
      at += r == 3 ? 13 * rs : rs;  // rows 0 1 2 3, 16 17 18 19, ..
    }
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) x[a][r] = 16 * a + r < rows ? to_f32(v[a][r]) : 0.0f;
}
template <class T, int PB>
__device__ __forceinline__ void ns_store(T* out, const NsMatrix& m, long j0, int c, const NsCols<PB>& x, int last, bool tall) {
  const int l = lane_id();
  const long j = j0 + 16 * c + (l & 15);
  const long rs = tall ? 1 : m.q, cs = tall ? m.p : 1;
  char* col = (char*)(out + (j0 + 16 * c) * cs);
  const unsigned step = (unsigned)rs * (unsigned)sizeof(T);
  int rows = j < m.q ? (int)m.p - 4 * (l >> 4) : 0;
  asm volatile("" : "+v"(rows));  // (compare again: the masks of the load are not worth keeping in scalar registers until here)
  unsigned at = 4 * (l >> 4) * step + (l & 15) * (unsigned)cs * (unsigned)sizeof(T);
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (16 * a + r < rows) *(T*)(col + at) = (T)ldexpf(x[a][r], last);
      at += r == 3 ? 13 * step : step;
    }
}
template <int PB>
__device__ __forceinline__ void ns_first(double first, NsCols<PB>& x) {
#pragma unroll
  for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) x[a][r] = (float)((double)x[a][r] * first);
}
// X <- keep X + add S X for the wave's column blocks w, w + 8, .. below `blocks`, two at a time
template <int PB, int CB, bool F>
__device__ __forceinline__ void ns_advance(const char* image, int rb, float keep, float add, int blocks, NsCols<PB> (&x)[CB]) {
  const int w = wave_id();
  constexpr int N = CB > 1 ? 2 : 1;
#pragma unroll
  for (int c = 0; c < CB; c += N)
    if (w + 8 * c < blocks) {
      NsCols<PB> y[N];
      const NsCols<PB>* from[N];
      NsCols<PB>* to[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        from[n] = &x[c + n];
        to[n] = &y[n];
      }
      ns_times<PB, F, N>(image, rb, from, to);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[c + n][a][r] = keep * x[c + n][a][r] + add * y[n][a][r];
    }
}

// One workgroup does a whole matrix of up to 32 PB x 128 CB.
template <class T, int PB, int CB>
__global__ __launch_bounds__(512) void k_ns_small(NsMatrix m, NsCoef cf, int steps, double eps, T* out, int tall) {
  extern __shared__ char lds[];
  __shared__ NsScales z;
  __shared__ NsCoef mine;
  __shared__ double part[8];
  const int l = lane_id(), w = wave_id();
  ns_fetch(cf, steps, &mine, z.f);
  constexpr bool F = ns_full<T, PB>();
  const int blocks = (int)((m.q + 31) / 32) * 2, rb = (int)(m.p + 15) / 16;
  const T* g = (const T*)m.g + blockIdx.x * m.batch_stride;
  NsCols<PB> x[CB];
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < CB; ++c) ns_load<T, PB>(g, m, 0, w + 8 * c, x[c]);
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int a = 0; a < 2 * PB; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += (double)x[c][a][r] * (double)x[c][a][r];
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
#pragma unroll
  for (int c = 0; c < CB; ++c) ns_first<PB>(z.first, x[c]);
  for (int t = 0; t < steps;) {
    int end = t;
    while (!(mine.ends >> end & 1)) ++end;
#pragma unroll
    for (int c = 0; c < CB; ++c)
      if (w + 8 * c < blocks) ns_rows<PB, CB, F>(lds, w + 8 * c, x[c]);
    __syncthreads();
    NsCols<PB> a;
    ns_gram<PB, CB, F>(lds, rb, blocks, a);
    const char* image = ns_chain<PB, F>(lds, rb, a, z, t, end);
    ns_advance<PB, CB, F>(image, rb, z.f[end].keep, z.f[end].add, blocks, x);
    t = end + 1;
    if (t < steps) __syncthreads();
  }
  T* y = out + blockIdx.x * (size_t)(m.p * m.q);
#pragma unroll
  for (int c = 0; c < CB; ++c) ns_store<T, PB>(y, m, 0, w + 8 * c, x[c], z.last, tall);
}

// ---- up to 128 rows, any number of columns --------------------------------------------------------------------------------------------------------
// Workgroups take slabs of 256 columns.  One launch a chain of steps: every workgroup adds the slabs' shares of A up (k_ns_sum has done so before where
// there are many), works the chain out for itself - all do the same, the result does not have to travel - multiplies its slab and leaves its share
// of the next A.  Between launches X lies in the workspace as the registers had it.
struct NsSlabs {
  NsMatrix m;
  const double* parts;   // sums of squares (k_ns_norm)
  int count;
  double eps;
  NsScales* scales;
  float* x;              // a matrix's X
  const float* a;        // its slabs' shares of A (32 PB x 32 PB floats each, in register order)
  float* next_a;         // .. of the next A: in another place, for a workgroup may be done before another one has begun
  size_t x_batch, a_batch;  // floats from matrix to matrix
  int shares;            // .. to add up
  int steps, t, end;     // the chain; first launch: t < 0
  void* out;
  int tall;
};
constexpr int NS_SLAB = 256;

template <class T, int PB, bool FIRST>
__global__ __launch_bounds__(512) void k_ns_slab(NsSlabs g, NsCoef cf) {
  constexpr bool F = ns_full<T, PB>();
  using S = NsRows<PB, F>;
  constexpr int CB = NS_SLAB / 128, FLOATS = S::RB * 4 * 64;  // of a column block
  extern __shared__ char lds[];
  __shared__ NsScales z;
  __shared__ NsCoef mine;
  const int l = lane_id(), w = wave_id();
  const long j0 = (long)blockIdx.x * NS_SLAB;
  const int blocks = (int)((min((long)NS_SLAB, g.m.q - j0) + 31) / 32) * 2, rb = (int)(g.m.p + 15) / 16;
  float* xs = g.x + blockIdx.y * g.x_batch + ((size_t)blockIdx.x * 8 + w) * CB * FLOATS + l * 4;
  const T* from = (const T*)g.m.g + blockIdx.y * g.m.batch_stride;
  const bool fresh = FIRST || g.t == 0;  // X_0 comes from G
  const bool last = !FIRST && g.end + 1 == g.steps;
  NsCols<PB> x[CB], m;
  if (fresh) {
#pragma unroll
    for (int c = 0; c < CB; ++c) ns_load<T, PB>(from, g.m, j0, w + 8 * c, x[c]);
  } else {
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int a = 0; a < S::RB; ++a) {
        const f32x4 v = *(const f32x4*)(xs + c * FLOATS + a * 256);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[c][a][r] = v[r];
      }
  }
  if constexpr (FIRST) {
    ns_fetch(cf, g.steps, &mine, z.f);
    double s = 0.0;
    if (w == 0)
      for (int i = l; i < g.count; i += 64) s += g.parts[(size_t)blockIdx.y * NS_PARTS + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    __syncthreads();
    if (threadIdx.x == 0) ns_scales(s, g.eps, mine, g.steps, z);
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < (int)(sizeof(NsScales) / 4); i += 512) ((int*)(g.scales + blockIdx.y))[i] = ((const int*)&z)[i];
  } else {
    for (int i = threadIdx.x; i < (int)(sizeof(NsScales) / 4); i += 512) ((int*)&z)[i] = ((const int*)(g.scales + blockIdx.y))[i];
    if (w < S::RB) {
      const float* at = g.a + blockIdx.y * g.a_batch + w * FLOATS + l * 4;
#pragma unroll
      for (int a = 0; a < S::RB; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) m[a][r] = 0.0f;
      for (int o = 0; o < g.shares; ++o, at += S::P * S::P)
#pragma unroll
        for (int a = 0; a < S::RB; ++a) {
          const f32x4 v = *(const f32x4*)(at + a * 256);
#pragma unroll
          for (int r = 0; r < 4; ++r) m[a][r] += v[r];
        }
    }
    __syncthreads();
  }
  if (fresh) {
#pragma unroll
    for (int c = 0; c < CB; ++c) ns_first<PB>(z.first, x[c]);
  }
  if constexpr (!FIRST) {
    const char* image = ns_chain<PB, F>(lds, rb, m, z, g.t, g.end);
    ns_advance<PB, CB, F>(image, rb, z.f[g.end].keep, z.f[g.end].add, blocks, x);
    if (last) {
      T* y = (T*)g.out + blockIdx.y * (size_t)(g.m.p * g.m.q);
#pragma unroll
      for (int c = 0; c < CB; ++c) ns_store<T, PB>(y, g.m, j0, w + 8 * c, x[c], z.last, g.tall);
      return;
    }
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int a = 0; a < S::RB; ++a) *(f32x4*)(xs + c * FLOATS + a * 256) = f32x4{x[c][a][0], x[c][a][1], x[c][a][2], x[c][a][3]};
    __syncthreads();  // the image has been read
  }
#pragma unroll
  for (int c = 0; c < CB; ++c)
    if (w + 8 * c < blocks) ns_rows<PB, CB, F>(lds, w + 8 * c, x[c]);
  __syncthreads();
  ns_gram<PB, CB, F>(lds, rb, blocks, m);
  if (w < S::RB) {
    float* at = g.next_a + blockIdx.y * g.a_batch + (size_t)blockIdx.x * S::P * S::P + w * FLOATS + l * 4;
#pragma unroll
    for (int a = 0; a < S::RB; ++a) *(f32x4*)(at + a * 256) = f32x4{m[a][0], m[a][1], m[a][2], m[a][3]};
  }
}

// The slabs' shares of A added up into the first, in order: one thread four numbers, from all slabs
__global__ __launch_bounds__(64) void k_ns_sum(float* a, size_t a_batch, int floats, int slabs) {
  float* at = a + blockIdx.y * a_batch + ((size_t)blockIdx.x * 64 + threadIdx.x) * 4;
  f32x4 s = *(const f32x4*)at;
#pragma unroll 8
  for (int o = 1; o < slabs; ++o) s += *(const f32x4*)(at + (size_t)o * floats);
  *(f32x4*)at = s;
}

}  // namespace lb
