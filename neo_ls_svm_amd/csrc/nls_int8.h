// 8-bit rows and their products: quantisation, the product of few rows (bound by reading b), the product of many rows (matrix cores).
#pragma once
#include "nls_tile.h"

namespace lb {

// ---- quantise rows --------------------------------------------------------------------------------------------------------------------------
// scale = max|x| / 127, q = 127 x / max|x| to the nearest integer, ties to even, decided as if in exact arithmetic:
// r = x * inv with inv = fl(127 / max|x|) is off by less than 127 * 2^-23 = 1.5e-5; only where a piece of the row has an r that near to a half is the
// quotient formed in 64 bits - 127 x is exact there, and a quotient of a 31-bit by a 24-bit number that is no half is at least 2^-26 away from one.
// Adding 1.5 * 2^23 rounds r and leaves the integer in the sum's low byte.
// A row with a NaN or an infinity gets that as its scale and zeros as q (the product then gives NaN in the whole row); a row of zeros, scale 0.
struct RowScale {
  float top, inv;
  int kind;  // 0: the usual row; 1: all through 64 bits (127 / top is out of range); 2: zeros
};
__device__ __forceinline__ RowScale row_scale(unsigned topbits) {
  RowScale s;
  s.top = __uint_as_float(topbits);
  s.kind = (topbits == 0u || topbits >= 0x7f800000u) ? 2 : s.top < 1e-35f ? 1 : 0;
  s.inv = s.kind == 0 ? 127.0f / s.top : 0.0f;
  return s;
}
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}
__device__ __forceinline__ unsigned exact4(const float* x, float top) {
  unsigned q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = (unsigned)(int)__builtin_rint((double)x[e] * 127.0 / (double)top);
  return low_bytes(q[0], q[1], q[2], q[3]);
}
// N (a multiple of four) elements to their bytes
template <int N>
__device__ __forceinline__ void quantise(const float (&x)[N], const RowScale& s, unsigned (&q)[N / 4]) {
  constexpr float ROUND = 12582912.0f;
  float far = 0.0f;
  unsigned bits[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float r = x[e] * s.inv, n = r + ROUND;
    bits[e] = __float_as_uint(n);
    far = fmaxf(far, fabsf(r - (n - ROUND)));
  }
#pragma unroll
  for (int e = 0; e < N; e += 4) q[e / 4] = low_bytes(bits[e], bits[e + 1], bits[e + 2], bits[e + 3]);
  if (__builtin_expect(far > 0.49998f || s.kind != 0, 0)) {
#pragma unroll
    for (int e = 0; e < N; e += 4) q[e / 4] = s.kind == 2 ? 0u : exact4(x + e, s.top);
  }
}
// The largest magnitude of a piece, as bits that order |x|, infinity, NaN: of the type itself for 16 bits (two at a time), float32's else
template <class T, int N>
__device__ __forceinline__ unsigned most_bits(const T __attribute__((ext_vector_type(N))) v, unsigned top) {
  if constexpr (sizeof(T) == 2) {
    typedef unsigned short U2 __attribute__((ext_vector_type(2)));
    typedef unsigned W __attribute__((ext_vector_type(N / 2)));
    const W w = __builtin_bit_cast(W, v) & 0x7fff7fffu;
    U2 t = __builtin_bit_cast(U2, top);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) t = __builtin_elementwise_max(t, __builtin_bit_cast(U2, (unsigned)w[e]));
    return __builtin_bit_cast(unsigned, t);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    return top;
  }
}
// .. of all the pieces a wave has seen, as float32's bits
template <class T>
__device__ __forceinline__ unsigned wave_most(unsigned top) {
  if constexpr (sizeof(T) == 2) top = max(top & 0xffffu, top >> 16);
  unsigned o;
#define NLS_MOST(ctrl) o = (unsigned)__builtin_amdgcn_mov_dpp((int)top, ctrl, 0xf, 0xf, true), top = max(top, o)
  NLS_MOST(0xb1);   // lanes 1 0 3 2
  NLS_MOST(0x4e);   // lanes 2 3 0 1
  NLS_MOST(0x141);  // half rows mirrored
  NLS_MOST(0x140);  // rows mirrored
#undef NLS_MOST
  top = max(max((unsigned)__builtin_amdgcn_readlane((int)top, 0), (unsigned)__builtin_amdgcn_readlane((int)top, 16)),
            max((unsigned)__builtin_amdgcn_readlane((int)top, 32), (unsigned)__builtin_amdgcn_readlane((int)top, 48)));
  if constexpr (sizeof(T) == 2) top = __float_as_uint(to_f32(__builtin_bit_cast(T, (unsigned short)top)));
  return top;
}

// Elements a thread takes at once: 16 bytes where the rows are dense (such a load may begin at any element), else four elements one by one.
template <class T, bool VEC>
struct Few {
  static constexpr int N = VEC ? 16 / (int)sizeof(T) : 4;
  typedef T type __attribute__((ext_vector_type(N)));
  typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T, bool VEC>
__device__ __forceinline__ typename Few<T, VEC>::type few_at(const T* x, long c, long k, long col_stride) {
  constexpr int N = Few<T, VEC>::N;
  typename Few<T, VEC>::type v = {};
  if (VEC && c + N <= k) {
    v = *(const typename Few<T, VEC>::loose*)(x + c);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < k) v[e] = x[(c + e) * col_stride];
  }
  return v;
}
template <int N, class V>
__device__ __forceinline__ void quantise_store(const V& v, const RowScale& s, signed char* at) {
  float x[N];
  unsigned q[N / 4];
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = to_f32(v[e]);
  quantise<N>(x, s, q);
  if constexpr (N == 8)
    *(i32x2*)at = i32x2{(int)q[0], (int)q[1]};
  else
    *(unsigned*)at = q[0];
}

// A group of G threads takes a row.  HELD > 0: the row fits into HELD pieces a thread, is read once and stays in registers between the maximum and
// the rounding; HELD = 0: longer rows are read twice (the second time mostly from L2).  Bound by memory: 8192 x 8192 bfloat16 (134 MB in, 67 MB out).
template <class T, int G, bool VEC, int HELD>
__global__ __launch_bounds__(256) void k_quantize_rows(const T* x, long rows, long k, long row_stride, long col_stride, signed char* q, long ldq,
                                                       float* scale) {
  using F = Few<T, VEC>;
  constexpr int N = F::N;
  const int g = threadIdx.x % G;
  const long row = group_id() * (256 / G) + threadIdx.x / G;
  const bool live = row < rows;
  const T* xr = x + (live ? row : rows - 1) * row_stride;
  unsigned top = 0;
  typename F::type held[HELD ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) held[h] = few_at<T, VEC>(xr, (long)N * (g + G * h), k, col_stride);
#pragma unroll
    for (int h = 0; h < HELD; ++h) top = most_bits<T, N>(held[h], top);
  } else {
    for (long c = N * g; c < k; c += N * G) top = most_bits<T, N>(few_at<T, VEC>(xr, c, k, col_stride), top);
  }
  top = wave_most<T>(top);
  if (G > 64) {
    __shared__ unsigned part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  if (!live) return;
  const RowScale s = row_scale(top);
  if (g == 0) scale[row] = s.top / 127.0f;
  signed char* qr = q + row * ldq;  // the row's padding is written as zeros (ldq is a multiple of N)
  if constexpr (HELD > 0) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const long c = (long)N * (g + G * h);
      if (c < ldq) quantise_store<N>(held[h], s, qr + c);
    }
    for (long c = (long)N * (g + G * HELD); c < ldq; c += N * G) quantise_store<N>(typename F::type{}, s, qr + c);
  } else {
    for (long c = N * g; c < ldq; c += N * G) quantise_store<N>(few_at<T, VEC>(xr, c, k, col_stride), s, qr + c);
  }
}

// Rows whose neighbours are neighbours in memory (the rows of a transposed matrix): a workgroup takes 32 of them, 16 bytes of a column a thread - once for
// the maxima, and once more, turned in LDS, for the numbers (which rows take it: see the host code).
template <class T>
struct Turned {
  static constexpr int ROWS = 32, N = 16 / (int)sizeof(T), ACROSS = ROWS / N, COLS = 1024 / ACROSS;  // columns at a time
  static constexpr int PITCH = ROWS * (int)sizeof(T) + 16, OUT = COLS + 16;
};
template <class T>
__global__ __launch_bounds__(1024) void k_quantize_turned(const T* x, long rows, long k, long col_stride, signed char* q, long ldq, float* scale) {
  using S = Turned<T>;
  constexpr int N = S::N;
  typedef T V __attribute__((ext_vector_type(N)));
  typedef T Loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  __shared__ __align__(16) char in[S::COLS * S::PITCH];
  __shared__ __align__(16) signed char out[S::ROWS * S::OUT];
  __shared__ unsigned most[S::ROWS];
  const long r0 = group_id() * S::ROWS;
  if (r0 >= rows) return;
  const int a = threadIdx.x % S::ACROSS, c0 = threadIdx.x / S::ACROSS;
  const int left = (int)min(rows - r0 - a * N, (long)N);
  auto piece = [&](long c) {
    V v = {};
    if (c >= k) return v;
    const T* from = x + c * col_stride + r0 + a * N;
    if (left == N) {
      v = *(const Loose*)from;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < left) v[e] = from[e];
    }
    return v;
  };
  if (threadIdx.x < S::ROWS) most[threadIdx.x] = 0;
  unsigned top[N] = {};
#pragma unroll 4
  for (long c = c0; c < k; c += S::COLS) {
    const V v = piece(c);
#pragma unroll
    for (int e = 0; e < N; ++e) top[e] = max(top[e], __float_as_uint(to_f32(v[e])) & 0x7fffffffu);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < N; ++e) {
#pragma unroll
    for (int o = S::ACROSS; o < 64; o *= 2) top[e] = max(top[e], (unsigned)__shfl_xor((int)top[e], o));
    if ((threadIdx.x & 63) < S::ACROSS) atomicMax(&most[a * N + e], top[e]);
  }
  __syncthreads();
  const int row = threadIdx.x % S::ROWS, group = threadIdx.x / S::ROWS;
  const RowScale s = row_scale(most[row]);
  if (group == 0 && r0 + row < rows) scale[r0 + row] = s.top / 127.0f;
  V next = piece(c0);
  for (long cb = 0; cb < ldq; cb += S::COLS) {
    *(V*)(in + c0 * S::PITCH + a * 16) = next;
    __syncthreads();
    if (cb + S::COLS < ldq) next = piece(cb + S::COLS + c0);
#pragma unroll
    for (int g = 0; g < S::COLS; g += 128) {
      const int c = g + 4 * group;
      float f[4];
      unsigned b[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = to_f32(*(const T*)(in + (c + e) * S::PITCH + row * sizeof(T)));
      quantise<4>(f, s, b);
      *(unsigned*)(out + row * S::OUT + c) = b[0];
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (t < S::ROWS * (S::COLS / 16)) {
      const int orow = t / (S::COLS / 16), c = t % (S::COLS / 16) * 16;
      if (r0 + orow < rows && cb + c < ldq) *(i32x4*)(q + (r0 + orow) * ldq + cb + c) = *(const i32x4*)(out + orow * S::OUT + c);
    }
  }
}

// n (up to 16) bytes from anywhere, the others zero
typedef int i32x4_loose __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ i32x4 loose_bytes(const signed char* p, int n) {
  if (n >= 16) return *(const i32x4_loose*)p;
  i32x4 v = {};
#pragma unroll
  for (int e = 0; e < 15; ++e)
    if (e < n) v[e >> 2] |= (int)((unsigned)(unsigned char)p[e] << (8 * (e & 3)));
  return v;
}
// Rows of 8-bit numbers that do not start at multiples of 16 bytes, laid out again so that they do (padding: zeros): one or two matrices a launch.
struct AlignRows {
  const signed char* x;
  signed char* y;
  long rows, ld;
};
__global__ __launch_bounds__(256) void k_align_rows(AlignRows a, AlignRows b, long k, long ldy) {
  const AlignRows g = blockIdx.y ? b : a;
  const long per = ldy / 16;
  for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < g.rows * per; t += (long)gridDim.x * 256) {
    const long r = t / per, c = (t - r * per) * 16;
    *(i32x4*)(g.y + r * ldy + c) = loose_bytes(g.x + r * g.ld + c, (int)min(k - c, 16l));
  }
}

// ---- products ----------------------------------------------------------------------------------------------------------------------------
struct Int8Args {
  Operand a, b;  // rows m and n
  const float *a_scale, *b_scale;
  const void* bias;
  int bias_type;
  int m, n, k;
  void* y;
};

template <class T>
__device__ __forceinline__ float bias_at(const Int8Args& g, int n) {
  if (!g.bias) return 0.0f;
  return g.bias_type == 0 ? ((const float*)g.bias)[n] : to_f32(((const T*)g.bias)[n]);
}
// (sum * a_scale) * b_scale, left to right: the product of the two scales alone may fall below the smallest float.
__device__ __forceinline__ float scaled(int sum, float as, float bs, float bias) { return (float)sum * as * bs + bias; }

// Many rows: P = b (its rows lie along a chunk's words, as neighbours in a row of y), Q = a.
// A thread writes 16 bytes of a row of y at once, wherever the row starts (a store may begin at any element), and has the same channels in all its rows.
template <class T, class TL, int BI, int BJ>
__global__ __launch_bounds__(TL::THREADS) void k_int8_tile(Int8Args g, int ti, int tj, int strip) {
  constexpr int N = 16 / (int)sizeof(T);
  extern __shared__ char lds[];
  int bi, bj;
  strip_order(die_order(blockIdx.x, ti * tj), ti, tj, strip, &bi, &bj);
  const int i0 = bi * BI, j0 = bj * BJ;
  // What the epilogue needs is on its way before the product begins: a_scale to LDS behind the tile, b_scale and the bias to registers.
  constexpr int ACROSS = TL::W / N, STEP = TL::TEAM / ACROSS, TURNS = TL::ROWS / STEP;
  static_assert(STEP * ACROSS == TL::TEAM && TURNS * STEP == TL::ROWS, "chunks must divide over the threads");
  float* a_scale = (float*)(lds + tile_bytes<TL>());
  for (int r = threadIdx.x; r < BJ; r += TL::THREADS) a_scale[r] = g.a_scale[min(j0 + r, g.m - 1)];
  const int iw = TL::who() % ACROSS * N, n = i0 + TL::row0() + iw, left = g.n - n;
  float bs[N], bias[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    bs[e] = e < left ? g.b_scale[n + e] : 0.0f;
    bias[e] = e < left ? bias_at<T>(g, n + e) : 0.0f;
  }
  TL t;
  const int steps = (g.k + 127) / 128;
  t.run(g.b, i0, g.a, j0, steps, g.k - (steps - 1) * 128, lds);
  T* y = (T*)g.y;
  char* mine = TL::part(lds);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < TL::CHUNKS; ++c) {
    t.spill(c, mine);
#pragma unroll 4
    for (int u = 0; u < TURNS; ++u) {
      const int r = TL::who() / ACROSS + u * STEP, j = TL::column0(c) + r, m = j0 + j;
      if (m >= g.m || left <= 0) continue;
      int s[N];
      chunk_sums<TL, N>(mine, r, iw, s);
      const float as = a_scale[j];
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = scaled(s[e], as, bs[e], bias[e]);
      store_some<T, N>(y + (size_t)m * g.n + n, v, left);
    }
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// Up to 64 rows of a against all of b: bound by reading b once.  A workgroup takes 16 NG rows of b; its eight waves deal the K range out among
// themselves in pairs of 64 bytes (a wave reads 128 bytes of 16 rows: whole lines) straight into the fragments of the 16 x 16 x 64 instruction,
// U loads under way before the first is used, and add their sums up in LDS - integers, so the order does not matter.  No second launch, no scratch memory.
// a comes from L2 for every workgroup: MG fragments for NG of b.  Rows of a and b may start anywhere (a load may); a last chunk is read byte by byte where
// the bytes behind it may not be there.
// FUSED: a is not there yet - the workgroup quantises the rows of x into LDS itself while the first reads of b are under way (rows, k as the caller
// allows them: see the host code).
constexpr int FEW_U = 8;

struct FewX {
  const void* x;  // FUSED: the rows to quantise
  long row_stride, col_stride;
  int vec;
  int a_padded, b_padded;  // a row's last chunk may be read whole
};

constexpr int FEW_ROWS = 4;  // FUSED: at most

// All 512 threads share a row: the piece of eight elements number threadIdx.x, + 512, ..; the rows' reads are under way together, and the first piece
// stays in registers between the maximum and the rounding.
template <class TX>
__device__ __forceinline__ void few_quantise(const Int8Args& g, const FewX& f, signed char* rows, long ld, float* scales, unsigned* parts) {
  typedef TX V __attribute__((ext_vector_type(8)));
  typedef TX Loose __attribute__((ext_vector_type(8), aligned(sizeof(TX))));
  const int w = threadIdx.x >> 6, c0 = 8 * threadIdx.x;
  auto piece = [&](int m, int c) {
    const TX* x = (const TX*)f.x + m * f.row_stride;
    V v = {};
    if (f.vec && c + 8 <= g.k) {
      v = *(const Loose*)(x + c);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < g.k) v[e] = x[(c + e) * f.col_stride];
    }
    return v;
  };
  V held[FEW_ROWS];
#pragma unroll
  for (int m = 0; m < FEW_ROWS; ++m)
    if (m < g.m) held[m] = piece(m, c0);
#pragma unroll
  for (int m = 0; m < FEW_ROWS; ++m)
    if (m < g.m) {
      unsigned top = most_bits<TX, 8>(held[m], 0);
      for (int c = c0 + 8 * 512; c < g.k; c += 8 * 512) top = most_bits<TX, 8>(piece(m, c), top);
      top = wave_most<TX>(top);
      if ((threadIdx.x & 63) == 0) parts[m * 8 + w] = top;
    }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < FEW_ROWS; ++m)
    if (m < g.m) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, parts[m * 8 + i]);
      const RowScale s = row_scale(top);
      if (threadIdx.x == 0) scales[m] = s.top / 127.0f;
      if (c0 < ld - 16) quantise_store<8>(held[m], s, rows + m * ld + c0);
      for (int c = c0 + 8 * 512; c < ld - 16; c += 8 * 512) quantise_store<8>(piece(m, c), s, rows + m * ld + c);
    }
  __syncthreads();
}

template <class T, int MG, int NG, bool FUSED>
__global__ __launch_bounds__(512) void k_int8_few(Int8Args g, FewX f) {
  extern __shared__ char lds[];
  const int l = (int)(threadIdx.x & 63), w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int row = l & 15, quarter = l >> 4;
  if (group_id() * 16 * NG >= g.n) return;
  const int n0 = (int)group_id() * 16 * NG;
  const int blocks = (g.k + 63) / 64;
  const char* pb[NG];
#pragma unroll
  for (int j = 0; j < NG; ++j) pb[j] = g.b.base + (size_t)min(n0 + 16 * j + row, g.n - 1) * g.b.ld + quarter * 16;
  // FUSED: rows of the LDS copy are 64 bytes of every block and 16 more apart (the 16 rows of a fragment then start in different banks)
  const long ldf = (long)blocks * 64 + 16;
  signed char* rows = (signed char*)lds;
  float* scales = (float*)(lds + (FUSED ? g.m * ldf : 0));
  unsigned* parts = (unsigned*)(scales + 16);
  const char* pa[MG];
#pragma unroll
  for (int i = 0; i < MG; ++i) {
    const int m = min(16 * i + row, g.m - 1);
    pa[i] = FUSED ? (const char*)rows + m * ldf + quarter * 16 : g.a.base + (size_t)m * g.a.ld + quarter * 16;
  }
  i32x4 acc[MG][NG];
#pragma unroll
  for (int i = 0; i < MG; ++i)
#pragma unroll
    for (int j = 0; j < NG; ++j) acc[i][j] = i32x4{};

  // block u of round s: the wave's pairs are s * U / 2 + u / 2, dealt out over the waves.  All of a round's reads, of a too, are under way together;
  // blocks past the end are zeros of b.
  const int whole = g.k / 64, rounds = (whole + 8 * FEW_U - 1) / (8 * FEW_U);
  auto block_of = [&](int s, int u) { return ((s * (FEW_U / 2) + u / 2) * 8 + w) * 2 + (u & 1); };
  auto load_b = [&](int s, i32x4 (&v)[FEW_U][NG]) {
#pragma unroll
    for (int u = 0; u < FEW_U; ++u) {
      const int b = block_of(s, u);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        v[u][j] = i32x4{};
        if (b < whole) v[u][j] = *(const i32x4_loose*)(pb[j] + (size_t)b * 64);
      }
    }
  };
  auto load_a = [&](int s, i32x4 (&v)[FEW_U][MG]) {
#pragma unroll
    for (int u = 0; u < FEW_U; ++u) {
      const int b = block_of(s, u);
      if (b < whole)
#pragma unroll
        for (int i = 0; i < MG; ++i) v[u][i] = *(const i32x4_loose*)(pa[i] + (size_t)b * 64);
    }
  };
  i32x4 v[FEW_U][NG], a[FEW_U][MG] = {};
  load_b(0, v);
  if constexpr (FUSED) few_quantise<T>(g, f, rows, ldf, scales, parts);
  for (int s = 0; s < rounds;) {
    load_a(s, a);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < FEW_U; ++u)
#pragma unroll
      for (int i = 0; i < MG; ++i)
#pragma unroll
        for (int j = 0; j < NG; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[u][j], a[u][i], acc[i][j], 0, 0, 0);
    if (++s < rounds) load_b(s, v);
  }
  if (whole < blocks && w == whole % 8) {  // the ragged block
    const int left = g.k - whole * 64 - quarter * 16;  // bytes of the lane's chunk
    auto chunk = [&](const char* row, int padded) {
      const signed char* p = (const signed char*)row + (size_t)whole * 64;
      return left <= 0 ? i32x4{} : keep_bytes(left >= 16 || padded ? (i32x4)(*(const i32x4_loose*)p) : loose_bytes(p, left), left);
    };
    i32x4 at[MG];
#pragma unroll
    for (int i = 0; i < MG; ++i) at[i] = chunk(pa[i], FUSED || f.a_padded);
#pragma unroll 1
    for (int j = 0; j < NG; ++j) {
      const i32x4 bt = chunk(j ? pb[NG - 1] : pb[0], f.b_padded);
#pragma unroll
      for (int i = 0; i < MG; ++i) {
        if (j == 0) acc[i][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bt, at[i], acc[i][0], 0, 0, 0);
        if (NG > 1 && j == 1) acc[i][NG - 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bt, at[i], acc[i][NG - 1], 0, 0, 0);
      }
    }
  }

  __syncthreads();  // (FUSED: the rows are read no more)
  i32x4* red = (i32x4*)(lds + (FUSED ? (g.m * ldf + 64 + 512 + 255) / 256 * 256 : 0));
#pragma unroll
  for (int i = 0; i < MG; ++i)
#pragma unroll
    for (int j = 0; j < NG; ++j) red[(w * MG * NG + i * NG + j) * 64 + l] = acc[i][j];
  __syncthreads();
  T* y = (T*)g.y;
  for (int t = threadIdx.x; t < MG * NG * 64; t += 512) {
    i32x4 sum = red[t];
#pragma unroll
    for (int o = 1; o < 8; ++o) sum += red[o * MG * NG * 64 + t];
    const int lane = t & 63, j = (t >> 6) % NG, i = (t >> 6) / NG;
    const int m = 16 * i + (lane & 15), n = n0 + 16 * j + 4 * (lane >> 4);
    if (m >= g.m) continue;
    const float as = FUSED ? scales[m] : g.a_scale[m];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < g.n) y[(size_t)m * g.n + n + e] = (T)scaled(sum[e], as, g.b_scale[n + e], bias_at<T>(g, n + e));
  }
}

}  // namespace lb
