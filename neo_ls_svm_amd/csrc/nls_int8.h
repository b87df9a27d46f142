// 8-bit rows and their products: quantisation, the product of few rows (bound by reading b), the product of many rows (matrix cores).
#pragma once
#include "nls_tile.h"

namespace lb {

// ---- quantise rows --------------------------------------------------------------------------------------------------------------------------
// scale = max|x| / 127, q = 127 x / max|x| to the nearest integer, ties to even, decided as if in exact arithmetic:
// r = x * inv with inv = fl(127 / max|x|) is off by less than 127 * 2^-23 + (its own rounding) < 2^-15.9; only where r lies that near to a half is
// the quotient formed in 64 bits - 127 x is exact there and a quotient of a 31-bit by a 24-bit number that is no half is at least 2^-26 away from one.
// A row with a NaN or an infinity gets that as its scale and zeros as q (the product then gives NaN in the whole row); a row of zeros, scale 0.
__device__ __forceinline__ int quantise_exact(float x, float top) {
  return (int)__builtin_rint((double)x * 127.0 / (double)top);
}
__device__ __forceinline__ int quantise_one(float x, float top, float inv) {
  const float r = x * inv;
  const float n = __builtin_rintf(r);
  if (__builtin_expect(fabsf(fabsf(r - n) - 0.5f) < 2.0e-5f, 0)) return quantise_exact(x, top);
  return (int)n;
}
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
__device__ __forceinline__ int quantise(float x, const RowScale& s) {
  return s.kind == 0 ? quantise_one(x, s.top, s.inv) : s.kind == 1 ? quantise_exact(x, s.top) : 0;
}
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }  // orders |x|, infinity, NaN
__device__ __forceinline__ unsigned pack4(int a, int b, int c, int d) {
  return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)d << 24;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
  return v;
}

// A group of G threads takes a row; four neighbouring elements a thread and turn.  VEC: the row starts are aligned to four elements.
template <class T, int G, bool VEC>
__global__ __launch_bounds__(256) void k_quantize_rows(const T* x, long rows, long k, long row_stride, long col_stride, signed char* q, long ldq,
                                                       float* scale) {
  using V = typename Vec4<T>::type;
  const int g = threadIdx.x % G;
  const long row = (long)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row < rows;
  const T* xr = x + (live ? row : rows - 1) * row_stride;
  unsigned top = 0;
  for (long c = 4 * g; c < k; c += 4 * G) {
    if (VEC && c + 4 <= k) {
      const V v = *(const V*)(xr + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, magnitude(to_f32(v[e])));
    } else {
      for (int e = 0; e < 4 && c + e < k; ++e) top = max(top, magnitude(to_f32(xr[(c + e) * col_stride])));
    }
  }
  top = wave_max(top);
  if (G > 64) {
    __shared__ unsigned part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  if (!live) return;
  const RowScale s = row_scale(top);
  if (g == 0) scale[row] = s.top / 127.0f;
  signed char* qr = q + row * ldq;
  for (long c = 4 * g; c < ldq; c += 4 * G) {  // the row's padding is written as zeros
    int v[4];
    for (int e = 0; e < 4; ++e) v[e] = c + e < k ? quantise(to_f32(xr[(c + e) * col_stride]), s) : 0;
    *(unsigned*)(qr + c) = pack4(v[0], v[1], v[2], v[3]);
  }
}

// Rows of 8-bit numbers that do not start at multiples of 16 bytes, laid out again so that they do (padding: zeros).
__global__ __launch_bounds__(256) void k_align_rows(const signed char* x, long rows, long k, long ld, signed char* y, long ldy) {
  const long per = ldy / 4;
  for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < rows * per; t += (long)gridDim.x * 256) {
    const long r = t / per, c = (t - r * per) * 4;
    int v[4];
    for (int e = 0; e < 4; ++e) v[e] = c + e < k ? x[r * ld + c + e] : 0;
    *(unsigned*)(y + r * ldy + c) = pack4(v[0], v[1], v[2], v[3]);
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

// Many rows: P = b (its rows run along a lane's four consecutive registers, which are four neighbours of an output row), Q = a.
template <class T, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(64 * WI * WJ) void k_int8_tile(Int8Args g, int ti, int tj, int strip) {
  using TL = Tile<MODE_I8, BI, BJ, WI, WJ>;
  extern __shared__ char lds[];
  int bi, bj;
  strip_order(die_order(blockIdx.x, ti * tj), ti, tj, strip, &bi, &bj);
  const int i0 = bi * BI, j0 = bj * BJ;
  TL t;
  const int steps = (g.k + 127) / 128;
  t.run(g.b, i0, g.a, j0, 0, steps, g.k - (steps - 1) * 128, lds);
  T* y = (T*)g.y;
  const bool vec = g.n % 4 == 0;
#pragma unroll
  for (int b = 0; b < TL::MJ; ++b) {
    const int m = j0 + TL::col_of(b);
    if (m >= g.m) continue;
    const float as = g.a_scale[m];
#pragma unroll
    for (int a = 0; a < TL::MI; ++a)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int n = i0 + TL::row_of(a) + 2 * r;
        if (vec && n < g.n) {
          typename Vec4<T>::type v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (T)scaled(t.acc[a][b][r + e], as, g.b_scale[n + e], bias_at<T>(g, n + e));
          *(typename Vec4<T>::type*)(y + (size_t)m * g.n + n) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < g.n) y[(size_t)m * g.n + n + e] = (T)scaled(t.acc[a][b][r + e], as, g.b_scale[n + e], bias_at<T>(g, n + e));
        }
      }
  }
}

}  // namespace lb
