// Matrix-core tile engine of the few-bit operators (nls_lowbit.hip): D[i][j] = sum_k P[i][k] Q[j][k], both operands row-major with k running
// along the row, in 8-bit integers, in fp16, or in fp16 pairs (hi + lo).
//
// One K step is 128 bytes of every operand row, whatever the type: 128 int8, 64 fp16, or 32 fp16 pairs (a row holds granules of 64 bytes hi and
// 64 bytes lo per 32 elements).  The rows travel from memory to LDS without touching registers (16 bytes a lane, a wave moves 8 whole rows =
// eight full 128-byte lines), into the other half of a double buffer while the matrix cores work on this half.
//
// LDS holds a tile row at r * 128, its 16-byte chunk c at slot c ^ (r & 7): a fragment read takes the same chunk of 32 rows, so any 8 neighbouring
// lanes touch 8 different slots - every bank once.  The writing side needs no scatter: the lane that fills slot s simply fetches chunk s ^ (r & 7).
//
// Rows past the end of an operand are fetched from its last row instead (their products land in outputs nobody stores), chunks past the end of the
// K range from the start of the step, so that no access leaves the operand; what they hold is masked to zero in ONE operand's registers.
#pragma once
#include <hip/hip_runtime.h>

namespace lb {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

enum Mode { MODE_I8 = 0, MODE_F16 = 1, MODE_F16PAIR = 2 };

template <int MODE>
struct AccOf {
  using type = f32x16;
};
template <>
struct AccOf<MODE_I8> {
  using type = i32x16;
};

// Bytes an operand row advances per K step.
template <int MODE>
constexpr int kstep_bytes() {
  return MODE == MODE_F16 ? 256 : 128;
}
// Byte offset, within a K step, of 16-byte chunk c: fp16 alone reads the hi half of two granules.
template <int MODE>
__device__ __forceinline__ unsigned chunk_offset(int c) {
  return MODE == MODE_F16 ? (unsigned)((c >> 2) * 128 + (c & 3) * 16) : (unsigned)(c * 16);
}

struct Operand {
  const char* base;  // 16-byte aligned
  unsigned ld;       // bytes from row to row, a multiple of 16
  int rows;
};

template <int MODE, int BI, int BJ, int WI, int WJ>
struct Tile {
  static constexpr int WAVES = WI * WJ;
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int MI = BI / WI / 32;  // 32 x 32 blocks of a wave
  static constexpr int MJ = BJ / WJ / 32;
  static constexpr int LOADS_P = BI / 8 / WAVES;  // 8-row moves a wave makes per step
  static constexpr int LOADS_Q = BJ / 8 / WAVES;
  static constexpr int BUF = (BI + BJ) * 128;
  static constexpr int LDS = 2 * BUF;
  static_assert(LOADS_P * 8 * WAVES == BI && LOADS_Q * 8 * WAVES == BJ && LOADS_P > 0 && LOADS_Q > 0, "tile rows must divide over the waves");
  static_assert(MI * WI * 32 == BI && MJ * WJ * 32 == BJ, "tile must divide over the waves");
  using Acc = typename AccOf<MODE>::type;

  Acc acc[MI][MJ];
  unsigned offp[LOADS_P], offq[LOADS_Q];

  __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
  __device__ __forceinline__ static int lane() { return (int)(threadIdx.x & 63); }

  __device__ __forceinline__ static void move(const char* base, unsigned off, char* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + off), (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
  }
  // The lane's place: row (lane >> 3) of the move, slot (lane & 7), hence chunk slot ^ (row & 7); moves start at multiples of 8 rows.
  __device__ __forceinline__ static int my_chunk() { return (lane() & 7) ^ ((lane() >> 3) & 7); }

  __device__ __forceinline__ void start(const Operand& P, int i0, const Operand& Q, int j0) {
    const int r = wave() * 8 + (lane() >> 3);
    const unsigned c = chunk_offset<MODE>(my_chunk());
#pragma unroll
    for (int l = 0; l < LOADS_P; ++l) offp[l] = (unsigned)min(l * 8 * WAVES + r, P.rows - 1 - i0) * P.ld + c;
#pragma unroll
    for (int l = 0; l < LOADS_Q; ++l) offq[l] = (unsigned)min(l * 8 * WAVES + r, Q.rows - 1 - j0) * Q.ld + c;
#pragma unroll
    for (int a = 0; a < MI; ++a)
#pragma unroll
      for (int b = 0; b < MJ; ++b) acc[a][b] = Acc{};
  }
  // valid: bytes of the step that exist (>= 128: all); only 8-bit operands have ragged ends, fp16 operands are padded to whole steps
  __device__ __forceinline__ void fetch(const char* p, const char* q, char* buf, int valid) const {
    const int w = wave();
    unsigned back = 0;
    if (MODE == MODE_I8 && valid < 128) back = my_chunk() * 16 >= valid ? (unsigned)my_chunk() * 16 : 0u;
#pragma unroll
    for (int l = 0; l < LOADS_P; ++l) move(p, offp[l] - back, buf + (l * WAVES + w) * 1024);
#pragma unroll
    for (int l = 0; l < LOADS_Q; ++l) move(q, offq[l] - back, buf + BI * 128 + (l * WAVES + w) * 1024);
  }
  __device__ __forceinline__ static i32x4 mask_bytes(i32x4 v, int n) {  // keep the first n of 16 bytes
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int b = n - 4 * w;
      v[w] = b >= 4 ? v[w] : b <= 0 ? 0 : (v[w] & ((1 << (8 * b)) - 1));
    }
    return v;
  }
  template <bool TAIL>
  __device__ __forceinline__ void multiply(const char* buf, int valid) {
    const int w = wave(), l = lane();
    const int wi = w / WJ, wj = w % WJ;
    const char* p = buf + (wi * MI * 32 + (l & 31)) * 128;
    const char* q = buf + BI * 128 + (wj * MJ * 32 + (l & 31)) * 128;
    const int x = l & 7, h = l >> 5;
    if constexpr (MODE == MODE_F16PAIR) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int hi = ((2 * s + h) ^ x) * 16, lo = ((4 + 2 * s + h) ^ x) * 16;
        f16x8 ph[MI], pl[MI], qh[MJ], ql[MJ];
#pragma unroll
        for (int a = 0; a < MI; ++a) ph[a] = *(const f16x8*)(p + a * 4096 + hi);
#pragma unroll
        for (int b = 0; b < MJ; ++b) qh[b] = *(const f16x8*)(q + b * 4096 + hi);
#pragma unroll
        for (int a = 0; a < MI; ++a) pl[a] = *(const f16x8*)(p + a * 4096 + lo);
#pragma unroll
        for (int b = 0; b < MJ; ++b) ql[b] = *(const f16x8*)(q + b * 4096 + lo);
#pragma unroll
        for (int a = 0; a < MI; ++a)
#pragma unroll
          for (int b = 0; b < MJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[a], qh[b], acc[a][b], 0, 0, 0);
#pragma unroll
        for (int a = 0; a < MI; ++a)
#pragma unroll
          for (int b = 0; b < MJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[a], qh[b], acc[a][b], 0, 0, 0);
#pragma unroll
        for (int a = 0; a < MI; ++a)
#pragma unroll
          for (int b = 0; b < MJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[a], ql[b], acc[a][b], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int c = ((2 * s + h) ^ x) * 16;
        if constexpr (MODE == MODE_I8) {
          i32x4 pf[MI], qf[MJ];
#pragma unroll
          for (int a = 0; a < MI; ++a) pf[a] = *(const i32x4*)(p + a * 4096 + c);
#pragma unroll
          for (int b = 0; b < MJ; ++b) {
            qf[b] = *(const i32x4*)(q + b * 4096 + c);
            if (TAIL) qf[b] = mask_bytes(qf[b], valid - (2 * s + h) * 16);
          }
#pragma unroll
          for (int a = 0; a < MI; ++a)
#pragma unroll
            for (int b = 0; b < MJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(pf[a], qf[b], acc[a][b], 0, 0, 0);
        } else {
          f16x8 pf[MI], qf[MJ];
#pragma unroll
          for (int a = 0; a < MI; ++a) pf[a] = *(const f16x8*)(p + a * 4096 + c);
#pragma unroll
          for (int b = 0; b < MJ; ++b) qf[b] = *(const f16x8*)(q + b * 4096 + c);
#pragma unroll
          for (int a = 0; a < MI; ++a)
#pragma unroll
            for (int b = 0; b < MJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pf[a], qf[b], acc[a][b], 0, 0, 0);
        }
      }
    }
  }
  // steps >= 1 whole or ragged K steps from byte kb of the rows on; ragged: valid bytes of the last one (128: whole).
  __device__ __forceinline__ void run(const Operand& P, int i0, const Operand& Q, int j0, size_t kb, int steps, int last_valid, char* lds) {
    start(P, i0, Q, j0);
    const char* p = P.base + (size_t)i0 * P.ld + kb;
    const char* q = Q.base + (size_t)j0 * Q.ld + kb;
    constexpr int STEP = kstep_bytes<MODE>();
    fetch(p, q, lds, steps == 1 ? last_valid : 128);
    for (int t = 0; t < steps - 1; ++t) {
      __syncthreads();  // step t has arrived (the barrier drains the moves), step t - 1 has been read
      p += STEP;
      q += STEP;
      fetch(p, q, lds + ((t + 1) & 1) * BUF, t + 2 == steps ? last_valid : 128);
      multiply<false>(lds + (t & 1) * BUF, 128);
    }
    __syncthreads();
    if (MODE == MODE_I8 && last_valid < 128)
      multiply<true>(lds + ((steps - 1) & 1) * BUF, last_valid);
    else
      multiply<false>(lds + ((steps - 1) & 1) * BUF, 128);
  }
  // Where register r (0 .. 15) of block (a, b) lies in the tile: i = row_of(a) + 8 (r / 4) + r % 4, j = col_of(b).
  __device__ __forceinline__ static int row_of(int a) { return (wave() / WJ * MI + a) * 32 + 4 * (lane() >> 5); }
  __device__ __forceinline__ static int col_of(int b) { return (wave() % WJ * MJ + b) * 32 + (lane() & 31); }
};

// Tiles in an order that keeps the ones a die works on together: workgroups are dealt to the 8 dies in turn, so die x takes the x-th eighth of the
// list (bijective for any count), and the list walks strips of `strip` tile rows, so that a die's tiles share operand rows in its L2.
__device__ __forceinline__ int die_order(int id, int total) {
  const int q = total >> 3, r = total & 7, x = id & 7;
  return x * q + min(x, r) + (id >> 3);
}
__device__ __forceinline__ void strip_order(int t, int ti, int tj, int strip, int* i, int* j) {
  const int per = strip * tj;
  const int s = t / per, first = s * strip, h = min(strip, ti - first);
  const int u = t - s * per;
  *i = first + u % h;
  *j = u / h;
}

// ---- element types ----------------------------------------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}
template <class T>
struct Vec4;
template <>
struct Vec4<float> {
  using type = f32x4;
};
template <>
struct Vec4<_Float16> {
  using type = f16x4;
};
template <>
struct Vec4<__bf16> {
  using type = bf16x4;
};

}  // namespace lb
