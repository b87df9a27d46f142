// Matrix-core tile engine of the few-bit operators (nls_lowbit.hip): D[i][j] = sum_k P[i][k] Q[j][k], both operands row-major with k running
// along the row, in 8-bit integers or in fp16 pairs (hi + lo).
//
// One K step is 128 bytes of every operand row, one whole line, whatever the type: 128 int8, or 32 fp16 pairs (64 bytes hi, then 64 bytes lo).
// The rows travel from memory to LDS without touching registers (16 bytes a lane, a wave moves 8 whole rows = eight full lines), into the next of STAGES
// buffers while the matrix cores work on this one: the fewer workgroups share a compute unit, the more steps have to be under way to cover the way
// to memory.
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

enum Mode { MODE_I8 = 0, MODE_F16PAIR = 1 };

template <int MODE>
struct AccOf {
  using type = f32x16;
};
template <>
struct AccOf<MODE_I8> {
  using type = i32x16;
};

__device__ __forceinline__ size_t step_at(int t) { return (size_t)t * 128; }  // where K step t of an operand row begins

__device__ __forceinline__ i32x4 keep_bytes(i32x4 v, int n) {  // the first n of 16 bytes, the others zero
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int b = n - 4 * w;
    v[w] = b >= 4 ? v[w] : b <= 0 ? 0 : (v[w] & ((1 << (8 * b)) - 1));
  }
  return v;
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
__device__ __forceinline__ int lane_id() { return (int)(threadIdx.x & 63); }
// 16 bytes a lane from memory to LDS (lane after lane from `lds` on)
__device__ __forceinline__ void move16(const char* base, unsigned off, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + off), (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// A move takes 8 rows: the lane's row is lane >> 3, its slot lane & 7, hence its chunk slot ^ (row & 7); moves start at multiples of 8 rows.
__device__ __forceinline__ int move_chunk() { return (lane_id() & 7) ^ ((lane_id() >> 3) & 7); }
// Chunks past the valid bytes of a ragged step are fetched from its start instead: how far back the lane goes.
__device__ __forceinline__ unsigned move_back(int valid) { return move_chunk() * 16 >= valid ? (unsigned)move_chunk() * 16 : 0u; }

// Fragments of one K step for MI x MJ blocks, and their products.  p, q: the lane's row (lane & 31) of the first block; blocks are 4096 bytes apart.
template <int MODE, int MI, int MJ>
struct Frags {
  static constexpr int SUB = MODE == MODE_F16PAIR ? 2 : 4;  // instructions' worth of K in a step
  static constexpr int KINDS = MODE == MODE_F16PAIR ? 2 : 1;
  i32x4 p[SUB][KINDS][MI], q[SUB][KINDS][MJ];
  using Acc = typename AccOf<MODE>::type;

  template <bool TAIL>
  __device__ __forceinline__ void read(int s, const char* pr, const char* qr, int valid) {
    const int x = lane_id() & 7, h = lane_id() >> 5;
#pragma unroll
    for (int k = 0; k < KINDS; ++k) {
      const int c = ((4 * k * (MODE == MODE_F16PAIR) + 2 * s + h) ^ x) * 16;
#pragma unroll
      for (int a = 0; a < MI; ++a) p[s][k][a] = *(const i32x4*)(pr + a * 4096 + c);
#pragma unroll
      for (int b = 0; b < MJ; ++b) {
        q[s][k][b] = *(const i32x4*)(qr + b * 4096 + c);
        if (TAIL) q[s][k][b] = keep_bytes(q[s][k][b], valid - (2 * s + h) * 16);
      }
    }
  }
  __device__ __forceinline__ static Acc product(const i32x4& u, const i32x4& v, const Acc& c) {
    if constexpr (MODE == MODE_I8)
      return __builtin_amdgcn_mfma_i32_32x32x32_i8(u, v, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, u), __builtin_bit_cast(f16x8, v), c, 0, 0, 0);
  }
  __device__ __forceinline__ void multiply(int s, Acc (&acc)[MI][MJ]) const {
#pragma unroll
    for (int k = 0; k < (KINDS == 2 ? 3 : 1); ++k)  // pairs: hi hi, lo hi, hi lo
#pragma unroll
      for (int a = 0; a < MI; ++a)
#pragma unroll
        for (int b = 0; b < MJ; ++b) acc[a][b] = product(p[s][KINDS == 2 ? k == 1 : 0][a], q[s][KINDS == 2 ? k == 2 : 0][b], acc[a][b]);
  }
};

struct Operand {
  const char* base;  // 16-byte aligned
  unsigned ld;       // bytes from row to row, a multiple of 16
  int rows;
};

template <int MODE, int BI, int BJ, int WI, int WJ, int STAGES>
struct Tile {
  static constexpr int WAVES = WI * WJ;
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int MI = BI / WI / 32;  // 32 x 32 blocks of a wave
  static constexpr int MJ = BJ / WJ / 32;
  static constexpr int LOADS_P = BI / 8 / WAVES;  // 8-row moves a wave makes per step
  static constexpr int LOADS_Q = BJ / 8 / WAVES;
  static constexpr int BUF = (BI + BJ) * 128;
  static constexpr int LDS = STAGES * BUF;
  static constexpr int FLIGHT = (LOADS_P + LOADS_Q) * (STAGES - 2);  // moves of a wave that may still be under way when a step begins
  static_assert(STAGES >= 2 && FLIGHT <= 63, "the counter of moves under way ends at 63");
  static_assert(LOADS_P * 8 * WAVES == BI && LOADS_Q * 8 * WAVES == BJ && LOADS_P > 0 && LOADS_Q > 0, "tile rows must divide over the waves");
  static_assert(MI * WI * 32 == BI && MJ * WJ * 32 == BJ, "tile must divide over the waves");
  using Acc = typename AccOf<MODE>::type;

  Acc acc[MI][MJ];
  unsigned offp[LOADS_P], offq[LOADS_Q];

  __device__ __forceinline__ void start(const Operand& P, int i0, const Operand& Q, int j0) {
    const int r = wave_id() * 8 + (lane_id() >> 3);
    const unsigned c = move_chunk() * 16;
#pragma unroll
    for (int l = 0; l < LOADS_P; ++l) offp[l] = (unsigned)min(l * 8 * WAVES + r, P.rows - 1 - i0) * P.ld + c;
#pragma unroll
    for (int l = 0; l < LOADS_Q; ++l) offq[l] = (unsigned)min(l * 8 * WAVES + r, Q.rows - 1 - j0) * Q.ld + c;
#pragma unroll
    for (int a = 0; a < MI; ++a)
#pragma unroll
      for (int b = 0; b < MJ; ++b) acc[a][b] = Acc{};
  }
  // valid: bytes of the step that exist (>= 128: all); only 8-bit operands have ragged ends, pairs are padded to whole steps
  __device__ __forceinline__ void fetch(const char* p, const char* q, char* buf, int valid) const {
    const int w = wave_id();
    const unsigned back = MODE == MODE_I8 && valid < 128 ? move_back(valid) : 0;
#pragma unroll
    for (int l = 0; l < LOADS_P; ++l) move16(p, offp[l] - back, buf + (l * WAVES + w) * 1024);
#pragma unroll
    for (int l = 0; l < LOADS_Q; ++l) move16(q, offq[l] - back, buf + BI * 128 + (l * WAVES + w) * 1024);
  }
  template <bool TAIL>
  __device__ __forceinline__ void multiply(const char* buf, int valid) {
    const int wi = wave_id() / WJ, wj = wave_id() % WJ, l = lane_id();
    const char* p = buf + (wi * MI * 32 + (l & 31)) * 128;
    const char* q = buf + BI * 128 + (wj * MJ * 32 + (l & 31)) * 128;
    Frags<MODE, MI, MJ> f;
#pragma unroll
    for (int s = 0; s < f.SUB; ++s) {
      f.template read<TAIL>(s, p, q, valid);
      f.multiply(s, acc);
    }
  }
  // Every wave's share of the oldest step has arrived and every wave has read what the next move overwrites.
  template <int N>
  __device__ __forceinline__ static void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  }
  // 8-bit waves with many blocks have the first fragments of a step in registers when the last products of the step before begin: the reads behind the
  // barrier are then off the matrix cores' path.  (256 x 256, int8 8192^3: 464 us against 497, 8192 x 8192 x 2048 149 / 153, K = 512 69 / 66.)  A step of
  // pairs has three products a fragment to cover them: five steps of 4096^2 4.12 ms against 4.06 without, of 8192^2 34.5 / 34.0.
  static constexpr bool AHEAD = MODE == MODE_I8 && MI * MJ >= 8;
  // steps >= 1 K steps; last_valid: valid bytes of the last one (128: whole).
  // STAGES - 1 steps are under way at any time; one barrier a step: behind it the next step is there and a buffer that all have read is free.
  __device__ __forceinline__ void run(const Operand& P, int i0, const Operand& Q, int j0, int steps, int last_valid, char* lds) {
    start(P, i0, Q, j0);
    const char* p = P.base + (size_t)i0 * P.ld;
    const char* q = Q.base + (size_t)j0 * Q.ld;
    auto move = [&](int t, char* buf) { fetch(p + step_at(t), q + step_at(t), buf, t + 1 == steps ? last_valid : 128); };
    constexpr int FIRST = AHEAD ? STAGES : STAGES - 1;
    for (int t = 0; t < min(FIRST, steps); ++t) move(t, lds + t * BUF);
    int now = 0;
    if constexpr (AHEAD) {
      const int wi = wave_id() / WJ, wj = wave_id() % WJ, l = lane_id();
      const int at_p = (wi * MI * 32 + (l & 31)) * 128, at_q = BI * 128 + (wj * MJ * 32 + (l & 31)) * 128;
      if (steps >= STAGES)
        arrive<FLIGHT + LOADS_P + LOADS_Q>();
      else
        arrive<0>();
      Frags<MODE, MI, MJ> f;
      f.template read<false>(0, lds + at_p, lds + at_q, 128);
      for (int t = 0; t < steps - 1; ++t) {
        const int next = now + BUF == LDS ? 0 : now + BUF;
#pragma unroll
        for (int s = 0; s < f.SUB; ++s) {
          if (s + 1 < f.SUB) {
            f.template read<false>(s + 1, lds + now + at_p, lds + now + at_q, 128);
          } else {  // all of step t is in registers
            if (t + STAGES <= steps)
              arrive<FLIGHT>();
            else
              arrive<0>();
            if (t + STAGES < steps) move(t + STAGES, lds + now);
            f.template read<false>(0, lds + next + at_p, lds + next + at_q, 128);
          }
          __builtin_amdgcn_sched_barrier(0);
          f.multiply(s, acc);
        }
        now = next;
      }
    } else {
      int next = (STAGES - 1) * BUF;
      for (int t = 0; t < steps - 1; ++t) {
        if (t + STAGES - 1 <= steps)
          arrive<FLIGHT>();
        else
          arrive<0>();
        if (t + STAGES - 1 < steps) move(t + STAGES - 1, lds + next);
        multiply<false>(lds + now, 128);
        now = now + BUF == LDS ? 0 : now + BUF;
        next = next + BUF == LDS ? 0 : next + BUF;
      }
      arrive<0>();
    }
    multiply<MODE == MODE_I8>(lds + now, last_valid);  // (masked whether ragged or not: two ways to the accumulators' end would double their registers)
  }
  // The epilogue goes through LDS, every wave for itself: column block c of its results, ROWS columns of the tile as rows of W words (i along the row)
  // that its 64 lanes read as whole lines.  No barriers but the one in front: the waves' parts overlie the tile's buffers.
  static constexpr int TEAM = 64, ROWS = 32, CHUNKS = MJ, PARTS = 1, W = 32 * MI, PITCH = W + 4;
  static constexpr int SCRATCH = WAVES * ROWS * PITCH * 4;
  __device__ __forceinline__ static int who() { return lane_id(); }
  __device__ __forceinline__ static char* part(char* lds) { return lds + wave_id() * (ROWS * PITCH * 4); }
  __device__ __forceinline__ static int row0() { return wave_id() / WJ * W; }
  __device__ __forceinline__ static int column0(int c) { return (wave_id() % WJ * MJ + c) * 32; }
  __device__ __forceinline__ static void settle() {  // what the wave wrote is there for the wave (LDS keeps a wave's order; the compiler has to as well)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __device__ __forceinline__ void spill(int c, char* mine) const {  // (c picks registers: unrolled by the callers)
    const int l = lane_id();
    int* t = (int*)mine + (l & 31) * PITCH + 4 * (l >> 5);
    settle();
#pragma unroll
    for (int b = 0; b < MJ; ++b)
      if (b == c)
#pragma unroll
        for (int a = 0; a < MI; ++a) {
          const i32x16 v = __builtin_bit_cast(i32x16, acc[a][b]);
#pragma unroll
          for (int r = 0; r < 16; r += 4) *(i32x4*)(t + a * 32 + 2 * r) = i32x4{v[r], v[r + 1], v[r + 2], v[r + 3]};
        }
    settle();
  }
};

// 64 x 64 tiles for products with few of them: each of the four waves has the whole tile and every fourth K step, in buffers of its own - no barriers,
// four independent accumulators a wave, half the LDS reads per product of four waves side by side - and the epilogue adds the four up.
template <int MODE, int STAGES>
struct Ring {
  static constexpr int THREADS = 256;
  static constexpr int BUF = 128 * 128;
  static constexpr int LDS = 4 * STAGES * BUF;
  using Acc = typename AccOf<MODE>::type;
  Acc acc[2][2];
  unsigned offp[8], offq[8];

  __device__ __forceinline__ void fetch(const char* p, const char* q, char* buf, int valid) const {
    const unsigned back = MODE == MODE_I8 && valid < 128 ? move_back(valid) : 0;
#pragma unroll
    for (int l = 0; l < 8; ++l) move16(p, offp[l] - back, buf + l * 1024);
#pragma unroll
    for (int l = 0; l < 8; ++l) move16(q, offq[l] - back, buf + 8192 + l * 1024);
  }
  template <bool TAIL>
  __device__ __forceinline__ void read(Frags<MODE, 2, 2>& f, const char* buf, int valid) const {
#pragma unroll
    for (int s = 0; s < f.SUB; ++s) f.template read<TAIL>(s, buf + (lane_id() & 31) * 128, buf + 8192 + (lane_id() & 31) * 128, valid);
  }
  __device__ __forceinline__ void run(const Operand& P, int i0, const Operand& Q, int j0, int steps, int last_valid, char* lds) {
    const int w = wave_id(), r = lane_id() >> 3;
    const unsigned c = move_chunk() * 16;
#pragma unroll
    for (int l = 0; l < 8; ++l) {
      offp[l] = (unsigned)min(l * 8 + r, P.rows - 1 - i0) * P.ld + c;
      offq[l] = (unsigned)min(l * 8 + r, Q.rows - 1 - j0) * Q.ld + c;
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b) acc[a][b] = Acc{};
    const char* p = P.base + (size_t)i0 * P.ld;
    const char* q = Q.base + (size_t)j0 * Q.ld;
    lds += w * STAGES * BUF;
    const int mine = (steps - w + 3) / 4;  // steps w, w + 4, ..
    auto valid_of = [&](int t) { return 4 * t + w + 1 == steps ? last_valid : 128; };
    for (int t = 0; t < min(STAGES, mine); ++t) fetch(p + step_at(4 * t + w), q + step_at(4 * t + w), lds + t * BUF, valid_of(t));
    int now = 0;
    for (int t = 0; t < mine; ++t) {
      if (t + STAGES <= mine)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(16 * (STAGES - 1)) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      Frags<MODE, 2, 2> f;
      if (MODE == MODE_I8 && valid_of(t) < 128)
        read<true>(f, lds + now, last_valid);
      else
        read<false>(f, lds + now, 128);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the step is in registers, its buffer free
      const int ahead = t + STAGES;
      if (ahead < mine) fetch(p + step_at(4 * ahead + w), q + step_at(4 * ahead + w), lds + now, valid_of(ahead));
#pragma unroll
      for (int s = 0; s < f.SUB; ++s) f.multiply(s, acc);
      now = now + BUF == STAGES * BUF ? 0 : now + BUF;
    }
  }
  static constexpr int TEAM = 256, ROWS = 64, CHUNKS = 1, PARTS = 4, W = 64, PITCH = W + 4;  // the epilogue: all waves together
  static constexpr int SCRATCH = PARTS * ROWS * PITCH * 4;
  __device__ __forceinline__ static int who() { return threadIdx.x; }
  __device__ __forceinline__ static char* part(char* lds) { return lds; }
  __device__ __forceinline__ static int row0() { return 0; }
  __device__ __forceinline__ static int column0(int) { return 0; }
  __device__ __forceinline__ static void settle() { __syncthreads(); }
  __device__ __forceinline__ void spill(int, char* lds) const {
    const int l = lane_id();
    int* t = (int*)lds + (wave_id() * ROWS + (l & 31)) * PITCH + 4 * (l >> 5);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const i32x16 v = __builtin_bit_cast(i32x16, acc[a][b]);
#pragma unroll
        for (int r = 0; r < 16; r += 4) *(i32x4*)(t + b * 32 * PITCH + a * 32 + 2 * r) = i32x4{v[r], v[r + 1], v[r + 2], v[r + 3]};
      }
    settle();
  }
};

template <class TL>
__host__ __device__ constexpr int tile_bytes() {
  return TL::LDS > TL::SCRATCH ? TL::LDS : TL::SCRATCH;
}
// Sums of a chunk: row r, words i .. i + N - 1 (N and i multiples of four)
template <class TL, int N, class V>
__device__ __forceinline__ void chunk_sums(const char* mine, int r, int i, V (&v)[N]) {
  typedef V V4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    V4 s = *(const V4*)((const V*)mine + r * TL::PITCH + i + e);
#pragma unroll
    for (int o = 1; o < TL::PARTS; ++o) s += *(const V4*)((const V*)mine + (o * TL::ROWS + r) * TL::PITCH + i + e);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[e + k] = s[k];
  }
}

// Workgroups of THREADS threads in two dimensions: the threads of one dimension are counted in 32 bits.
constexpr long GRID_X = 1l << 21;
template <int THREADS>
inline dim3 grid_of(long groups) {
  static_assert(GRID_X * THREADS < 1l << 32, "more threads along x than a launch counts");
  return dim3((unsigned)(groups < GRID_X ? groups : GRID_X), (unsigned)((groups + GRID_X - 1) / GRID_X));
}
__device__ __forceinline__ long group_id() { return blockIdx.y * GRID_X + blockIdx.x; }

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
// N neighbouring results, rounded to T, to an output row: 16 bytes at a time wherever they fall, at the row's end one by one
template <class T, int N>
__device__ __forceinline__ void store_some(T* at, const float (&v)[N], int left) {
  constexpr int W = 16 / (int)sizeof(T);
  static_assert(N % W == 0, "whole stores");
  typedef T V __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  if (left >= N) {
#pragma unroll
    for (int e = 0; e < N; e += W) {
      V w;
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = (T)v[e + k];
      *(V*)(at + e) = w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) at[e] = (T)v[e];
  }
}

}  // namespace lb
