// Matrix operators of few bits behind the C ABI: nls_quantize_rows, nls_int8_matmul, nls_int8_linear, nls_orthogonalize (include/neolssvm_hip.h).
// A translation unit of its own: the kernels here are 8- and 16-bit matrix code with a float epilogue and take other compiler options than the
// 64-bit engines (Makefile).  All arrays are the caller's device memory, the workspace included, and every launch goes to the caller's stream: nothing
// is allocated, waited for or kept, so calls on different streams do not meet and any of them can be captured into a graph.
#include "nls_host.h"

#include "nls_int8.h"
#include "nls_ortho.h"

using namespace lb;

namespace {

// The context's device for the length of a call; the caller's current device comes back afterwards.
struct DeviceGuard {
  int before = -1;
  hipError_t err = hipSuccess;
  explicit DeviceGuard(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device)
      err = hipSetDevice(device);
    else
      before = -1;
  }
  ~DeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// A launch that says itself whether it failed: the thread's last error may be that of some call before, which is neither this one's nor this one's to clear.
template <class P>
struct Given {
  using type = P;
};
template <class... P>
int launch(nls_ctx* ctx, const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t lds, hipStream_t st, typename Given<P>::type... args) {
  void* at[] = {&args...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3((unsigned)threads), at, lds, st);
  if (e == hipSuccess) return NLS_OK;
  (void)hipGetLastError();  // (reported here)
  return fail(ctx, NLS_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

// Dynamic LDS beyond 64 KB has to be asked for, once per kernel and device.
template <auto F>
int ask_lds(nls_ctx* ctx, int bytes) {
  static std::atomic<unsigned long long> asked{0};  // a bit a device (the first 64; asking again does no harm)
  const unsigned long long bit = ctx->device < 64 ? 1ull << ctx->device : 0;
  if (bytes <= 65536 || (asked.load(std::memory_order_relaxed) & bit)) return NLS_OK;
  HIPCHK(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(F), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  asked.fetch_or(bit, std::memory_order_relaxed);
  return NLS_OK;
}

int type_size(int t) { return t == NLS_TYPE_F32 ? 4 : (t == NLS_TYPE_F16 || t == NLS_TYPE_BF16) ? 2 : 0; }

// The tile a product is cut into.  Measured (int8 and fp16 products of 300 .. 8192 rows and columns, 10 .. 256 K steps):
//   256 x 256 (eight waves, two steps held) reads the least and is first once its tiles keep more than half of the compute units busy: int8
//     2500 x 4096 x 4096 53 us against 59 with 128 x 128, 8192 x 8192 x 256 55 / 62;
//   128 x 128, four waves, two workgroups a unit, when there are more of them than units: int8 2047 x 4096 x 4096 41.7 us against 51 with eight waves,
//     52 (256 x 256) and 57 (64 x 64); 256 x 128 with eight waves 46, with four 53;
//   128 x 128, eight waves, three steps held, when they cover 0.6 .. 1 of the units: int8 1024 x 4096 x 4096 26.7 us against 27.8 (four waves) and 33
//     (64 x 64), pairs 2048^2 59 / 66 / 72;
//   64 x 64, four waves side by side, three workgroups a unit: more of them than units, or few K steps: 1536^2 symmetric pairs 25 us against 34 (128 x 128)
//     and 27 (K dealt out), int8 512 x 4096 x 4096 18.2 / 25 / 20; more than three steps held 0 .. 10 us slower (fewer workgroups a unit);
//   64 x 64 with the K steps dealt out over the waves otherwise: X X^T of 512 x 2048 pairs 15.5 us against 22 (side by side) and 42 (128 x 128), int8
//     256 x 4096 x 4096 11.6 / 14.5 / 24; at 16 steps (five Newton-Schulz steps of 512^2) 145 / 147, at 13 (400^2) 135 / 128, at 5 .. 7 (130 x 200) 98 / 86,
//     int8 at 8 .. 12 steps equal within 4 %.
enum TileKind { TILE_256, TILE_128, TILE_128_DEEP, TILE_64, TILE_64_RING };
template <class F>
TileKind tile_kind(const nls_ctx* ctx, F tiles, int steps) {
  const long cus = ctx->cus;
  if (20 * tiles(256) > 11 * cus) return TILE_256;
  if (tiles(128) > cus) return TILE_128;
  if (5 * tiles(128) >= 3 * cus) return TILE_128_DEEP;
  return tiles(64) > cus || steps < 16 ? TILE_64 : TILE_64_RING;
}

// ---- quantise ----
// Short rows: a wave each; others: a workgroup.  The number of pieces a thread holds follows from the length; rows past 8 pieces are read twice.
template <class T, bool VEC>
int quantize(nls_ctx* ctx, const T* x, long rows, long k, long rs, long cs, signed char* q, long ldq, float* scale, hipStream_t st) {
  constexpr long N = Few<T, VEC>::N;
  const dim3 waves = grid_of<256>((rows + 3) / 4), groups = grid_of<256>(rows);
#define QUANTIZE(G, HELD, GRID) return launch(ctx, "quantize_rows", k_quantize_rows<T, G, VEC, HELD>, GRID, 256, 0, st, x, rows, k, rs, cs, q, ldq, scale)
  if (k <= 64 * N) QUANTIZE(64, 1, waves);
  if (k <= 128 * N) QUANTIZE(64, 2, waves);
  if (k <= 512 * N) QUANTIZE(256, 2, groups);
  if (k <= 1024 * N) QUANTIZE(256, 4, groups);
  if (k <= 2048 * N) QUANTIZE(256, 8, groups);
  QUANTIZE(256, 0, groups);
#undef QUANTIZE
}
template <class T>
int quantize(nls_ctx* ctx, const T* x, long rows, long k, long rs, long cs, signed char* q, long ldq, float* scale, hipStream_t st) {
  // Transposed: where 32 rows a workgroup are enough workgroups (8192 x 8192 bfloat16 109 us against 441, 4096 x 4096 45 / 76, 4096 x 128 float32 5.2 / 6.8;
  // 1024 x 4096 42 / 28, 2048 x 64 6.2 / 4.3).
  if (rs == 1 && cs != 1 && rows >= 2048 && k >= 128)
    return launch(ctx, "quantize_rows", k_quantize_turned<T>, grid_of<1024>((rows + Turned<T>::ROWS - 1) / Turned<T>::ROWS), 1024, 0, st, x, rows, k, cs, q, ldq, scale);
  return cs == 1 ? quantize<T, true>(ctx, x, rows, k, rs, cs, q, ldq, scale, st) : quantize<T, false>(ctx, x, rows, k, rs, cs, q, ldq, scale, st);
}
int quantize_any(nls_ctx* ctx, const void* x, int type, long rows, long k, long rs, long cs, signed char* q, long ldq, float* scale, hipStream_t st) {
  switch (type) {
    case NLS_TYPE_F32: return quantize(ctx, (const float*)x, rows, k, rs, cs, q, ldq, scale, st);
    case NLS_TYPE_F16: return quantize(ctx, (const _Float16*)x, rows, k, rs, cs, q, ldq, scale, st);
    default: return quantize(ctx, (const __bf16*)x, rows, k, rs, cs, q, ldq, scale, st);
  }
}

// ---- 8-bit product ----
template <class T, class TL, int BI, int BJ>
int int8_tile(nls_ctx* ctx, const Int8Args& g, hipStream_t st) {
  const int ti = (g.n + BI - 1) / BI, tj = (g.m + BJ - 1) / BJ;
  constexpr int LDS = tile_bytes<TL>() + BJ * 4;
  NLSCHK((ask_lds<&k_int8_tile<T, TL, BI, BJ>>(ctx, LDS)));
  return launch(ctx, "int8_matmul", k_int8_tile<T, TL, BI, BJ>, dim3((unsigned)((long)ti * tj)), TL::THREADS, LDS, st, g, ti, tj, 8);
}
template <class T>
int int8_tile(nls_ctx* ctx, const Int8Args& g, hipStream_t st) {
  auto tiles = [&](long b) { return ((g.n + b - 1) / b) * ((g.m + b - 1) / b); };
  switch (tile_kind(ctx, tiles, (g.k + 127) / 128)) {
    case TILE_256: return int8_tile<T, Tile<MODE_I8, 256, 256, 2, 4, 2>, 256, 256>(ctx, g, st);
    case TILE_128: return int8_tile<T, Tile<MODE_I8, 128, 128, 2, 2, 2>, 128, 128>(ctx, g, st);
    case TILE_128_DEEP: return int8_tile<T, Tile<MODE_I8, 128, 128, 4, 2, 3>, 128, 128>(ctx, g, st);
    case TILE_64: return int8_tile<T, Tile<MODE_I8, 64, 64, 2, 2, 3>, 64, 64>(ctx, g, st);
    default: return int8_tile<T, Ring<MODE_I8, 2>, 64, 64>(ctx, g, st);
  }
}
template <class T, int MG, int NG, bool FUSED>
int int8_few(nls_ctx* ctx, const Int8Args& g, const FewX& f, hipStream_t st) {
  const size_t rows = FUSED ? ((size_t)g.m * ((g.k + 63) / 64 * 64 + 16) + 64 + 512 + 255) / 256 * 256 : 0;
  const size_t lds = rows + (size_t)8 * MG * NG * 1024;
  return launch(ctx, "int8_matmul", k_int8_few<T, MG, NG, FUSED>, grid_of<512>((g.n + 16l * NG - 1) / (16 * NG)), 512, lds, st, g, f);
}
// Two row groups of b a workgroup halve what is read of a; taken where that leaves a workgroup for every compute unit.
template <class T, int MG>
int int8_few(nls_ctx* ctx, const Int8Args& g, const FewX& f, hipStream_t st) {
  if (MG > 1 && (g.n + 31) / 32 >= ctx->cus) return int8_few<T, MG, 2, false>(ctx, g, f, st);
  return int8_few<T, MG, 1, false>(ctx, g, f, st);
}
// Few rows of a: fragments straight from memory, or tiles.  Measured, m x n x k, the kernel alone with b from memory (the last of it still in the
// caches: 1 .. 6 us less): 16 x 4096 x 4096 8.3 us against 11.0 with tiles, 16 x 2048 x 2048 5.2 / 7.6, 16 x 1024 x 8192 10.8 / 16.8, 48 x 4096 x 4096 12.4 / 12.2,
// 48 x 2048 x 2048 7.3 / 8.4; from 8192 channels on there are tiles enough: 32 x 8192 x 8192 24.3 / 20.7, 48 x 8192 x 8192 28.4 / 22.4.  Up to 16 rows stay
// with the fragments there, which take b from any address: 16 x 8192 x 8192 20.2 / 19.3 (in the caches 18.9 / 14.5), 16 x 14336 x 4096 20.9 / 14.8.
bool int8_is_few(long m, long n) { return m <= 16 || (m <= 48 && n < 8192); }
template <class T>
int int8_product(nls_ctx* ctx, const Int8Args& g, const FewX& f, hipStream_t st) {
  if (int8_is_few(g.m, g.n)) return g.m <= 16 ? int8_few<T, 1>(ctx, g, f, st) : g.m <= 32 ? int8_few<T, 2>(ctx, g, f, st) : int8_few<T, 3>(ctx, g, f, st);
  return int8_tile<T>(ctx, g, st);
}
// Whether int8_linear quantises inside the product: every workgroup does all the rows of x over again, which has to stay small beside its share of b.
// Measured, one launch / two: 1 x 4096 x 4096 8.2 / 9.6 us, 1 x 8192 x 8192 18.9 / 20.9; 4 x 4096 x 4096 11.5 / 10.8 (and a launch less to make, which is
// what a caller waits for there), 2 x 8192 x 8192 23.7 / 21.6, 4 x 8192 x 8192 30.6 / 22.9.
bool int8_fused(long m, long n, long k) { return m * k <= 32768 && (m == 1 || (m <= FEW_ROWS && n * k <= 1l << 24)); }
template <class T>
int int8_fused_product(nls_ctx* ctx, const Int8Args& g, const FewX& f, hipStream_t st) {
  return int8_few<T, 1, 1, true>(ctx, g, f, st);
}
int int8_product_any(nls_ctx* ctx, const Int8Args& g, const FewX& f, int type, hipStream_t st) {
  switch (type) {
    case NLS_TYPE_F32: return int8_product<float>(ctx, g, f, st);
    case NLS_TYPE_F16: return int8_product<_Float16>(ctx, g, f, st);
    default: return int8_product<__bf16>(ctx, g, f, st);
  }
}

long up16(long k) { return (k + 15) / 16 * 16; }
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// Rows that the product can read where they are.  Tiles: those that start at multiples of 16 bytes and may be read up to one.  Few rows: any start for up
// to 16 of them (16 x 4097 x 4099 from odd addresses 11 us, aligned 7.6), multiples of 16 bytes for more (48 x 4097 x 4099: 43 us from odd addresses, 22 us
// with the copy, 13 aligned).
bool rows_ready(long m, long n, const void* p, long ld, long k, int flags, int flag) {
  const bool aligned = (uintptr_t)p % 16 == 0 && ld % 16 == 0;
  if (int8_is_few(m, n)) return m <= 16 || aligned;
  return aligned && ld >= up16(k) && (k % 16 == 0 || (flags & flag));
}

int check_int8(nls_ctx* ctx, const char* what, int64_t m, int64_t n, int64_t k, int type, int bias_type, const void* bias) {
  if (m < 0 || n < 0) return fail(ctx, NLS_ERR_ARG, "%s: negative size", what);
  if (k < 1 || k > NLS_INT8_MAX_K) return fail(ctx, NLS_ERR_ARG, "%s: k = %lld; 1 .. %d products are summed in 32 bits without overflow", what, (long long)k, NLS_INT8_MAX_K);
  if (m > INT32_MAX - 256 || n > INT32_MAX - 256) return fail(ctx, NLS_ERR_ARG, "%s: more than 2^31 rows", what);
  if (type_size(type) == 0) return fail(ctx, NLS_ERR_ARG, "%s: unknown element type %d", what, type);
  if (bias && bias_type != NLS_TYPE_F32 && bias_type != type) return fail(ctx, NLS_ERR_ARG, "%s: the bias must be float32 or of the result's type", what);
  return NLS_OK;
}

// a and b as the kernels take them: laid out again in the workspace, in one launch, where the caller's rows do not start at multiples of 16 bytes.
struct Int8Rows {
  const int8_t* p;
  long rows, ld;
  bool ready;
};
int operands(nls_ctx* ctx, const Int8Rows& a, const Int8Rows& b, long k, char* ws, Operand* oa, Operand* ob, hipStream_t st) {
  AlignRows todo[2] = {};
  int count = 0;
  long most = 0;
  const long ldy = up16(k);
  for (int i = 0; i < 2; ++i) {
    const Int8Rows& r = i ? b : a;
    Operand* o = i ? ob : oa;
    if (r.ready) {
      *o = Operand{(const char*)r.p, (unsigned)r.ld, (int)r.rows};
      continue;
    }
    todo[count++] = AlignRows{(const signed char*)r.p, (signed char*)ws, r.rows, r.ld};
    *o = Operand{ws, (unsigned)ldy, (int)r.rows};
    ws += up256((size_t)r.rows * ldy);
    most = std::max(most, r.rows * (ldy / 16));
  }
  if (!count) return NLS_OK;
  return launch(ctx, "int8_matmul (alignment)", k_align_rows, dim3((unsigned)std::min<long>((most + 255) / 256, 32768), (unsigned)count), 256, 0, st, todo[0], todo[1], k, ldy);
}

// ---- Newton-Schulz ----
// Matrices of at most 128 rows (nls_ortho.h): NS_SMALL, one workgroup holds X in registers and in LDS; NS_SLABS, workgroups share its columns.  Both
// read a matrix with 32-bit offsets.  NS_TILES: all others.  (float32 of up to 32 rows, whose products are of float32 itself, takes slabs earlier:
// 23 x 761 42 us against 53 in one workgroup.)
enum NsPath { NS_SMALL, NS_SLABS, NS_TILES };
NsPath ns_path(long p, long q, long row_stride, long col_stride, bool f32) {
  const long reach = 1l << 28;
  if (p > 128 || row_stride < 0 || col_stride < 0 || row_stride >= reach || col_stride >= reach || (p + 32) * row_stride + 16 * col_stride >= reach) return NS_TILES;
  return (q <= 256 || (p <= 64 && q <= 512) || (p <= 32 && q <= 1024 && !f32)) ? NS_SMALL : NS_SLABS;
}
// Workgroups that sum squares: four rows (of the direction that is dense in memory) each
int ns_parts(const NsMatrix& w) { return (int)std::min<long>(NS_PARTS, ((w.col_stride <= w.row_stride ? w.p : w.q) + 3) / 4); }

struct NsPlan {
  NsPath path;
  long p, q;
  size_t x, xt, a, parts, scales, batch_bytes, total;  // (NS_TILES: X, two X^T, A and B a matrix)
};
NsPlan ns_slab_plan(long p, long q, long batch) {
  NsPlan w{};
  w.p = p;
  w.q = q;
  const size_t rows = (size_t)(p + 31) / 32 * 32, slabs = (size_t)(q + NS_SLAB - 1) / NS_SLAB;
  w.x = slabs * NS_SLAB * rows * 4;
  w.a = slabs * rows * rows * 4;
  w.parts = up256((size_t)batch * NS_PARTS * sizeof(double));
  w.scales = up256((size_t)batch * sizeof(NsScales));
  w.total = w.parts + w.scales + (size_t)batch * (w.x + 2 * w.a);
  return w;
}
NsPlan ns_plan(long m, long n, long batch, long row_stride, long col_stride, bool f32) {
  NsPlan w{};
  w.p = std::min(m, n);
  w.q = std::max(m, n);
  const NsPath path = ns_path(w.p, w.q, m > n ? col_stride : row_stride, m > n ? row_stride : col_stride, f32);
  if (path == NS_SLABS) w = ns_slab_plan(w.p, w.q, batch);
  w.path = path;
  if (path != NS_TILES) return w;
  w.x = (size_t)w.p * pair_ld(w.q);
  w.xt = (size_t)w.q * pair_ld(w.p);
  w.a = (size_t)w.p * pair_ld(w.p);
  w.batch_bytes = w.x + 2 * w.xt + 2 * w.a;
  w.parts = up256((size_t)batch * NS_PARTS * sizeof(double));
  w.scales = up256((size_t)batch * sizeof(NsScales));
  w.total = w.parts + w.scales + (size_t)batch * w.batch_bytes;
  return w;
}

template <int KIND, class T, class TL, int B>
int ns_product_tile(nls_ctx* ctx, NsArgs g, long batch, hipStream_t st) {
  g.ti = (g.I + B - 1) / B;
  g.tj = (g.J + B - 1) / B;
  g.strip = 8;
  constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
  constexpr int LDS = tile_bytes<TL>();
  const long tiles = SYM ? (long)g.ti * (g.ti + 1) / 2 : (long)g.ti * g.tj;
  NLSCHK((ask_lds<&k_ns_product<KIND, T, TL, B, B>>(ctx, LDS)));
  return launch(ctx, "orthogonalize", k_ns_product<KIND, T, TL, B, B>, dim3((unsigned)tiles, 1, (unsigned)batch), TL::THREADS, LDS, st, g);
}
template <int KIND, class T>
int ns_product(nls_ctx* ctx, const NsArgs& g, long batch, hipStream_t st) {
  constexpr int MODE = MODE_F16PAIR;
  constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
  auto tiles = [&](long b) {
    const long i = (g.I + b - 1) / b, j = (g.J + b - 1) / b;
    return (SYM ? i * (i + 1) / 2 : i * j) * batch;
  };
  // 192 x 192, four waves with a SIMD each, where they cover the card in one go and 128 x 128 in more than one: five steps of a call against the rule below
  // alone, 2850 x 2950 2.02 ms / 2.26, 4000^2 3.90 / 4.51, 4096^2 4.12 / 4.61, 4200^2 5.46 / 6.11, 2048 x 4200 1.31 / 1.43, three of 2300^2 2.48 / 2.72, five of
  // 1700^2 1.95 / 2.18 (its symmetric or its last product, or both, have such sizes).
  if (tiles(128) > 2 * ctx->cus && tiles(192) <= ctx->cus) return ns_product_tile<KIND, T, Tile<MODE, 192, 192, 2, 2, 3>, 192>(ctx, g, batch, st);
  switch (tile_kind(ctx, tiles, (g.K + 31) / 32)) {
    case TILE_256: return ns_product_tile<KIND, T, Tile<MODE, 256, 256, 2, 4, 2>, 256>(ctx, g, batch, st);
    case TILE_128: return ns_product_tile<KIND, T, Tile<MODE, 128, 128, 2, 2, 2>, 128>(ctx, g, batch, st);
    case TILE_128_DEEP: return ns_product_tile<KIND, T, Tile<MODE, 128, 128, 4, 2, 3>, 128>(ctx, g, batch, st);
    case TILE_64: return ns_product_tile<KIND, T, Tile<MODE, 64, 64, 2, 2, 3>, 64>(ctx, g, batch, st);
    default: return ns_product_tile<KIND, T, Ring<MODE, 2>, 64>(ctx, g, batch, st);
  }
}

template <class T, int PB, int CB>
int ns_small(nls_ctx* ctx, const NsMatrix& w, bool tall, long batch, const NsCoef& cf, int steps, double eps, T* out, hipStream_t st) {
  constexpr int lds = NsLds<PB, CB, ns_full<T, PB>()>::BYTES;
  NLSCHK((ask_lds<&k_ns_small<T, PB, CB>>(ctx, lds)));
  return launch(ctx, "orthogonalize", k_ns_small<T, PB, CB>, dim3((unsigned)batch), 512, lds, st, w, cf, steps, eps, out, tall);
}
template <class T>
int ns_small_any(nls_ctx* ctx, const NsMatrix& w, bool tall, long batch, const NsCoef& cf, int steps, double eps, T* out, hipStream_t st) {
#define NS_SMALL_OF(PB, CB) return ns_small<T, PB, CB>(ctx, w, tall, batch, cf, steps, eps, out, st)
  if (w.q <= 128) {
    if (w.p <= 32) NS_SMALL_OF(1, 1);
    if (w.p <= 64) NS_SMALL_OF(2, 1);
    if (w.p <= 96) NS_SMALL_OF(3, 1);
    NS_SMALL_OF(4, 1);
  }
  if (w.q <= 256) {
    if (w.p <= 32) NS_SMALL_OF(1, 2);
    if (w.p <= 64) NS_SMALL_OF(2, 2);
    if (w.p <= 96) NS_SMALL_OF(3, 2);
    NS_SMALL_OF(4, 2);
  }
  if (w.q <= 512) {
    if (w.p <= 32) NS_SMALL_OF(1, 4);
    NS_SMALL_OF(2, 4);
  }
  NS_SMALL_OF(1, 8);
#undef NS_SMALL_OF
}

// p <= 128, more columns than one workgroup holds.  Up to four slabs' shares of A are added up by every workgroup, more by a launch of their own.
template <class T, int PB>
int ns_slabs(nls_ctx* ctx, const NsMatrix& w, bool tall, long batch, const NsCoef& cf, int steps, double eps, T* out, char* ws, hipStream_t st) {
  constexpr int P = 32 * PB, lds = NsLds<PB, NS_SLAB / 128, ns_full<T, PB>()>::BYTES;
  NLSCHK((ask_lds<&k_ns_slab<T, PB, true>>(ctx, lds)));
  NLSCHK((ask_lds<&k_ns_slab<T, PB, false>>(ctx, lds)));
  NsSlabs g{};
  g.m = w;
  g.count = ns_parts(w);
  g.eps = eps;
  g.steps = steps;
  g.out = out;
  g.tall = tall;
  const int slabs = (int)((w.q + NS_SLAB - 1) / NS_SLAB);
  const NsPlan plan = ns_slab_plan(w.p, w.q, batch);
  g.parts = (const double*)ws;
  g.scales = (NsScales*)(ws + plan.parts);
  g.x = (float*)(ws + plan.parts + plan.scales);
  float* a = (float*)(ws + plan.parts + plan.scales + batch * plan.x);
  float* next_a = a + batch * plan.a / 4;
  g.next_a = a;
  g.x_batch = plan.x / 4;
  g.a_batch = plan.a / 4;
  const dim3 grid((unsigned)slabs, (unsigned)batch);
  NLSCHK(launch(ctx, "orthogonalize", k_ns_norm<T>, dim3(g.count, (unsigned)batch), 256, 0, st, w, (double*)ws));
  NLSCHK((launch(ctx, "orthogonalize", k_ns_slab<T, PB, true>, grid, 512, lds, st, g, cf)));
  const bool sum = slabs > 4;
  g.shares = sum ? 1 : slabs;
  for (g.t = 0; g.t < steps; g.t = g.end + 1) {
    g.end = g.t;
    while (!(cf.ends >> g.end & 1)) ++g.end;
    if (sum) NLSCHK(launch(ctx, "orthogonalize", k_ns_sum, dim3(P * P / 256, (unsigned)batch), 64, 0, st, a, g.a_batch, P * P, slabs));
    g.a = a;
    g.next_a = next_a;
    NLSCHK((launch(ctx, "orthogonalize", k_ns_slab<T, PB, false>, grid, 512, lds, st, g, cf)));
    std::swap(a, next_a);
  }
  return NLS_OK;
}

// Which steps are done in one chain: as many as let small singular values grow by no more than `most` (nls_ortho.h); one at least.
void ns_chains(NsCoef& cf, int steps, double most) {
  cf.ends = 0;
  double grown = 1.0;
  for (int t = 0; t < steps; ++t) {
    const double g = std::max(1.0, cf.s[t].grow);
    if (t > 0 && grown * g > most) {
      cf.ends |= 1u << (t - 1);
      grown = 1.0;
    }
    grown *= g;
  }
  cf.ends |= 1u << (steps - 1);
  const double u = 1.0 + 1e-3;
  cf.first = ns_exponent(u);
  cf.last = -ns_factors(u, cf.s, cf.ends, steps, cf.f);
}
template <class T>
int orthogonalize(nls_ctx* ctx, const NsMatrix& w, const NsPlan& plan, bool tall, long batch, NsCoef& cf, int steps, double eps, T* out, char* ws, hipStream_t st) {
  // 16-bit matrices take pairs in every step as well.  Single products of the hi halves in the early ones would be a third of the work (4096^2 bfloat16, three
  // of five steps: 2.6 ms against 3.9), but the roundings of A and B to 11 bits couple strong and weak singular directions and the steps after them spread
  // that: the error against 64 bits was 0.75 (bfloat16) and 1.4 (float16) of the result's own rounding after five standard steps, 1.1 and 6.5 after six, 2.7
  // and 21 after twelve, where pairs stay at float32's error throughout.
  if (plan.path != NS_TILES) {
    const double half = std::is_same<T, __bf16>::value ? 0x1p-8 : 0x1p-11;  // half a step of the result, relative
    ns_chains(cf, steps, sizeof(T) == 4 ? 0.0 : std::sqrt(0x1p23 * half / 16.0));
    if (plan.path == NS_SMALL) return ns_small_any(ctx, w, tall, batch, cf, steps, eps, out, st);
    if (w.p <= 32) return ns_slabs<T, 1>(ctx, w, tall, batch, cf, steps, eps, out, ws, st);
    if (w.p <= 64) return ns_slabs<T, 2>(ctx, w, tall, batch, cf, steps, eps, out, ws, st);
    if (w.p <= 96) return ns_slabs<T, 3>(ctx, w, tall, batch, cf, steps, eps, out, ws, st);
    return ns_slabs<T, 4>(ctx, w, tall, batch, cf, steps, eps, out, ws, st);
  }
  ns_chains(cf, steps, 0.0);
  double* parts = (double*)ws;
  NsScales* scales = (NsScales*)(ws + plan.parts);
  char* base = ws + plan.parts + plan.scales;
  char *X = base, *XT = X + plan.x, *XU = XT + plan.xt, *A = XU + plan.xt, *B = A + plan.a;
  const int count = ns_parts(w);
  NLSCHK(launch(ctx, "orthogonalize", k_ns_norm<T>, dim3(count, (unsigned)batch), 256, 0, st, w, parts));
  NLSCHK(launch(ctx, "orthogonalize", k_ns_pack<T>, dim3((unsigned)((w.q + 63) / 64), (unsigned)((w.p + 63) / 64), (unsigned)batch), 256, 0, st, w, parts, count, eps, cf,
                steps, scales, X, XT, plan.batch_bytes));
  NsArgs g{};
  g.scales = scales;
  g.batch_bytes = plan.batch_bytes;
  const int p = (int)w.p, q = (int)w.q;
  for (int t = 0; t < steps; ++t) {
    g.t = t;
    g.P = g.Q = X;
    g.D = A;
    g.I = g.J = p;
    g.K = q;
    NLSCHK((ns_product<NS_GRAM, float>(ctx, g, batch, st)));
    g.P = g.Q = g.E = A;
    g.D = B;
    g.K = p;
    NLSCHK((ns_product<NS_POLY, float>(ctx, g, batch, st)));
    g.P = XT;
    g.Q = B;
    g.E = X;
    g.I = q;
    if (t + 1 < steps) {
      g.D = X;  // X stays where it is: a thread reads what it writes
      g.DT = XU;
      NLSCHK((ns_product<NS_STEP, float>(ctx, g, batch, st)));
      std::swap(XT, XU);
    } else {
      g.out = out;
      g.out_stride = (size_t)p * q;
      g.transposed = tall;
      NLSCHK((ns_product<NS_LAST, T>(ctx, g, batch, st)));
    }
  }
  return NLS_OK;
}

}  // namespace

extern "C" int nls_ctx_stream(nls_ctx* ctx, void** stream) {
  if (!ctx || !stream) return NLS_ERR_ARG;
  *stream = ctx->stream;
  return NLS_OK;
}

extern "C" int nls_quantize_rows(nls_ctx* ctx, const void* x, int type, int64_t rows, int64_t k, int64_t row_stride, int64_t col_stride, int8_t* q,
                                 int64_t ldq, float* scale, void* stream) {
  if (!ctx) return NLS_ERR_ARG;
  if (type_size(type) == 0) return fail(ctx, NLS_ERR_ARG, "quantize_rows: unknown element type %d", type);
  if (rows < 0 || k < 1) return fail(ctx, NLS_ERR_ARG, "quantize_rows: %lld rows of %lld elements", (long long)rows, (long long)k);
  if (rows > INT32_MAX) return fail(ctx, NLS_ERR_ARG, "quantize_rows: more than 2^31 rows");
  if (ldq < up16(k) || ldq % 16 != 0 || (uintptr_t)q % 16 != 0) return fail(ctx, NLS_ERR_ARG, "quantize_rows: rows of q must start at multiples of 16 bytes and hold k rounded up to them");
  if (rows == 0) return NLS_OK;
  if (!x || !q || !scale) return fail(ctx, NLS_ERR_ARG, "quantize_rows: null pointer");
  DeviceGuard dev(ctx->device);
  HIPCHK(ctx, dev.err);
  return quantize_any(ctx, x, type, rows, k, row_stride, col_stride, (signed char*)q, ldq, scale, (hipStream_t)stream);
}

extern "C" int nls_int8_matmul_workspace(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, int64_t m, int64_t n, int64_t k, int flags,
                                         size_t* bytes) {
  if (!bytes || m < 0 || n < 0 || k < 1) return NLS_ERR_ARG;
  *bytes = (rows_ready(m, n, a, lda, k, flags, NLS_INT8_A_PADDED) ? 0 : up256((size_t)m * up16(k))) +
           (rows_ready(m, n, b, ldb, k, flags, NLS_INT8_B_PADDED) ? 0 : up256((size_t)n * up16(k)));
  return NLS_OK;
}

extern "C" int nls_int8_matmul(nls_ctx* ctx, const int8_t* a, int64_t lda, const float* a_scale, const int8_t* b, int64_t ldb, const float* b_scale,
                               const void* bias, int bias_type, int64_t m, int64_t n, int64_t k, void* y, int type, int flags, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (!ctx) return NLS_ERR_ARG;
  NLSCHK(check_int8(ctx, "int8_matmul", m, n, k, type, bias_type, bias));
  if (lda < k || ldb < k || lda > UINT32_MAX / 512 || ldb > UINT32_MAX / 512) return fail(ctx, NLS_ERR_ARG, "int8_matmul: row strides %lld, %lld", (long long)lda, (long long)ldb);
  if (m == 0 || n == 0) return NLS_OK;
  if (!a || !a_scale || !b || !b_scale || !y) return fail(ctx, NLS_ERR_ARG, "int8_matmul: null pointer");
  size_t need = 0;
  (void)nls_int8_matmul_workspace(a, lda, b, ldb, m, n, k, flags, &need);
  if (workspace_bytes < need) return fail(ctx, NLS_ERR_ARG, "int8_matmul: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if ((uintptr_t)workspace % 256) return fail(ctx, NLS_ERR_ARG, "int8_matmul: the workspace must be aligned to 256 bytes");
  DeviceGuard dev(ctx->device);
  HIPCHK(ctx, dev.err);
  hipStream_t st = (hipStream_t)stream;
  Int8Args g{};
  NLSCHK(operands(ctx, {a, m, lda, rows_ready(m, n, a, lda, k, flags, NLS_INT8_A_PADDED)}, {b, n, ldb, rows_ready(m, n, b, ldb, k, flags, NLS_INT8_B_PADDED)}, k,
                  (char*)workspace, &g.a, &g.b, st));
  g.a_scale = a_scale;
  g.b_scale = b_scale;
  g.bias = bias;
  g.bias_type = bias_type;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.y = y;
  FewX f{};
  f.a_padded = flags & NLS_INT8_A_PADDED;
  f.b_padded = flags & NLS_INT8_B_PADDED;
  return int8_product_any(ctx, g, f, type, st);
}

extern "C" int nls_int8_linear_workspace(const int8_t* b, int64_t ldb, int64_t m, int64_t n, int64_t k, int flags, size_t* bytes) {
  if (!bytes || m < 0 || n < 0 || k < 1) return NLS_ERR_ARG;
  *bytes = (int8_fused(m, n, k) ? 0 : up256((size_t)m * up16(k)) + up256((size_t)m * 4)) +
           (rows_ready(m, n, b, ldb, k, flags, NLS_INT8_B_PADDED) ? 0 : up256((size_t)n * up16(k)));
  return NLS_OK;
}

extern "C" int nls_int8_linear(nls_ctx* ctx, const void* x, int type, int64_t row_stride, int64_t col_stride, const int8_t* b, int64_t ldb,
                               const float* b_scale, const void* bias, int bias_type, int64_t m, int64_t n, int64_t k, void* y, int flags,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (!ctx) return NLS_ERR_ARG;
  NLSCHK(check_int8(ctx, "int8_linear", m, n, k, type, bias_type, bias));
  if (ldb < k || ldb > UINT32_MAX / 512) return fail(ctx, NLS_ERR_ARG, "int8_linear: row stride %lld", (long long)ldb);
  if (m == 0 || n == 0) return NLS_OK;
  if (!x || !b || !b_scale || !y) return fail(ctx, NLS_ERR_ARG, "int8_linear: null pointer");
  size_t need = 0;
  (void)nls_int8_linear_workspace(b, ldb, m, n, k, flags, &need);
  if (workspace_bytes < need) return fail(ctx, NLS_ERR_ARG, "int8_linear: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if ((uintptr_t)workspace % 256) return fail(ctx, NLS_ERR_ARG, "int8_linear: the workspace must be aligned to 256 bytes");
  DeviceGuard dev(ctx->device);
  HIPCHK(ctx, dev.err);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  Int8Args g{};
  g.b_scale = b_scale;
  g.bias = bias;
  g.bias_type = bias_type;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.y = y;
  const bool b_ready = rows_ready(m, n, b, ldb, k, flags, NLS_INT8_B_PADDED);
  NLSCHK(operands(ctx, {nullptr, 0, 0, true}, {b, n, ldb, b_ready}, k, ws, &g.a, &g.b, st));
  if (!b_ready) ws += up256((size_t)n * up16(k));
  const int b_padded = flags & NLS_INT8_B_PADDED;
  if (int8_fused(m, n, k)) {
    const FewX f{x, row_stride, col_stride, col_stride == 1, 0, b_padded};
    switch (type) {
      case NLS_TYPE_F32: return int8_fused_product<float>(ctx, g, f, st);
      case NLS_TYPE_F16: return int8_fused_product<_Float16>(ctx, g, f, st);
      default: return int8_fused_product<__bf16>(ctx, g, f, st);
    }
  }
  const long ldq = up16(k);
  signed char* q = (signed char*)ws;
  float* scale = (float*)(ws + up256((size_t)m * ldq));
  NLSCHK(quantize_any(ctx, x, type, m, k, row_stride, col_stride, q, ldq, scale, st));
  g.a = Operand{(const char*)q, (unsigned)ldq, (int)m};
  g.a_scale = scale;
  FewX f{};
  f.a_padded = 1;
  f.b_padded = b_padded;
  return int8_product_any(ctx, g, f, type, st);
}

extern "C" int nls_orthogonalize_workspace(int64_t batch, int64_t m, int64_t n, int64_t row_stride, int64_t col_stride, size_t* bytes) {
  if (!bytes || batch < 0 || m < 0 || n < 0) return NLS_ERR_ARG;
  *bytes = std::max(ns_plan(m, n, batch, row_stride, col_stride, false).total, ns_plan(m, n, batch, row_stride, col_stride, true).total);
  return NLS_OK;
}

extern "C" int nls_orthogonalize(nls_ctx* ctx, const void* g, int type, int64_t batch, int64_t m, int64_t n, int64_t batch_stride, int64_t row_stride,
                                 int64_t col_stride, const double* coefficients, int steps, double eps, void* out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!ctx) return NLS_ERR_ARG;
  if (type_size(type) == 0) return fail(ctx, NLS_ERR_ARG, "orthogonalize: unknown element type %d", type);
  if (batch < 0 || m < 0 || n < 0) return fail(ctx, NLS_ERR_ARG, "orthogonalize: negative size");
  if (steps < 1 || steps > NS_MAX_STEPS) return fail(ctx, NLS_ERR_ARG, "orthogonalize: %d steps; 1 .. %d", steps, NS_MAX_STEPS);
  if (!(eps >= 0.0) || !(eps < 1e30)) return fail(ctx, NLS_ERR_ARG, "orthogonalize: eps must be a number >= 0");
  if (!coefficients) return fail(ctx, NLS_ERR_ARG, "orthogonalize: null pointer");
  NsCoef cf{};
  double u = 1.0 + 1e-3;
  for (int t = 0; t < steps; ++t) {
    ns_step(coefficients[3 * t], coefficients[3 * t + 1], coefficients[3 * t + 2], u, &cf.s[t]);
    u = ns_peak_x(cf.s[t], u) * (1.0 + 1e-3);
    if (!(u < 1e6)) return fail(ctx, NLS_ERR_ARG, "orthogonalize: the coefficients let singular values grow past 1e6 in step %d", t + 1);
  }
  if (m > (1 << 20) || n > (1 << 20) || batch > 65535) return fail(ctx, NLS_ERR_ARG, "orthogonalize: at most 2^20 rows and columns and 65535 matrices");
  if (batch == 0 || m == 0 || n == 0) return NLS_OK;
  const NsPlan plan = ns_plan(m, n, batch, row_stride, col_stride, type == NLS_TYPE_F32);
  if (!g || !out || (plan.total && !workspace)) return fail(ctx, NLS_ERR_ARG, "orthogonalize: null pointer");
  if (workspace_bytes < plan.total) return fail(ctx, NLS_ERR_ARG, "orthogonalize: workspace of %zu bytes, %zu needed", workspace_bytes, plan.total);
  if ((uintptr_t)workspace % 256) return fail(ctx, NLS_ERR_ARG, "orthogonalize: the workspace must be aligned to 256 bytes");
  DeviceGuard dev(ctx->device);
  HIPCHK(ctx, dev.err);
  const bool tall = m > n;
  NsMatrix w{g, plan.p, plan.q, tall ? col_stride : row_stride, tall ? row_stride : col_stride, batch_stride};
  hipStream_t st = (hipStream_t)stream;
  switch (type) {
    case NLS_TYPE_F32: return orthogonalize(ctx, w, plan, tall, batch, cf, steps, eps, (float*)out, (char*)workspace, st);
    case NLS_TYPE_F16: return orthogonalize(ctx, w, plan, tall, batch, cf, steps, eps, (_Float16*)out, (char*)workspace, st);
    default: return orthogonalize(ctx, w, plan, tall, batch, cf, steps, eps, (__bf16*)out, (char*)workspace, st);
  }
}
