// The choice of kernels of the products by expert, compiled once for each element type (prod_bf16.hip and its like).
#pragma once
#include "prod_rows.h"

namespace ktmi {

template <typename T, int MODE, bool GATED, bool DIRECT, bool TAIL, int SIZE>
int launch_tile_of(const TileArgs& a, hipStream_t stream) {
  constexpr bool FOUR = SIZE == TILE_SMALL || SIZE == TILE_LOW;  // waves
  constexpr int BM = tile_m(SIZE), BN = tile_n(SIZE) / (GATED ? 2 : 1), THREADS = FOUR ? 256 : 512;
  const int64_t nt = (a.N + BN - 1) / BN;
  int64_t mt = (a.M + BM - 1) / BM;
  if (a.seg.offsets) mt = MODE == PROD_DW ? mt * a.seg.E : a.M / BM + a.seg.E + 2;
  const int64_t grid = (mt * nt * a.splits + 7) / 8 * 8;
  KTMI_REQUIRE(grid < (int64_t)0xffffffff / THREADS, KTMI_EINVAL, "a grid of %lld blocks (below 2^32 threads)", (long long)grid);
  if constexpr (SIZE == TILE_LARGE) prod_tile<T, MODE, GATED, DIRECT, TAIL, 2, 4, 4, 2, 2><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else if constexpr (SIZE == TILE_DEEP) prod_tile<T, MODE, GATED, DIRECT, TAIL, 2, 4, 2, 2, 3><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else if constexpr (SIZE == TILE_LOW) prod_tile<T, MODE, GATED, DIRECT, TAIL, 2, 2, 1, 2, (DIRECT && T::ES == 2 ? 3 : 2)><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else prod_tile<T, MODE, GATED, DIRECT, TAIL, 2, 2, 2, 2, 2><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

// Rows at multiples of 4 bytes, whose tiles 32-bit offsets reach.
inline bool rows_direct(const void* p, int64_t stride, int64_t span) {
  return ((uintptr_t)p | (uintptr_t)stride) % 4 == 0 && span * stride < 0x7fffffff;
}

template <typename T, int MODE, bool GATED>
int launch_tile(const TileArgs& a, int size, hipStream_t stream) {
  const int64_t wide = MODE == PROD_FWD && GATED ? 2 * (int64_t)a.N : 256;
  const bool direct = rows_direct(a.p, a.p_stride, 256) && rows_direct(a.q, a.q_stride, wide) && a.q_expert % 4 == 0;
  if constexpr (MODE != PROD_DW) {
    if (direct && a.K % (STEP_BYTES / T::ES)) {
      if (size == TILE_LOW) return launch_tile_of<T, MODE, GATED, true, true, TILE_LOW>(a, stream);
      if (size == TILE_LARGE) return launch_tile_of<T, MODE, GATED, true, true, TILE_LARGE>(a, stream);
      return launch_tile_of<T, MODE, GATED, true, true, TILE_SMALL>(a, stream);
    }
    if (size == TILE_LOW)
      return direct ? launch_tile_of<T, MODE, GATED, true, false, TILE_LOW>(a, stream)
                    : launch_tile_of<T, MODE, GATED, false, false, TILE_LOW>(a, stream);
  }
  if (!direct) return launch_tile_of<T, MODE, GATED, false, false, TILE_SMALL>(a, stream);
  if constexpr (MODE == PROD_FWD) {
    if (size == TILE_DEEP) return launch_tile_of<T, MODE, GATED, true, false, TILE_DEEP>(a, stream);
  }
  if (size == TILE_LARGE) return launch_tile_of<T, MODE, GATED, true, false, TILE_LARGE>(a, stream);
  return launch_tile_of<T, MODE, GATED, true, false, TILE_SMALL>(a, stream);
}

// ---- the sums of a tile's k shared by `splits` blocks, in the blocks' order (the same bits from run to run; 512 x 4096 in three slices 5
// us, bound by the caches and its launch): four values a thread where rows
// hold multiples of four (VEC), else one. gated: rows [g; u] of 2 N, h = act(g) u.
template <typename T, bool GATED, bool VEC>
__global__ __launch_bounds__(256) void sum_parts(const float* part, int splits, int64_t slice, int64_t rows, int N, int act,
                                                 uint8_t* out, float* gu) {
  using S = typename T::S;
  constexpr int V = VEC ? 4 : 1;
  const int64_t n = N / V, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * n) return;
  const int64_t row = i / n, col = (i - row * n) * V;
  const float* p = part + row * (GATED ? 2 : 1) * N + col;
  float g[V] = {}, u[V] = {};
  for (int s = 0; s < splits; ++s, p += slice) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      g[v] += p[v];
      if constexpr (GATED) u[v] += p[N + v];
    }
  }
  S* o = (S*)out + row * N + col;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (GATED) {
      o[v] = (S)(act_of<S>(act, g[v]) * u[v]);
      if (gu) gu[row * 2 * N + col + v] = g[v], gu[row * 2 * N + N + col + v] = u[v];
    } else {
      o[v] = (S)g[v];
    }
  }
}

template <typename T, bool GATED>
int launch_sum_parts(const float* part, int splits, int64_t slice, int64_t rows, int64_t N, int act, void* out, float* gu,
                     hipStream_t stream) {
  const bool vec = N % 4 == 0;
  const int64_t grid = (rows * (vec ? N / 4 : N) + 255) / 256;
  KTMI_REQUIRE(grid < (int64_t)0xffffffff / 256, KTMI_EINVAL, "a grid of %lld blocks (below 2^32 threads)", (long long)grid);
  if (vec) sum_parts<T, GATED, true><<<(unsigned)grid, 256, 0, stream>>>(part, splits, slice, rows, (int)N, act, (uint8_t*)out, gu);
  else sum_parts<T, GATED, false><<<(unsigned)grid, 256, 0, stream>>>(part, splits, slice, rows, (int)N, act, (uint8_t*)out, gu);
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

template <typename X, bool FP8, bool GATED, int CT, int NRF, int WK>
int launch_rows_of(RowsArgs a, hipStream_t stream) {
  constexpr int WAVES = 8, OUT = (GATED ? 8 : 16) * NRF * (WAVES / WK);
  a.row_tiles = (a.N + OUT - 1) / OUT;
  int64_t tiles = (a.R + 16 * CT - 1) / (16 * CT);
  if (a.ids) tiles = a.R;
  else if (a.seg.offsets) tiles = a.R / (16 * CT) + min(a.seg.E + 2, a.R);
  const int64_t grid = tiles * a.row_tiles;
  KTMI_REQUIRE(grid < (int64_t)0xffffffff / (64 * WAVES), KTMI_EINVAL, "a grid of %lld blocks (below 2^32 threads)",
               (long long)grid);
  prod_rows<X, FP8, GATED, CT, NRF, WK, WAVES / WK><<<(unsigned)grid, 64 * WAVES, 0, stream>>>(a);
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

// mean: rows of a matrix. Rows of w a wave: 16 where more would leave CUs without a block, else 32 or 64, which share the rows of
// x and, of e4m3, their quantisation (one row by 16384 x 4096 e4m3: 25 us with 16). Rows of w below 16 units are too
// short for eight waves: two share one.
template <typename X, bool FP8, bool GATED>
int launch_rows(const RowsArgs& a, int mean, hipStream_t stream) {
  constexpr int UE = 128 / (FP8 ? 1 : X::ES);
  const bool shorter = a.K < 16 * UE;
  const int64_t cols = mean <= 16 ? 16 : 32;
  const int64_t parts = a.ids || a.seg.offsets ? min((int64_t)a.seg.E, (int64_t)a.R) : (a.R + cols - 1) / cols;
  const int64_t frags = parts * (GATED ? 2 : 1) * a.N / 16;
  if (cols == 16) {
    if (frags < (FP8 ? 512 : 4 * 512)) return launch_rows_of<X, FP8, GATED, 1, 1, 8>(a, stream);
    if (shorter) return launch_rows_of<X, FP8, GATED, 1, 2, 2>(a, stream);
    if constexpr (FP8) {
      if (frags < 1024) return launch_rows_of<X, FP8, GATED, 1, 2, 8>(a, stream);
    }
    return launch_rows_of<X, FP8, GATED, 1, 4, 8>(a, stream);
  }
  if constexpr (FP8) {  // (without ids few_rows() ends below)
    if (frags >= 4 * 512)
      return shorter ? launch_rows_of<X, FP8, GATED, 2, 2, 2>(a, stream) : launch_rows_of<X, FP8, GATED, 2, 2, 8>(a, stream);
  }
  return launch_rows_of<X, FP8, GATED, 2, 1, 8>(a, stream);
}

template <typename S, bool EXACT, bool DIRECT, int SIZE>
int launch_fp8_tile_of(const Fp8TileArgs& a, hipStream_t stream) {
  constexpr int BM = tile_m(SIZE), BN = tile_n(SIZE), THREADS = SIZE == TILE_LARGE ? 512 : 256;
  const int64_t mt = a.seg.offsets ? a.M / BM + a.seg.E + 2 : (a.M + BM - 1) / BM;
  const int64_t grid = (mt * ((a.N + BN - 1) / BN) * a.splits + 7) / 8 * 8;
  KTMI_REQUIRE(grid < (int64_t)0xffffffff / THREADS, KTMI_EINVAL, "a grid of %lld blocks (below 2^32 threads)", (long long)grid);
  if constexpr (SIZE == TILE_LARGE) fp8_tile<S, EXACT, DIRECT, 2, 4, 8, 4><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else if constexpr (SIZE == TILE_LOW) fp8_tile<S, EXACT, DIRECT, 2, 2, 2, 4><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else fp8_tile<S, EXACT, DIRECT, 2, 2, 4, 4><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

template <typename X>
int launch_fp8_tile(const Fp8TileArgs& a, int size, hipStream_t stream) {
  using S = typename X::S;
  constexpr bool EXACT = std::is_same<X, F32>::value;
  const bool direct = a.K % 16 == 0 && rows_direct(a.w, a.K, 256);
  if (size == TILE_LOW)
    return direct ? launch_fp8_tile_of<S, EXACT, true, TILE_LOW>(a, stream) : launch_fp8_tile_of<S, EXACT, false, TILE_LOW>(a, stream);
  if constexpr (!EXACT) {  // (whose operands as bf16 leave no registers for 256 rows)
    if (direct && size == TILE_LARGE) return launch_fp8_tile_of<S, EXACT, true, TILE_LARGE>(a, stream);
  }
  return direct ? launch_fp8_tile_of<S, EXACT, true, TILE_SMALL>(a, stream) : launch_fp8_tile_of<S, EXACT, false, TILE_SMALL>(a, stream);
}

// ---- one group of 16 lanes a group of 128 values: codes [rows, blocks * 128], scales [blocks, rows] (a tile takes the scales of
// its rows for a block at a time). Bound by HBM: 91750 of 131072 rows of 2048 bf16 126 us, 4.5 TB/s.
template <typename X>
__global__ __launch_bounds__(256) void fp8_quantise(const uint8_t* x, int64_t stride, int K, int64_t rows, const int32_t* end,
                                                    uint8_t* codes, float* scales) {
  const int blocks = (K + 127) / 128;
  const int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int i = threadIdx.x & 15;
  // sixteen rows of a column of groups after each other, then the next column's
  const int64_t band = g / (16 * (int64_t)blocks);
  const int in = (int)(g - band * 16 * blocks);
  const int64_t row = band * 16 + in % 16;
  const int b = in / 16;
  if (row >= rows || (end && row >= *end)) return;  // the whole group; end: rows behind the last segment have no product
  constexpr int XC = 8 / X::EPC;
  u32x4_t c[XC];
  const uint8_t* r = x + row * stride * X::ES;
#pragma unroll
  for (int j = 0; j < XC; ++j) c[j] = load_chunk<X::ES>(r, (int64_t)b * 128 + 8 * i + X::EPC * j, K);
  float v[8];
  unpack_chunks<X>(c, v);
  float top = 0x1p-116f;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float inv = 448.0f / top;
  const u32x2_t q = {e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
  *(u32x2_t*)(codes + (row * blocks + b) * 128 + 8 * i) = q;
  if (i == 0) scales[b * rows + row] = top / 448.0f;
}

template <typename X>
int launch_quantise(const void* x, int64_t stride, int64_t K, int64_t rows, const int32_t* end, uint8_t* codes, float* scales,
                    hipStream_t stream) {
  const int64_t groups = (rows + 15) / 16 * 16 * ((K + 127) / 128);
  KTMI_REQUIRE(groups / 16 < (int64_t)0xffffffff / 256, KTMI_EINVAL, "fp8: %lld groups of 128 values (below 2^28)",
               (long long)groups);
  fp8_quantise<X><<<(unsigned)(groups / 16), 256, 0, stream>>>((const uint8_t*)x, stride, (int)K, rows, end, codes, scales);
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

// ---- the gradients of the sums from that of h = act(g) u: dg = dh u act'(g), du = dh act(g), from the fp32 sums, rounded once to
// the type that the products take. Bound by HBM: 4096 x 2048 bf16 20 us, 5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void gated_grad(const float* gu, const uint8_t* dh, int64_t dh_stride, int N, int64_t rows,
                                                  int act, uint8_t* dgu) {
  using S = typename T::S;
  const int64_t n4 = (N + 3) / 4, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / n4;
  const int n = 4 * (int)(at - row * n4);
  if (row >= rows) return;
  const float *g = gu + row * 2 * N + n, *u = g + N;
  const S* d = (const S*)dh + row * dh_stride + n;
  S *dg = (S*)dgu + row * 2 * N + n, *du = dg + N;
  typedef typename vec4_of<S>::type V;
  // vectors of four where every row starts at one
  if (N % 4 == 0 && dh_stride % 4 == 0 && ((uintptr_t)dh | (uintptr_t)dgu) % sizeof(V) == 0) {
    const f32x4_t gv = gload<f32x4_t>(g), uv = gload<f32x4_t>(u);
    const V dv = gload<V>(d);
    V a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f, df;
      act_grad<S>(act, gv[i], f, df);
      a[i] = (S)((float)dv[i] * uv[i] * df);
      b[i] = (S)((float)dv[i] * f);
    }
    *(V*)dg = a;
    *(V*)du = b;
  } else {
    for (int i = 0; i < 4 && n + i < N; ++i) {
      float f, df;
      act_grad<S>(act, g[i], f, df);
      dg[i] = (S)((float)d[i] * u[i] * df);
      du[i] = (S)((float)d[i] * f);
    }
  }
}

template <typename T>
int launch_gated_grad(const float* gu, const void* dh, int64_t dh_stride, int64_t N, int64_t rows, int act, void* dgu,
                      hipStream_t stream) {
  const int64_t grid = ((N + 3) / 4 * rows + 255) / 256;
  KTMI_REQUIRE(grid < (int64_t)0xffffffff / 256, KTMI_EINVAL, "gated_grad: %lld values (below 2^34)", (long long)(N * rows));
  gated_grad<T><<<(unsigned)grid, 256, 0, stream>>>(gu, (const uint8_t*)dh, dh_stride, (int)N, rows, act, (uint8_t*)dgu);
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

template <typename T>
struct ProdOps {
  static int tile(int mode, bool gated, const TileArgs& a, int size, hipStream_t s) {
    if (mode == PROD_DX) return launch_tile<T, PROD_DX, false>(a, size, s);
    if (mode == PROD_DW) return launch_tile<T, PROD_DW, false>(a, size, s);
    return gated ? launch_tile<T, PROD_FWD, true>(a, size, s) : launch_tile<T, PROD_FWD, false>(a, size, s);
  }
  static int sum(bool gated, const float* part, int splits, int64_t slice, int64_t rows, int64_t N, int act, void* out, float* gu,
                 hipStream_t s) {
    return gated ? launch_sum_parts<T, true>(part, splits, slice, rows, N, act, out, gu, s)
                 : launch_sum_parts<T, false>(part, splits, slice, rows, N, act, out, gu, s);
  }
  static int rows(bool fp8, bool gated, const RowsArgs& a, int mean, hipStream_t s) {
    if (fp8) return launch_rows<T, true, false>(a, mean, s);
    return gated ? launch_rows<T, false, true>(a, mean, s) : launch_rows<T, false, false>(a, mean, s);
  }
};

}  // namespace ktmi
