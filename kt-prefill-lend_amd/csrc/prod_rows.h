// Products of few rows: y[r, n] = sum over k of x[r, k] w[n, k], for decode windows, bound by the bytes of w.
//
// A wave takes 16 NRF rows of w (gated: 8 of the gate and the 8 rows of up beside them, for each 16) and at most 16 CT rows of
// x, which are the columns of the matrix cores' tiles. WK waves of a block share the k: wave i takes the 128-byte units
// i, i + WK, .. of the rows, so that they read neighbouring bytes, and each unit of x is read by one of them
// only, straight into the operands' registers; their sums meet in LDS. The block's other waves take the rows behind.
// One row by 4096 x 7168, calls in a graph: e4m3 10.6 us with weights from HBM, which their bytes take 6.0 of, and 9.0 from the
// last-level cache; bf16 gate and up 12.9 (12.0) and 11.3; an empty kernel of that grid 1.6. 16 rows 15 us, 32 rows 21 in both,
// where the rows of x from L2 take as long as w: tiles go on from there.
#pragma once
#include "prod_fp8.h"

namespace ktmi {

struct RowsArgs {
  const void* x;           // rows of K values, or codes' own type
  int64_t x_stride;        // elements
  const uint8_t* w;
  const float* ws;         // e4m3: scales [experts, ceil(N / 128), ceil(K / 128)]
  void* y;                 // [routes, N]
  int64_t w_expert;        // bytes from expert to expert
  int N, K;                // gated: N the width of h
  int R;                   // rows of y
  int act;
  float* gu;               // gated: the sums [R, 2 N] (NULL: not kept)
  const int32_t* ids;      // route r's expert (at most 64 of them): its row of x is r / top_k
  int top_k;
  Segments seg;            // without ids: rows by expert; offsets NULL: one matrix for all rows
  const int32_t* perm;     // with segments: row p's row of x is perm[p] / top_k, its place in y perm[p] (NULL: p)
  int row_tiles;           // blocks that share a tile of x's rows
};

// The codes of 128 values of a row, the lane's chunks of x (elements 16 q4 on, 64 + 16 q4 on) of lanes l16 + 16 q4,
// and their scale: a = max(|x|, 2^-116), x f32(448 / a) rounded to e4m3, f32(a / 448).
template <typename X, int XC>
__device__ __forceinline__ float quantise_unit(const u32x4_t (&x)[XC], u32x4_t codes[2]) {
  float v[32];
  unpack_chunks<X>(x, v);
  float top = 0x1p-116f;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(v[i]));
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const float r = 448.0f / top;
#pragma unroll
  for (int i = 0; i < 8; ++i) codes[i / 4][i % 4] = e4m3x4(v[4 * i] * r, v[4 * i + 1] * r, v[4 * i + 2] * r, v[4 * i + 3] * r);
  return top / 448.0f;
}

// FP8: e4m3 rows of w against rows of type X, quantised on the way; else rows of X's type.
template <typename X, bool FP8, bool GATED, int CT, int NRF, int WK, int WR>
__global__ __launch_bounds__(64 * WK * WR) void prod_rows(RowsArgs a) {
  using S = typename X::S;
  static_assert(!FP8 || !GATED, "");
  constexpr int ES = FP8 ? 1 : X::ES;                 // bytes of an element of w
  constexpr int UE = 128 / ES;                        // elements of a unit
  constexpr int XC = UE * X::ES / 64;                 // chunks of x a lane a unit
  constexpr int COLS = 16 * CT, MINE = GATED ? 8 * NRF : 16 * NRF, OUT = MINE * WR;  // rows of y a wave, a block
  constexpr int DEPTH = CT * NRF == 1 ? 4 : 2;        // units on their way at once
  __shared__ float red[WK][WR * NRF * CT * 4][64];
  __shared__ int list[64];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q4 = lane >> 4, wk = wave % WK, wr = wave / WK;
  const int tile = blockIdx.x / a.row_tiles, n0 = (blockIdx.x - tile * a.row_tiles) * OUT, nw = n0 + wr * MINE;

  // the block's expert and rows
  int expert, row0 = 0, rows;
  if (a.ids) {
    const int mine = lane < a.R ? a.ids[lane] : -1;
    expert = __builtin_amdgcn_readlane(mine, tile);  // tile: a route
    if (expert < 0 || expert >= a.seg.E) {
      expert = -1, rows = 1;
      if (wave == 0 && lane == 0) list[0] = tile;
    } else {
      const uint64_t same = __ballot(mine == expert);
      const int rank = __popcll(same & ((1ull << tile) - 1));
      if (rank % COLS) return;  // a block before has this route among its columns
      const int at = __popcll(same & ((1ull << lane) - 1)) - rank;
      if (wave == 0 && (same >> lane & 1) && at >= 0 && at < COLS) list[at] = lane;
      rows = min(__popcll(same) - rank, COLS);
    }
    __syncthreads();
  } else if (a.seg.offsets) {
    int mine;
    const int total = count_tiles(a.seg, COLS, mine);
    if (tile >= total) return;
    const RowTile t = find_tile(a.seg, COLS, tile, mine);
    if (!t.there) return;
    expert = t.expert, row0 = t.row0, rows = t.rows;
  } else {
    expert = 0, row0 = tile * COLS, rows = min(COLS, a.R - row0);
  }
  // column c's row of x, and its row of y
  auto out_row = [&](int c) {
    if (a.ids) return list[c];
    if (!a.perm) return row0 + c;
    const int p = a.perm[row0 + c];
    return p >= 0 ? p : ~p;
  };

  f32x4_t acc[NRF][CT] = {};
  if (expert >= 0) {
    const uint8_t* xr[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const int r = out_row(min(16 * t + l16, rows - 1));
      xr[t] = (const uint8_t*)a.x + (int64_t)(a.ids || a.perm ? r / a.top_k : r) * a.x_stride * X::ES;
    }
    const uint8_t* rows_w[NRF];
    const float* ws[NRF];
    const int units = (a.K + UE - 1) / UE;
#pragma unroll
    for (int f = 0; f < NRF; ++f) {
      int n;
      if constexpr (GATED) n = min(nw + 8 * f + (l16 & 7), a.N - 1) + (l16 >> 3) * a.N;
      else n = min(nw + 16 * f + l16, a.N - 1);
      rows_w[f] = a.w + expert * a.w_expert + (int64_t)n * a.K * ES;
      if constexpr (FP8) ws[f] = a.ws + ((int64_t)expert * ((a.N + 127) / 128) + min(nw + 16 * f, a.N - 1) / 128) * units;
    }
    struct Unit {
      u32x4_t w[NRF][2], x[CT][XC];
      float s[NRF];
    };
    // chunk c of a lane's row of w: bytes 64 c + 16 q4 of the unit; of x the same elements
    auto load = [&](int u, Unit& v) {
      const int64_t k = (int64_t)u * UE;
      constexpr int CE = 16 / ES;  // elements of a chunk of w
      if (k + UE <= a.K) {
#pragma unroll
        for (int f = 0; f < NRF; ++f)
#pragma unroll
          for (int c = 0; c < 2; ++c) v.w[f][c] = gload<u32x4_a1_t>(rows_w[f] + (k + 4 * CE * c + CE * q4) * ES);
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int c = 0; c < XC; ++c)
            v.x[t][c] = gload<u32x4_a1_t>(xr[t] + (k + 4 * CE * (c / (XC / 2)) + CE * q4) * X::ES + 16 * (c % (XC / 2)));
      } else {
#pragma unroll
        for (int f = 0; f < NRF; ++f)
#pragma unroll
          for (int c = 0; c < 2; ++c) v.w[f][c] = load_chunk<ES>(rows_w[f], k + 4 * CE * c + CE * q4, a.K);
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int c = 0; c < XC; ++c)
            v.x[t][c] = load_chunk<X::ES>(xr[t], k + 4 * CE * (c / (XC / 2)) + CE * q4 + X::EPC * (c % (XC / 2)), a.K);
      }
      if constexpr (FP8) {
#pragma unroll
        for (int f = 0; f < NRF; ++f) v.s[f] = gload<float>(ws[f] + u);
      }
    };
    auto compute = [&](const Unit& v) {
      float most[NRF];
      if constexpr (FP8) {
#pragma unroll
        for (int f = 0; f < NRF; ++f) most[f] = most_product(v.s[f]);
      }
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        if constexpr (FP8) {
          u32x4_t codes[2];
          const float s = quantise_unit<X>(v.x[t], codes);
          f32x4_t c[NRF];
#pragma unroll
          for (int f = 0; f < NRF; ++f) c[f] = mma_block<std::is_same<X, F32>::value>(v.w[f], codes);
#pragma unroll
          for (int f = 0; f < NRF; ++f) {
            asm volatile("" : "+v"(c[f]));  // read in the products' block: see settle()
            const float sc = scales_product(s, v.s[f], most[f]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[f][t][r] = __builtin_fmaf(c[f][r], sc, acc[f][t][r]);
          }
        } else {
#pragma unroll
          for (int f = 0; f < NRF; ++f)
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[f][t] = X::mma16(v.w[f][c], v.x[t][c], acc[f][t]);
        }
      }
    };
    // the wave's units, DEPTH of them on their way
    const int mine = units > wk ? (units - wk + WK - 1) / WK : 0;
    Unit ring[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
      if (i < mine) load(wk + WK * i, ring[i]);
    for (int i = 0; i < mine; i += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        if (i + d >= mine) break;
        compute(ring[d]);
        if (i + d + DEPTH < mine) load(wk + WK * (i + d + DEPTH), ring[d]);
      }
    }
    settle(acc);
#pragma unroll
    for (int f = 0; f < NRF; ++f)
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wk][((wr * NRF + f) * CT + t) * 4 + r][lane] = acc[f][t][r];
  }
  __syncthreads();

  // thread by thread one output: column c, row n of the block's
  auto sum = [&](int f, int row, int c) {  // of the fragment's row 0 .. 15
    const int at = (f * CT + (c >> 4)) * 4 + (row & 3), l = 16 * (row >> 2) + (c & 15);
    float s = 0;
#pragma unroll
    for (int i = 0; i < WK; ++i) s += red[i][at][l];
    return s;
  };
  for (int o = tid; o < OUT * rows; o += 64 * WK * WR) {
    const int c = o / OUT, n = o - c * OUT;
    if (n0 + n >= a.N) continue;
    const int64_t at = out_row(c);
    float v = 0;
    if constexpr (GATED) {
      float g = 0, u = 0;
      if (expert >= 0) g = sum(n >> 3, n & 7, c), u = sum(n >> 3, 8 + (n & 7), c), v = act_of<S>(a.act, g) * u;
      if (a.gu) {
        a.gu[at * 2 * a.N + n0 + n] = g;
        a.gu[at * 2 * a.N + a.N + n0 + n] = u;
      }
    } else if (expert >= 0) {
      v = sum(n >> 4, n & 15, c);
    }
    ((S*)a.y)[at * a.N + n0 + n] = (S)v;
  }
}

// Tiles of 256 x 256 by 8 waves (LARGE), of 128 x 256 by 8 waves with a step more of loads on their way (DEEP), of 128 x 128
// (SMALL) and 64 x 128 (LOW) by 4 waves, of which two and three blocks share a CU.
enum { TILE_SMALL = 0, TILE_DEEP = 1, TILE_LARGE = 2, TILE_LOW = 3 };
constexpr int tile_m(int size) { return size == TILE_LARGE ? 256 : size == TILE_LOW ? 64 : 128; }
constexpr int tile_n(int size) { return size == TILE_LARGE || size == TILE_DEEP ? 256 : 128; }

// The launches of one element type.
struct ProdTable {
  int (*tile)(int mode, bool gated, const TileArgs& a, int size, hipStream_t stream);
  int (*sum)(bool gated, const float* part, int splits, int64_t slice, int64_t rows, int64_t N, int act, void* out, float* gu,
             hipStream_t stream);
  int (*rows)(bool fp8, bool gated, const RowsArgs& a, int mean, hipStream_t stream);
  int (*fp8_tile)(const Fp8TileArgs& a, int size, hipStream_t stream);
  int (*quantise)(const void* x, int64_t stride, int64_t K, int64_t rows, const int32_t* end, uint8_t* codes, float* scales,
                  hipStream_t stream);
  int (*gated_grad)(const float* gu, const void* dh, int64_t dh_stride, int64_t N, int64_t rows, int act, void* dgu,
                    hipStream_t stream);
};
ProdTable prod_table_bf16();
ProdTable prod_table_f16();
ProdTable prod_table_f32();

}  // namespace ktmi
