// Products in 8-bit floating point (e4m3) of many rows: y[m, n] = sum over blocks g of 128 k of xs[m, g] ws[n / 128, g]
// sum over k in g of x[m, k] w[n, k], on v_mfma_f32_16x16x128, whose k is one block.
//
// The matrix cores add e4m3 products of one instruction with about 16 bits below the largest (measured:
// codes of normal values 1.5e-5 of the sums' norm, any codes 1.1e-4 of the terms' sum at worst). For y in 16 bits, rounded
// at 2^-9 or 2^-12, that is enough; for y in fp32 the codes become bf16, which holds them exactly, and
// the sums are those of v_mfma_f32_16x16x32_bf16.
#pragma once
#include "prod_tile.h"

namespace ktmi {

struct E4M3 {
  using S = uint8_t;
  static constexpr int ES = 1, EPC = 16;
};

// codes 8 hi .. 8 hi + 7 of a chunk's 16 as bf16, whose bits are the high half of the fp32 value's
__device__ __forceinline__ bf16x8_t e4m3_to_bf16(u32x4_t c, int hi) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = (int)c[2 * hi + i];
    const u32x2_t a = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8(d, false));
    const u32x2_t b = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8(d, true));
    v[2 * i] = __builtin_amdgcn_perm(a[1], a[0], 0x07060302);
    v[2 * i + 1] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302);
  }
  return __builtin_bit_cast(bf16x8_t, v);
}

// The products of 16 rows by 16 over one block: lane l holds chunks l / 16 and 4 + l / 16 of row l % 16.
template <bool EXACT>
__device__ __forceinline__ f32x4_t mma_block(const u32x4_t a[2], const u32x4_t b[2]) {
  f32x4_t c = {0, 0, 0, 0};
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3_to_bf16(a[i / 2], i & 1), e4m3_to_bf16(b[i / 2], i & 1), c, 0, 0, 0);
  } else {
    const i32x8_t x = {(int)a[0][0], (int)a[0][1], (int)a[0][2], (int)a[0][3], (int)a[1][0], (int)a[1][1], (int)a[1][2], (int)a[1][3]};
    const i32x8_t y = {(int)b[0][0], (int)b[0][1], (int)b[0][2], (int)b[0][3], (int)b[1][0], (int)b[1][1], (int)b[1][2], (int)b[1][3]};
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);  // no scales: their operands 0
  }
  return c;
}

// Chunks of X's as fp32 values.
template <typename X, int XC>
__device__ __forceinline__ void unpack_chunks(const u32x4_t (&x)[XC], float (&v)[XC * X::EPC]) {
#pragma unroll
  for (int c = 0; c < XC; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = x[c][i];  // (a bit cast of a vector's element takes its first one)
      if constexpr (X::ES == 4) {
        v[4 * c + i] = __builtin_bit_cast(float, d);
      } else if constexpr (std::is_same<X, F16>::value) {
        v[8 * c + 2 * i] = half_bits_to_float((uint16_t)d);
        v[8 * c + 2 * i + 1] = half_bits_to_float((uint16_t)(d >> 16));
      } else {
        v[8 * c + 2 * i] = __builtin_bit_cast(float, d << 16);
        v[8 * c + 2 * i + 1] = __builtin_bit_cast(float, d & 0xffff0000u);
      }
    }
}

// four values as e4m3 codes, to nearest, ties to even
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int u = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, u, true);
}

// The product of a scale of x and one of w, held at fp32's largest number where it is past it: with an infinite one a block whose
// codes sum to 0 would add NaN in place of 0. most = most_product(ws), which for an infinite or NaN ws leaves the product as it
// is. (x that is not finite has NaN codes, whatever the scales.)
__device__ __forceinline__ float most_product(float ws) { return __builtin_isfinite(ws) ? 0x1.fffffep127f : fabsf(ws); }
__device__ __forceinline__ float scales_product(float xs, float ws, float most) { return __builtin_amdgcn_fmed3f(xs * ws, -most, most); }

struct Fp8TileArgs {
  const uint8_t* x;         // codes [rows, x_stride], quantised rows padded with zeros to whole blocks
  const float* xs;          // scales [blocks, xs_stride]
  int64_t x_stride, xs_stride, x_rows;
  const uint8_t* w;         // codes [experts, N, K]
  const float* ws;          // scales [experts, ceil(N / 128), blocks]
  void* y;                  // [M, N]
  int M, N, K;
  Segments seg;             // offsets NULL: one matrix for all rows
  const int32_t* perm;      // sorted routes: row p's codes are row perm[p] / top_k, its place in y perm[p] (its
  int top_k;                // complement without an expert); NULL: row p
  int splits;               // as TileArgs'
  float* part;
  int64_t slice;
};

// A tile of y: WM x WN waves, each MF x NF fragments of 16 x 16, two buffers in LDS; see prod_tile, whose step of 128 bytes is a
// block here. Bound by the matrix cores and the vector instructions that scale their sums, which the waves of a SIMD overlap
// only in part (8192 cubed: 52 and 35% of the cycles, at 1.96 GHz; 4096 x 4096 x 7168: 130 us with the quantisation, 1.85 PFLOP/s); of
// few rows a matrix by HBM (128 experts of 2048 x 2048, up to 16 rows each: 109 us, 4.9 TB/s).
template <typename S, bool EXACT, bool DIRECT, int WM, int WN, int MF, int NF>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tile(Fp8TileArgs a) {
  constexpr int THREADS = 64 * WM * WN, BM = 16 * WM * MF, BN = 16 * WN * NF;
  using P = TileOperand<E4M3, false, true, BM, THREADS>;
  using Q = TileOperand<E4M3, false, DIRECT, BN, THREADS>;
  constexpr int SCALES = P::BYTES + Q::BYTES, BUF = SCALES + THREADS * 4;  // rows, and a scale for each thread
  constexpr int NLOAD = P::NJ + Q::NJ + 1;  // of a thread a step
  static_assert(MF % 2 == 0, "");
  static_assert(BM % 64 == 0 && BM <= THREADS && 128 % (16 * NF) == 0 && BN % 128 == 0, "a wave's columns lie in one block");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * BUF];

  Place pl;
  TileArgs t = {};
  t.M = a.M, t.N = a.N, t.seg = a.seg, t.splits = a.splits;
  if (!place_of<PROD_FWD, BM, BN>(t, pl)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM, l16 = lane & 15, q4 = lane >> 4;
  const int blocks = (a.K + 127) / 128;

  f32x4_t acc[NF][MF] = {};
  const int share = (blocks + a.splits - 1) / a.splits, begin = pl.split * share, end_k = min(blocks, begin + share) - 1;
  if (pl.expert >= 0 && begin <= end_k) {
    const int last = pl.rows - 1;
    const uint8_t* pb = a.x;
    int64_t pbytes = a.x_rows * a.x_stride;
    int64_t sbase = 0;
    if (!a.perm) pb += pl.m0 * a.x_stride, pbytes -= pl.m0 * a.x_stride, sbase = pl.m0;
    auto row_of = [&](int i) {
      const int r = min(i, last);
      return a.perm ? a.perm[pl.m0 + r] / a.top_k : r;
    };
    P p;
    Q q;
    p.init(tid, a.x_stride, 0, row_of);
    const uint8_t* qb = a.w + ((int64_t)pl.expert * a.N + pl.n0) * a.K;
    const int64_t qbytes = (int64_t)(a.N - pl.n0) * a.K;
    const int end = a.N - 1 - pl.n0;
    q.init(tid, a.K, 0, [&](int i) { return min(i, end); });
    // The scales of a step go to LDS too, a value a thread: wave i < BM / 64 takes those of 64 rows, the next one those of
    // the columns' blocks, any other loads that one's again, which nobody reads (by scalar loads, which count with the
    // LDS reads, every step waited for them).
    constexpr int SW = BM / 64;
    static_assert(SW < WM * WN, "");
    const int col_blocks = (a.N + 127) / 128;
    const bool of_rows = wave < SW;
    const int col = min(pl.n0 / 128 + (lane & (BN / 128 - 1)), col_blocks - 1);
    const float* sb = of_rows ? a.xs + sbase : a.ws + ((int64_t)pl.expert * col_blocks + col) * blocks;
    const float* sp = sb + (of_rows ? row_of(tid) : 0);
    const int64_t s_step = of_rows ? a.xs_stride : 1;
    auto load = [&](int k, int buf) {
      uint8_t* b = lds + buf * BUF;
      __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(sp + k * s_step),
                                       (__attribute__((address_space(3))) void*)(b + SCALES + wave * 256), 4, 0, 0);
      p.template load<false>(pb, pbytes, a.x_stride, k, true, blocks * 128, 0, b, tid);
      q.template load<true>(qb, qbytes, a.K, k, true, a.K, 0, b + P::BYTES, tid);
    };
    auto put = [&](int buf) { q.put(lds + buf * BUF + P::BYTES, tid); };
    u32x4_t pf[2][2], qf[NF][2];
    float sx[2];
    // a lane's chunks of fragment 0 of x's and w's rows (fragment j is 16 rows on, with the same slots), its scale
    const int slot[2] = {16 * row_slot<1>(l16, q4), 16 * row_slot<1>(l16, 4 + q4)};
    const int p_at = (16 * MF * wm + l16) * STEP_BYTES, q_at = P::BYTES + (16 * NF * wn + l16) * STEP_BYTES;
    const int s_at = SCALES + 4 * (16 * MF * wm + l16), sw_at = SCALES + 4 * BM + 4 * (16 * NF * wn / 128);
    auto read_p = [&](int buf, int j, int to) {
      const uint8_t* b = lds + buf * BUF;
#pragma unroll
      for (int c = 0; c < 2; ++c) pf[to][c] = *(const u32x4_t*)(b + p_at + slot[c] + 16 * j * STEP_BYTES);
      sx[to] = *(const float*)(b + s_at + 64 * j);
    };
    auto read_q = [&](int buf, int i) {
#pragma unroll
      for (int c = 0; c < 2; ++c) qf[i][c] = *(const u32x4_t*)(lds + buf * BUF + q_at + slot[c] + 16 * i * STEP_BYTES);
    };
    // loads past the last step read that one again, into the buffer that is free: the loop has no branches
    load(begin, 0);
    if constexpr (DIRECT) {
      load(min(begin + 1, end_k), 1);
      __builtin_amdgcn_s_waitcnt(wait_vm(NLOAD));
      block_barrier();
    } else {
      put(0);
      __builtin_amdgcn_s_waitcnt(WAIT_ALL);
      block_barrier();
      load(min(begin + 1, end_k), 1);
    }
#pragma unroll
    for (int i = 0; i < NF; ++i) read_q(0, i);
    read_p(0, 0, 0);
    float sw = *(const float*)(lds + sw_at), most = most_product(sw);
    // The products of 16 rows of x go to c[0] and c[1] in turn: while the matrix cores work on one, the other's are
    // scaled and added, four instructions behind each of theirs. The asm keeps the compiler from moving that past
    // the branches below, with every block's sums in registers till then. A c is read behind the four products of the other,
    // which follow one another in the matrix cores' pipe, so it is there, past a branch too (see settle()).
    f32x4_t c[2][NF] = {};
    float s[2] = {0, 0};
    auto products = [&](int j, auto between) {
      const int cur = j & 1, prev = cur ^ 1, jp = (j + MF - 1) % MF;  // jp of the step before at first
      s[cur] = scales_product(sx[cur], sw, most);
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        c[cur][i] = mma_block<EXACT>(qf[i], pf[cur]);
        __builtin_amdgcn_sched_barrier(0);
        between(i);
        if (i > 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i - 1][jp][r] = __builtin_fmaf(c[prev][i - 1][r], s[prev], acc[i - 1][jp][r]);
          asm volatile("" : "+v"(acc[i - 1][jp]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[NF - 1][jp][r] = __builtin_fmaf(c[prev][NF - 1][r], s[prev], acc[NF - 1][jp][r]);
      asm volatile("" : "+v"(acc[NF - 1][jp]));
    };
    for (int k = begin; k <= end_k; ++k) {
      const int buf = (k - begin) & 1, next = buf ^ 1;
#pragma unroll
      for (int j = 0; j + 1 < MF; ++j) {
        read_p(buf, j + 1, (j + 1) & 1);
        products(j, [](int) {});
      }
      // The step's last rows are in registers, and its columns too: the buffer is free for step k + 2 once every wave is
      // here, and step k + 1's loads, on their way since the last such place, have to be there.
      put(next);
      __builtin_amdgcn_s_waitcnt(WAIT_ALL);
      block_barrier();
      load(min(k + 2, end_k), buf);
      products(MF - 1, [&](int i) { read_q(next, i); });
      read_p(next, 0, 0);
      sw = *(const float*)(lds + next * BUF + sw_at), most = most_product(sw);
    }
    settle(c);
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][MF - 1][r] = __builtin_fmaf(c[1][i][r], s[1], acc[i][MF - 1][r]);
  }

  // fragment (i, j): the lane holds row 16 j + lane % 16 of x's, rows 4 (lane / 16) + r of w's
  const int n0 = pl.n0 + 16 * NF * wn;
  auto place = [&](int m) {
    const int p = pl.m0 + m;
    return a.perm ? (pl.expert >= 0 ? a.perm[p] : ~a.perm[p]) : p;
  };
  __builtin_amdgcn_s_waitcnt(WAIT_ALL);  // the last steps' loads, into the buffers that the waves stage their rows in
  block_barrier();
  uint8_t* stage = lds + wave * STAGE_BYTES;
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    const int m = 16 * (MF * wm + j);
    if (m >= pl.rows) break;
    if (a.splits > 1) {  // (its rows in the order of y already)
      store_rows<float, 16, NF, false>(stage, [&](int i, int r) { return acc[i][j][r]; }, a.part + pl.split * a.slice + n0,
                                [&](int i) { return (int64_t)place(m + i) * a.N; }, pl.rows - m, a.N - n0, lane);
      continue;
    }
    store_rows<S, 16, NF, false>(stage, [&](int i, int r) { return acc[i][j][r]; }, (S*)a.y + n0,
                          [&](int i) { return (int64_t)place(m + i) * a.N; }, pl.rows - m, a.N - n0, lane);
  }
}

}  // namespace ktmi
