// Products of many rows on the matrix cores: C[m, n] = sum over k of P[m, k] Q[n, k], in three forms:
//   forward       P rows of activations, Q a matrix of weights, both with k along their rows; rows by expert
//   gradient of x P rows of gradients, k along them; Q the weights again, k across them; rows by expert
//   gradient of w P rows of gradients, Q rows of activations, k (the rows) across both; an expert's rows
//                 are the k of its matrix
#pragma once
#include "prod_common.h"

namespace ktmi {

enum { PROD_FWD = 0, PROD_DX = 1, PROD_DW = 2 };

struct TileArgs {
  const uint8_t* p;
  const uint8_t* q;
  int64_t p_stride, q_stride;    // bytes from row to row
  int64_t p_bytes, q_bytes;      // of all of P, of one expert's Q (PROD_DW: of all of Q)
  int64_t q_expert;              // bytes from expert to expert
  void* c;
  int64_t c_stride, c_expert;    // elements
  int M, N, K;                   // PROD_DW: K the rows of all experts; gated: N the width of h
  Segments seg;                  // offsets NULL: one matrix for all rows
  float* gu;                     // gated: the sums, [M, 2 N] (NULL: not kept)
  int act;
};

// s_waitcnt operands: until at most n vector memory operations are outstanding, or no LDS ones
constexpr int wait_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }
constexpr int WAIT_ALL = 0;

// Workgroup barrier without the fence that __syncthreads has, which would wait for every load on its way.
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int STEP_BYTES = 128;  // of a row along k a step

// The place of a row's 16-byte chunk c in LDS, k along the rows of 128 bytes. The 64 banks hold two rows, and a read of
// 16 bytes a lane takes lanes 0-3, 12-15, 20-23 and 24-27 of 32 at once, then the others: 16 different places of
// the two rows are 16 lanes without a conflict. Lanes of 32 rows, one chunk (ES 2, 4): the rows are 16 different ones
// modulo 16. Lanes of 16 rows, a chunk for each 16 lanes (ES 1): rows 0-3 and 12-15 of one chunk, 4-11 of the next.
// (With the first rule for both, the 8-bit products had 5.1e7 conflict cycles in 1.1e8 of LDS.)
template <int ES>
__device__ __forceinline__ int row_slot(int row, int c) {
  return ES == 1 ? c ^ (row & 7) : c ^ (row & 7) ^ ((row >> 3) & 1);
}

// One operand's tile of W rows by 128 bytes of k, on its way from memory to LDS and from there to registers.
// TR: k runs across the rows in memory, and the tile is 128 / ES rows of W elements. DIRECT: loads straight
// into LDS, for rows that start at multiples of 16 bytes; otherwise through registers, at any alignment.
template <typename T, bool TR, bool DIRECT, int W, int THREADS>
struct TileOperand {
  static constexpr int ES = T::ES, EPC = T::EPC, BK = STEP_BYTES / ES;
  static constexpr int BYTES = W * STEP_BYTES, NJ = BYTES / 16 / THREADS;
  static constexpr int SLOTS = TR ? W * ES / 16 : 8;  // of a row in LDS
  static constexpr int ROWS = THREADS / SLOTS;        // rows that the block loads with one instruction a thread
  static_assert(NJ * THREADS * 16 == BYTES && (TR || ROWS % 16 == 0), "");
  static_assert(!TR || (SLOTS >= 16 && ROWS % 8 == 0), "the swizzle of a row is that of the row ROWS further on");

  // TR: two bits of the row (ES 2) or one (ES 4) move its chunks, so that the reads below have no conflicts
  static __device__ __forceinline__ int slot(int row, int c) {
    if constexpr (!TR) return row_slot<ES>(row, c);
    else if constexpr (ES == 2) return c ^ (4 * (row & 3));
    else return c ^ (8 * ((row >> 2) & 1));
  }

  uint32_t off[NJ];  // bytes from the tile's base (DIRECT), else rows
  int first;         // this thread's chunk: !TR its first k, TR the row (k) of load 0
  int col;           // TR: its first element of the row
  u32x4_t reg[DIRECT ? 1 : NJ];

  // row_of(i): the row in memory, from the base on, of the tile's row i (!TR; rows not there: one that is)
  template <typename F>
  __device__ __forceinline__ void init(int tid, int64_t stride, int col0, F row_of) {
    const int r = tid / SLOTS, c = slot(r, tid % SLOTS);
    if constexpr (TR) {
      first = r;
      col = col0 + c * EPC;
#pragma unroll
      for (int j = 0; j < NJ; ++j) off[j] = DIRECT ? (uint32_t)((r + j * ROWS) * (int)stride + col * ES) : 0;
    } else {
      first = c * EPC;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = row_of(r + j * ROWS);
        off[j] = DIRECT ? (uint32_t)row * (uint32_t)stride + 16 * c : (uint32_t)row;
      }
    }
  }

  // Loads step `step` of the k up to kend into dst (DIRECT) or registers. base: row 0, k = 0; bytes: from there
  // to the operand's end; width: elements of a row in memory (TR). Chunks past kend become zeros (ENDS: there are some).
  template <bool ENDS = true>
  __device__ __forceinline__ void load(const uint8_t* base, int64_t bytes, int64_t stride, int step, int kend, int width,
                                       uint8_t* dst, int tid) {
    const int k0 = step * BK;
    if constexpr (DIRECT) {
      const int64_t at = TR ? (int64_t)k0 * stride : (int64_t)k0 * ES;
      const uint64_t left = (uint64_t)(bytes - at);  // at most 2^31 - 1 of them, in scalar instructions
      const uint32_t records = (uint32_t)(left >> 32) ? 0x7fffffffu : min((uint32_t)left, 0x7fffffffu);
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(base + at), (short)0, (int)records, 0x00020000);
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      const bool whole = k0 + BK <= kend;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        uint32_t o = off[j];
        // past the operand's end, where a buffer load gives zeros
        if (ENDS && !whole && k0 + first + (TR ? j * ROWS : 0) >= kend) o = 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (__attribute__((address_space(3))) void*)(dst + (j * THREADS + wave * 64) * 16), 16, (int)o, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (TR) {
          const int k = k0 + first + j * ROWS;
          reg[j] = k < kend && col < width ? load_chunk<ES>(base + (int64_t)k * stride, col, width) : u32x4_t{0, 0, 0, 0};
        } else {
          const int k = k0 + first;
          reg[j] = k < kend ? load_chunk<ES>(base + (int64_t)off[j] * stride, k, kend) : u32x4_t{0, 0, 0, 0};
        }
      }
    }
  }
  // Puts what load() has in registers into dst.
  __device__ __forceinline__ void put(uint8_t* dst, int tid) {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) *(u32x4_t*)(dst + (j * THREADS + tid) * 16) = reg[j];
    }
  }

  // The chunk of rows 32 f + lane % 32 with the k of sub-step s: the lane's half h takes chunk 2 s + h.
  static __device__ __forceinline__ u32x4_t frag(const uint8_t* src, int row0, int f, int s, int lane) {
    const int h = lane >> 5, l = lane & 31;
    if constexpr (!TR) {
      const int row = row0 + 32 * f + l;
      return *(const u32x4_t*)(src + row * STEP_BYTES + 16 * row_slot<ES>(l, 2 * s + h));
    } else if constexpr (ES == 2) {
      // two transposing reads of four k each: in a group of 16 lanes, lane i gives the address of k i / 4,
      // elements 4 (i % 4) on, and gets the four k of element i
      const int i = lane & 15, z = i >> 2;
      const int c = (row0 + 32 * f + (l & 16)) / 8 + ((i & 3) >> 1);
      const uint8_t* p = src + (16 * s + 8 * h + z) * (W * ES) + 16 * (c ^ (4 * z)) + 8 * (i & 1);
      const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)p);
      const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(p + 4 * W * ES));
      const u32x2_t a = __builtin_bit_cast(u32x2_t, lo), b = __builtin_bit_cast(u32x2_t, hi);
      return u32x4_t{a[0], a[1], b[0], b[1]};
    } else {
      const int e = row0 + 32 * f + l, c = e / 4;
      const uint8_t* p = src + (8 * s + 4 * h) * (W * ES) + 16 * (c ^ (8 * h)) + 4 * (e & 3);
      u32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *(const uint32_t*)(p + i * (W * ES));
      return v;
    }
  }
};

// The result of an MFMA is there some cycles after the instruction. The compiler (ROCm 7.2) keeps a reader
// behind it by wait states, but not past a conditional branch, as at a loop's end: there the sums pass through
// this first. (The last of 16 passes needs 18; instructions in order.)
template <typename V, int N, int M>
__device__ __forceinline__ void settle(V (&acc)[N][M]) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(acc[0][0]));
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < M; ++j) asm volatile("" : "+v"(acc[i][j]));
}

// A tile's place: which rows and columns of which expert's C.
struct Place {
  int expert;    // -1: rows of no expert
  int m0, rows;  // rows of C (and of P unless PROD_DW), from m0 on
  int n0;
  int k0, k1;    // PROD_DW: the expert's rows
};

// The tile of this block. Blocks b, b + 8, .. run on one XCD: each XCD takes a run of neighbouring tiles, panels
// of up to 8 tiles of m by all of n, m fastest, so that its 32 blocks at a time share rows of both operands in
// its L2.
template <int MODE, int BM, int BN>
__device__ __forceinline__ bool place_of(const TileArgs& a, Place& pl) {
  const int nt = (a.N + BN - 1) / BN;
  int mt, mine = 0;
  int64_t total;
  if constexpr (MODE == PROD_DW) {
    mt = (a.M + BM - 1) / BM;
    total = (int64_t)mt * nt * (a.seg.offsets ? a.seg.E : 1);
  } else {
    mt = a.seg.offsets ? count_tiles(a.seg, BM, mine) : (a.M + BM - 1) / BM;
    total = (int64_t)mt * nt;
  }
  const int64_t per = (total + 7) / 8, at = blockIdx.x >> 3;
  int64_t t = (blockIdx.x & 7) * per + at;
  if (at >= per || t >= total) return false;
  int e = 0;
  if constexpr (MODE == PROD_DW) {
    e = (int)(t / ((int64_t)mt * nt));
    t -= (int64_t)e * mt * nt;
  }
  const int panel = (int)(t / (8 * (int64_t)nt)), in = (int)(t - (int64_t)panel * 8 * nt), high = min(8, mt - panel * 8);
  const int m = panel * 8 + in % high, n = in / high;
  pl.n0 = n * BN;
  if constexpr (MODE == PROD_DW) {
    pl.expert = e;
    pl.m0 = m * BM;
    pl.rows = min(BM, a.M - pl.m0);
    pl.k0 = a.seg.offsets ? a.seg.bound(e + 1) : 0;
    pl.k1 = a.seg.offsets ? max(a.seg.bound(e + 2), pl.k0) : a.K;
  } else if (a.seg.offsets) {
    const RowTile r = find_tile(a.seg, BM, m, mine);
    if (!r.there) return false;
    pl.expert = r.expert, pl.m0 = r.row0, pl.rows = r.rows;
  } else {
    pl.expert = 0, pl.m0 = m * BM, pl.rows = min(BM, a.M - pl.m0);
  }
  return true;
}

template <typename S>
__device__ __forceinline__ void store4(S* c, int n, int width, bool vec, f32x4_t v) {
  if (vec && n + 4 <= width) {
    typename vec4_of<S>::type o = {(S)v[0], (S)v[1], (S)v[2], (S)v[3]};
    *(typename vec4_of<S>::type*)(c + n) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < width) c[n + i] = (S)v[i];
  }
}

// WM x WN waves, each MF x NF fragments of 32 x 32.
template <typename T, int MODE, bool GATED, bool DIRECT, int WM, int WN, int MF, int NF>
__global__ __launch_bounds__(64 * WM * WN, 2) void prod_tile(TileArgs a) {
  using S = typename T::S;
  constexpr int THREADS = 64 * WM * WN, BM = 32 * WM * MF, BN = 32 * WN * NF;
  constexpr bool PTR = MODE == PROD_DW, QTR = MODE != PROD_FWD;
  constexpr int CN = GATED ? BN / 2 : BN;  // columns of C in a tile
  static_assert(!GATED || (MODE == PROD_FWD && NF % 2 == 0), "");
  using P = TileOperand<T, PTR, DIRECT, BM, THREADS>;
  using Q = TileOperand<T, QTR, DIRECT, BN, THREADS>;
  constexpr int BUF = P::BYTES + Q::BYTES, BK = P::BK, SUBS = 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * BUF];

  Place pl;
  if (!place_of<MODE, BM, CN>(a, pl)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;

  f32x16_t acc[NF][MF] = {};
  if (pl.expert >= 0) {
    const uint8_t *pb, *qb;
    int64_t pbytes, qbytes;
    int kend;
    P p;
    Q q;
    if constexpr (MODE == PROD_DW) {
      pb = a.p + pl.k0 * a.p_stride, pbytes = a.p_bytes - pl.k0 * a.p_stride;
      qb = a.q + pl.k0 * a.q_stride, qbytes = a.q_bytes - pl.k0 * a.q_stride;
      kend = pl.k1 - pl.k0;
      p.init(tid, a.p_stride, pl.m0, [](int) { return 0; });
      q.init(tid, a.q_stride, pl.n0, [](int) { return 0; });
    } else {
      pb = a.p + pl.m0 * a.p_stride, pbytes = a.p_bytes - pl.m0 * a.p_stride;
      qb = a.q + pl.expert * a.q_expert, qbytes = a.q_bytes;
      kend = a.K;
      const int last = pl.rows - 1;
      p.init(tid, a.p_stride, 0, [&](int i) { return min(i, last); });
      if constexpr (MODE == PROD_FWD) {
        if constexpr (GATED) {
          // a wave's first NF / 2 fragments are rows of the gate, the others the same rows of up
          q.init(tid, a.q_stride, 0, [&](int i) {
            const int w = i / (32 * NF), f = i / 32 % NF, up = f >= NF / 2;
            return min(pl.n0 + (w * (NF / 2) + f - up * (NF / 2)) * 32 + i % 32, a.N - 1) + up * a.N;
          });
        } else {
          // from the tile's first row on, so that 32 bits hold the offsets
          qb += (int64_t)pl.n0 * a.q_stride, qbytes -= (int64_t)pl.n0 * a.q_stride;
          const int end = a.N - 1 - pl.n0;
          q.init(tid, a.q_stride, 0, [&](int i) { return min(i, end); });
        }
      } else {
        q.init(tid, a.q_stride, pl.n0, [](int) { return 0; });
      }
    }
    // elements of a row in memory (operands with k across the rows)
    const int pw = a.M, qw = a.N;
    const int steps = (kend + BK - 1) / BK;
    auto load = [&](int k, int buf) {
      p.load(pb, pbytes, a.p_stride, k, kend, pw, lds + buf * BUF, tid);
      q.load(qb, qbytes, a.q_stride, k, kend, qw, lds + buf * BUF + P::BYTES, tid);
    };
    auto put = [&](int buf) {
      p.put(lds + buf * BUF, tid);
      q.put(lds + buf * BUF + P::BYTES, tid);
    };
    u32x4_t pf[2][MF], qf[2][NF];
    auto read = [&](int buf, int s, int to) {
#pragma unroll
      for (int i = 0; i < NF; ++i) qf[to][i] = Q::frag(lds + buf * BUF + P::BYTES, 32 * NF * wn, i, s, lane);
#pragma unroll
      for (int j = 0; j < MF; ++j) pf[to][j] = P::frag(lds + buf * BUF, 32 * MF * wm, j, s, lane);
    };
    auto mma = [&](int from) {
#pragma unroll
      for (int j = 0; j < MF; ++j)
#pragma unroll
        for (int i = 0; i < NF; ++i) acc[i][j] = T::mma32(qf[from][i], pf[from][j], acc[i][j]);
    };
    if (steps > 0) {
      // loads past the last step read that one again, into the buffer that is free: the loop has no branches
      const int last = steps - 1;
      load(0, 0);
      put(0);
      __builtin_amdgcn_s_waitcnt(WAIT_ALL);
      block_barrier();
      load(min(1, last), 1);
      read(0, 0, 0);
      for (int k = 0; k < steps; ++k) {
        const int buf = k & 1;
#pragma unroll
        for (int s = 0; s < SUBS - 1; ++s) {
          read(buf, s + 1, (s + 1) & 1);
          mma(s & 1);
        }
        // this step's last operands are in registers: its buffer is free for step k + 2 once every wave
        // is here, and step k + 1's loads, on their way since the last such place, have to be there
        put(buf ^ 1);
        __builtin_amdgcn_s_waitcnt(WAIT_ALL);
        block_barrier();
        load(min(k + 2, last), buf);
        read(buf ^ 1, 0, 0);
        mma((SUBS - 1) & 1);
      }
      settle(acc);
    }
  }

  // fragment (i, j): the lane holds row 32 j + lane % 32 of P's, rows 8 r / 4 + 4 (lane / 32) + r % 4 of Q's
  const int h = lane >> 5, l32 = lane & 31;
  S* c = (S*)a.c + (MODE == PROD_DW ? pl.expert * a.c_expert : 0);
  const bool vec = (a.c_stride | a.c_expert) % 4 == 0 && (uintptr_t)a.c % (4 * sizeof(S)) == 0;
  const bool gu_vec = a.N % 4 == 0;
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    const int m = 32 * (MF * wm + j) + l32;
    if (m >= pl.rows) continue;
    S* row = c + (int64_t)(pl.m0 + m) * a.c_stride;
#pragma unroll
    for (int i = 0; i < (GATED ? NF / 2 : NF); ++i) {
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int n = pl.n0 + 32 * ((GATED ? NF / 2 : NF) * wn + i) + 2 * r + 4 * h;
        f32x4_t v = {acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
        if constexpr (GATED) {
          const f32x16_t& u16 = acc[i + NF / 2][j];
          const f32x4_t u = {u16[r], u16[r + 1], u16[r + 2], u16[r + 3]};
          if (a.gu && n < a.N) {
            float* gu = a.gu + (int64_t)(pl.m0 + m) * 2 * a.N;
            store4(gu, n, a.N, gu_vec, v);
            store4(gu + a.N, n, a.N, gu_vec, u);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = act_of(a.act, v[x]) * u[x];
        }
        if (n < a.N) store4(row, n, a.N, vec, v);
      }
    }
  }
}

}  // namespace ktmi
