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
  int splits;                    // blocks that share a tile's k; more than one: their sums go to part, one slice
  float* part;                   // of `slice` values each, in C's layout (gated: in gu's), and sum_parts adds them up
  int64_t slice;
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
// into LDS, for rows that start at multiples of 4 bytes (what a buffer load asks for); otherwise through registers, at
// any alignment.
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
  // to the operand's end; width: elements of a row in memory (TR). DIRECT: whole chunks, of which ENDS puts zeros for
  // those past kend; otherwise elements past it become zeros. A step that is not `there` is past every operand's end: its
  // loads are counted as the others and fetch nothing.
  template <bool ENDS>
  __device__ __forceinline__ void load(const uint8_t* base, int64_t bytes, int64_t stride, int step, bool there, int kend, int width,
                                       uint8_t* dst, int tid) {
    const int k0 = step * BK;
    if constexpr (DIRECT) {
      const int64_t at = TR ? (int64_t)k0 * stride : (int64_t)k0 * ES;
      const uint64_t left = (uint64_t)(bytes - at);  // at most 2^31 - 1 of them, in scalar instructions
      const uint32_t records = !there ? 0u : (uint32_t)(left >> 32) ? 0x7fffffffu : min((uint32_t)left, 0x7fffffffu);
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(base + at), (short)0, (int)records, 0x00020000);
      uint8_t* to = dst + __builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
      auto issue = [&](auto ends) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          uint32_t o = off[j];
          // past the operand's end, where a buffer load gives zeros
          if (decltype(ends)::value && k0 + first + (TR ? j * ROWS : 0) >= kend) o = 0x80000000u;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(to + j * THREADS * 16), 16,
                                                   (int)o, 0, 0, 0);
        }
      };
      if (!ENDS || k0 + BK <= kend) issue(std::false_type{});
      else issue(std::true_type{});
    } else if (k0 + BK <= kend && (!TR || (k0 + BK - 1) * stride + (int64_t)(width + EPC) * ES <= bytes)) {
      // whole chunks, at any alignment: across the end of a row (TR) they run into the next one, in columns that C
      // does not have, but never past the operand
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint8_t* p = TR ? base + (int64_t)(k0 + first + j * ROWS) * stride + min(col, width - 1) * ES
                              : base + (int64_t)off[j] * stride + (int64_t)(k0 + first) * ES;
        reg[j] = gload<u32x4_a1_t>(p);
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
  // A DIRECT operand's step that ends inside a chunk: chunk by chunk through registers.
  __device__ __forceinline__ void load_end(const uint8_t* base, int64_t stride, int step, int kend, int width, uint8_t* dst,
                                           int tid) {
    const int k0 = step * BK;
#pragma unroll 1
    for (int j = 0; j < NJ; ++j) {
      u32x4_t v = {0, 0, 0, 0};
      if constexpr (TR) {
        const int k = k0 + first + j * ROWS;
        if (k < kend && col < width) v = load_chunk<ES>(base + (int64_t)k * stride, col, width);
      } else {
        const int k = k0 + first;
        if (k < kend) v = load_chunk<ES>(base + (off[j] - 16 * (uint32_t)(first / EPC)), k, kend);
      }
      *(u32x4_t*)(dst + (j * THREADS + tid) * 16) = v;
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
  int split;
};

// The tile of this block. Blocks b, b + 8, .. run on one XCD: each XCD takes a run of neighbouring tiles, panels
// of up to 8 tiles of m by all of n, m fastest, so that its 32 blocks at a time share rows of both operands in
// its L2. (Gradients of w, which they write: n fastest, so that neighbours write whole rows.)
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
  const int64_t per = (total * a.splits + 7) / 8, at = blockIdx.x >> 3;
  int64_t t = (blockIdx.x & 7) * per + at;
  if (at >= per || t >= total * a.splits) return false;
  pl.split = a.splits > 1 ? (int)(t / total) : 0;
  t -= pl.split * total;
  int e = 0;
  if constexpr (MODE == PROD_DW) {
    e = (int)(t / ((int64_t)mt * nt));
    t -= (int64_t)e * mt * nt;
  }
  const int panel = (int)(t / (8 * (int64_t)nt)), in = (int)(t - (int64_t)panel * 8 * nt), high = min(8, mt - panel * 8);
  const int m = MODE == PROD_DW ? panel * 8 + in / nt : panel * 8 + in % high, n = MODE == PROD_DW ? in % nt : in / high;
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

// A wave's FR rows by NO fragments of FR columns of C, from the fragments' values v(i, r) to memory: through an LDS area of
// its own, so that every store writes whole runs of FR NO values (stored from the fragments a lane had 8 bytes of each
// row; rows by expert, 128 gradients of 1536 x 2048: 479 us instead of 364). A wave's LDS operations complete in order,
// so only the compiler is kept from moving them. Fragment (i): lane l holds row l % FR, columns 4 (l / FR) + r % 4 of
// every group of 256 / FR. C's rows start at(row) elements from c, at any address, for rows that are there; cols: columns that
// are. STREAM: past the caches, for what is read much later, if at all (gradients of w and the sums that a backward pass
// takes: 2047 tokens of 128 experts forward and backward 925 -> 871 us).
constexpr int STAGE_BYTES = 8192;
template <typename O, int FR, int NO, bool STREAM, typename F, typename A>
__device__ __forceinline__ void store_rows(uint8_t* stage, F v, O* c, A at, int rows, int cols, int lane) {
  constexpr int ROW = FR * NO * sizeof(O), CH = ROW / 16, EPC = 16 / sizeof(O), VALUES = FR * FR / 64;
  static_assert(FR * ROW <= STAGE_BYTES, "");
  const int q = lane / FR, l = lane % FR;
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int r = 0; r < VALUES; r += 4) {
      const typename vec4_of<O>::type o = {(O)v(i, r), (O)v(i, r + 1), (O)v(i, r + 2), (O)v(i, r + 3)};
      const int b = (FR * i + 256 / FR * (r / 4) + 4 * q) * (int)sizeof(O);  // in the row
      *(typename vec4_of<O>::type*)(stage + l * ROW + 16 * ((b / 16) ^ (l & (CH - 1))) + b % 16) = o;
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int t = 0; t < FR * CH / 64; ++t) {
    const int row = (t * 64 + lane) / CH, ch = lane % CH, left = cols - ch * EPC;
    const uint8_t* from = stage + row * ROW + 16 * (ch ^ (row & (CH - 1)));
    if (row >= rows || left <= 0) continue;
    O* to = c + at(row) + ch * EPC;  // (at(row) may read memory, which ends with the last row)
    if (left >= EPC) {
      gstore<STREAM>(to, *(const u32x4_t*)from);
    } else {
      for (int i = 0; i < left; ++i) to[i] = ((const O*)from)[i];
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A tile of C: WM x WN waves, each MF x NF fragments of 32 x 32, NB buffers of a step's operands in LDS. Q's rows are the
// matrix cores' rows and P's their columns, so that a lane has four neighbouring columns of C. A wave's 128 x 64 (LARGE)
// reads 6 KB of LDS for 8 products of 32 cycles, 64 x 64 reads 8 KB: at 2.4 GHz 230 and 307 GB/s a CU, of the 498 that reads of
// 16 bytes a lane reach.
// Bound by the matrix cores where tiles are whole (4096 x 4096 x 7168 bf16: forward 184 us, 1.3 PFLOP/s, gradient of x 215 to 230, of w
// 218; fp32 8192 cubed 141 TFLOP/s of 157), by HBM where an expert has few rows (128 experts of 1536 x 2048, up to 32 rows
// each: 153 us, 5.3 TB/s; their gradients 195 us, 4.1 TB/s).
template <typename T, int MODE, bool GATED, bool DIRECT, bool TAIL, int WM, int WN, int MF, int NF, int NB>
__global__ __launch_bounds__(64 * WM * WN, 2) void prod_tile(TileArgs a) {
  using S = typename T::S;
  constexpr int THREADS = 64 * WM * WN, BM = 32 * WM * MF, BN = 32 * WN * NF;
  constexpr bool PTR = MODE == PROD_DW, QTR = MODE != PROD_FWD;
  constexpr int CN = GATED ? BN / 2 : BN;  // columns of C in a tile
  static_assert(!GATED || (MODE == PROD_FWD && NF % 2 == 0), "");
  using P = TileOperand<T, PTR, DIRECT, BM, THREADS>;
  using Q = TileOperand<T, QTR, DIRECT, BN, THREADS>;
  constexpr int BUF = P::BYTES + Q::BYTES, BK = P::BK, SUBS = 4;
  constexpr int NLOAD = P::NJ + Q::NJ;  // of a thread a step
  static_assert(DIRECT || NB == 2, "");
  __shared__ __attribute__((aligned(16))) uint8_t lds[NB * BUF];

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
    const int all = (kend + BK - 1) / BK, share = (all + a.splits - 1) / a.splits;
    const int begin = pl.split * share, stop = min(all, begin + share);  // the block's steps
    // TAIL: k runs along rows and does not end with a whole step: the last one comes after the loop, whose loads need no
    // masks. (A kernel of its own: with this code in one for whole steps its loop, itself unchanged, took up to 15% longer.)
    static_assert(!TAIL || (DIRECT && MODE != PROD_DW), "");
    const bool tail = TAIL && stop == all && begin < stop;
    const int end = stop - tail;
    auto load = [&](int k, int buf) {
      const bool there = k < end;
      const int step = there ? k : end - 1;
      p.template load<MODE != PROD_FWD>(pb, pbytes, a.p_stride, step, there, kend, pw, lds + buf * BUF, tid);
      q.template load<MODE != PROD_FWD>(qb, qbytes, a.q_stride, step, there, kend, qw, lds + buf * BUF + P::BYTES, tid);
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
    if (begin < end) {
      // loads past the last step are issued too, and fetch nothing: the loop has no branches
      if constexpr (DIRECT) {
#pragma unroll
        for (int i = 0; i < NB; ++i) load(begin + i, i);
        __builtin_amdgcn_s_waitcnt(wait_vm((NB - 1) * NLOAD));
        block_barrier();
      } else {
        load(begin, 0);
        put(0);
        __builtin_amdgcn_s_waitcnt(WAIT_ALL);
        block_barrier();
        load(begin + 1, 1);
      }
      read(0, 0, 0);
      int buf = 0;
      for (int k = begin; k < end; ++k) {
        const int next = buf + 1 == NB ? 0 : buf + 1;
#pragma unroll
        for (int s = 0; s < SUBS - 1; ++s) {
          read(buf, s + 1, (s + 1) & 1);
          mma(s & 1);
        }
        // This step's last operands are in registers: its buffer is free for step k + NB once every wave is here. Step
        // k + 1's loads have to be there; those of the NB - 2 steps behind it stay on their way (counted: loads
        // end in order, and a thread has no others).
        put(next);
        __builtin_amdgcn_s_waitcnt(DIRECT ? wait_vm((NB - 2) * NLOAD) & ~(15 << 8) : WAIT_ALL);
        block_barrier();
        load(k + NB, buf);
        read(next, 0, 0);
        mma((SUBS - 1) & 1);
        buf = next;
      }
    }
    if (TAIL && tail) {
      __builtin_amdgcn_s_waitcnt(WAIT_ALL);
      block_barrier();
      p.load_end(pb, a.p_stride, end, kend, pw, lds, tid);
      q.load_end(qb, a.q_stride, end, kend, qw, lds + P::BYTES, tid);
      __builtin_amdgcn_s_waitcnt(WAIT_ALL);
      block_barrier();
#pragma unroll
      for (int s = 0; s < SUBS; ++s) {
        read(0, s, 0);
        mma(0);
      }
    }
    settle(acc);
  }

  // fragment (i, j): the lane holds row 32 j + lane % 32 of P's, rows 8 r / 4 + 4 (lane / 32) + r % 4 of Q's
  constexpr int NO = GATED ? NF / 2 : NF;  // fragments of C's columns
  S* c = (S*)a.c + (MODE == PROD_DW ? pl.expert * a.c_expert : 0);
  const int n0 = pl.n0 + 32 * NO * wn;  // the wave's first column
  float* const sums = a.splits > 1 ? a.part + pl.split * a.slice : a.gu;
  __builtin_amdgcn_s_waitcnt(WAIT_ALL);  // the last steps' loads, into the buffers that the waves stage their rows in
  block_barrier();
  uint8_t* stage = lds + wave * STAGE_BYTES;
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    const int m = 32 * (MF * wm + j), rows = pl.rows - m;
    if (rows <= 0) break;
    S* row = c + (int64_t)(pl.m0 + m) * a.c_stride + n0;
    const int cols = a.N - n0;
    auto at = [&](int i) { return i * a.c_stride; };
    if constexpr (GATED) {
      if (sums) {
        float* gu = sums + (int64_t)(pl.m0 + m) * 2 * a.N + n0;
        auto gu_at = [&](int i) { return (int64_t)i * 2 * a.N; };
        store_rows<float, 32, NO, true>(stage, [&](int i, int r) { return acc[i][j][r]; }, gu, gu_at, rows, cols, lane);
        store_rows<float, 32, NO, true>(stage, [&](int i, int r) { return acc[i + NO][j][r]; }, gu + a.N, gu_at, rows, cols, lane);
      }
      if (a.splits > 1) continue;
      store_rows<S, 32, NO, MODE == PROD_DW>(stage, [&](int i, int r) { return act_of<S>(a.act, acc[i][j][r]) * acc[i + NO][j][r]; }, row, at, rows,
                            cols, lane);
    } else if (a.splits > 1) {
      store_rows<float, 32, NO, false>(stage, [&](int i, int r) { return acc[i][j][r]; }, sums + (row - (S*)a.c), at, rows, cols, lane);
    } else {
      store_rows<S, 32, NO, MODE == PROD_DW>(stage, [&](int i, int r) { return acc[i][j][r]; }, row, at, rows, cols, lane);
    }
  }
}

}  // namespace ktmi
