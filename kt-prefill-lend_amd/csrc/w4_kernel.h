// Products with 4-bit weights and group scales:
//   y[r, n] = sum_g s[e, n, g] * sum_{c in g} (q[e, n, c] - z[e, n, g]) * x[r, c]
//
// w4_mfma_kernel, for rows of a step (128 columns) or more, runs the matrix cores for any number of
// activation rows from one: v_mfma_f32_16x16x32 with 16 weight rows as its columns and 16
// activation rows as its rows. A wave takes 16 weight rows in steps of 128 columns, 16 bytes of
// codes a lane (lane l: row l % 16, column piece g = l / 16), eight steps ahead in a ring of registers.
//
// Codes become operands exactly: an e4m3 byte of value n < 16 is n * 2^-9 (the subnormals run on
// into the first normal binade), so one v_cvt_scalef32_pk turns two masked nibbles into two bf16 or
// f16 integers, seven instructions for eight codes. The zero point is a second product of the same
// activations with the constant -z, so the group's sum D = sum (q - z) x is exact but for fp32 sums, and
// acc += s D: no rounding of a weight. Infinite or NaN
// activations (and products past fp32) make that inf - inf: a block whose sums are not all finite
// runs again with q - z as the operand, which gives the plain sum's infinities and NaN. It takes the rows of x
// that had such sums from there, the others from the first run: what one row holds changes no bit of another's.
//
// fp32 activations are three bf16 parts (8 + 8 + 8 bits of the significand, cut, so that nothing
// overflows), each with a product of its own: exact but for parts below bf16's smallest number.
//
// The activations of the block's rows pass through LDS in column stages, values of each eight in the
// order 0 2 4 6 1 3 5 7 in which the nibbles come out; columns past the row's end are zeros there.
//
// What bounds it: large calls the weights' bytes, of which 3.8 TB/s come (18 experts of 4096 x 7168 bf16,
// 13 tokens: 72 us for 276 MB; a build of 95 us took 66 with nothing but its loads); small ones the chain
// from the ids to the loads to the sums (one row of 4096 x 7168 8.3 us; a build of 10.0 took 6.3 with
// nothing but its loads). What it took to get there, the former case: loads and products of a step at a
// time 115 us; both 64-byte halves of a row's line and the scales of eight steps asked for together 95;
// row tiles after each other on the same activations, no condition inside a turn of the ring, as many
// blocks as the chip holds 72. Many rows of x cost their passage through LDS: 4096 x 7168 at 16 rows 18
// us, at 64 rows 27.
#pragma once
#include <type_traits>

#include "kernels.h"

namespace ktmi {

namespace {

constexpr int W4_RING = 8;             // steps of codes in flight a wave, a turn of the ring
constexpr int W4_VMCNT0 = 0xF70;       // s_waitcnt operand: vector memory loads only
constexpr int W4_X_BYTES = 64 << 10;   // LDS for a stage's activations, about: two blocks a CU
constexpr int W4_CU_LDS = 160 << 10;
constexpr int W4_X_SPLIT = 136 << 10;  // where the blocks are few: one a CU

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// what the MFMA takes: bf16 for bf16 and fp32 activations, f16 for f16
template <typename T>
struct Operand {
  static __device__ __forceinline__ f32x4_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t codes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, HI));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return f2bf2(lo, hi); }
  static __device__ __forceinline__ float low(uint32_t w) { return bf2f((uint16_t)w); }
};
template <>
struct Operand<_Float16> {
  static __device__ __forceinline__ f32x4_t mfma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t codes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.0f, HI));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return (uint32_t)float_to_half_bits(lo) | (uint32_t)float_to_half_bits(hi) << 16;
  }
  static __device__ __forceinline__ float low(uint32_t w) { return half_bits_to_float((uint16_t)w); }
};

// eight codes of a word as operand values in the order 0 2 4 6 1 3 5 7
template <typename T>
__device__ __forceinline__ u32x4_t decode(uint32_t w) {
  using O = Operand<T>;
  const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
  return u32x4_t{O::template codes<false>(lo), O::template codes<true>(lo), O::template codes<false>(hi),
                 O::template codes<true>(hi)};
}
// the same less the zero point (negz = -z), exact: both are integers below 2^8
template <typename T>
__device__ __forceinline__ u32x4_t decode_plain(uint32_t w, float negz) {
  using O = Operand<T>;
  const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.0f, false);
  const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.0f, true);
  const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.0f, false);
  const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.0f, true);
  return u32x4_t{O::pack(a[0] + negz, a[1] + negz), O::pack(b[0] + negz, b[1] + negz), O::pack(c[0] + negz, c[1] + negz),
                 O::pack(d[0] + negz, d[1] + negz)};
}

// a lane's 16 bytes shifted down by n bytes, 0 <= n < 16, zeros from above
__device__ __forceinline__ u32x4_t shift_down(u32x4_t w, int n) {
  if (n & 8) w = u32x4_t{w[2], w[3], 0, 0};
  if (n & 4) w = u32x4_t{w[1], w[2], w[3], 0};
  return u32x4_t{__builtin_amdgcn_alignbyte(w[1], w[0], n & 3), __builtin_amdgcn_alignbyte(w[2], w[1], n & 3),
                 __builtin_amdgcn_alignbyte(w[3], w[2], n & 3), __builtin_amdgcn_alignbyte(0, w[3], n & 3)};
}

__device__ __forceinline__ float scale_as_float(const void* s, int dtype, int64_t i) {
  if (dtype == KTMI_F32) return gload<float>((const float*)s + i);
  const uint16_t v = gload<uint16_t>((const uint16_t*)s + i);
  return dtype == KTMI_F16 ? half_bits_to_float(v) : bf2f(v);
}

// One launch's plan. A block's WR * KS waves: WR sets of 16 weight rows, the KS waves of a set split
// its columns. With KS = 1 a block takes `deep` tiles of 16 WR weight rows after each other against the
// same activations in LDS. Items: (expert, pass of up to 16 MT of its activation rows).
struct W4Plan {
  int blocks;   // of an item
  int deep;     // row tiles a block
  int steps;    // steps a wave over all columns
  int x_bytes;  // LDS of a stage's activations; the row tiles' sums between stages come behind it
};

// Columns of MFMA m of a step for lane group g, relative to the step: base + fixed, chosen so that one
// scale covers each MFMA. SPS scales a step: 1 (groups of whole steps): words as loaded; 2: words
// swapped between the wave's halves; 4: words transposed between the four lane groups.
template <int SPS>
__device__ __forceinline__ int x_base(int g) {
  return SPS == 1 ? 32 * g : SPS == 2 ? 32 * (g & 1) + 16 * (g >> 1) : 8 * g;
}
template <int SPS>
constexpr int x_fixed(int m) {
  return SPS == 1 ? 8 * m : SPS == 2 ? 64 * (m >> 1) + 8 * (m & 1) : 32 * m;
}
template <int SPS>
__device__ __forceinline__ void regroup(uint32_t (&w)[4]) {
  if constexpr (SPS == 4) {
    const auto a = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
    w[0] = a[0], w[1] = a[1], w[2] = b[0], w[3] = b[1];
  }
  if constexpr (SPS >= 2) {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    w[0] = a[0], w[2] = a[1], w[1] = b[0], w[3] = b[1];
  }
}

// inclusive sum over the wave's lanes by DPP: inside each row of 16 lanes, then the rows' last lanes on
__device__ __forceinline__ int wave_sum_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr 4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ void w4_wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The block's item: expert e, its rows of x at src[0 .. m) and of y at dst[0 .. m); returns m, 0 for
// none. Every wave writes the same lists and reads what it wrote: no barrier.
template <typename T, int MT>
__device__ __forceinline__ int find_item(const W4Args& a, int item, int& e, const T** src, T** dst) {
  const int lane = threadIdx.x & 63;
  constexpr int ROWS = 16 * MT;
  if (a.ids) {
    // route `item`: the first of every ROWS routes of its expert takes them
    const int id = lane < a.n_routes ? a.ids[lane] : -1;
    e = __builtin_amdgcn_readlane(id, item);
    if (e < 0 || e >= a.n_experts) return 0;
    const uint64_t same = __ballot(id == e);
    const int rank = __popcll(same & ((1ull << item) - 1ull));
    if (rank % ROWS) return 0;
    const int mine = __popcll(same & ((1ull << lane) - 1ull)) - rank;
    if (id == e && mine >= 0 && mine < ROWS) {
      src[mine] = (const T*)a.x + lane / (int)a.top_k * a.x_stride;
      dst[mine] = (T*)a.y + lane * a.rows;
    }
    w4_wave_fence();
    const int m = __popcll(same) - rank;
    return m < ROWS ? m : ROWS;
  }
  int first = 0, m = (int)a.n_routes, pass = item;
  e = 0;
  if (a.offsets) {
    // the item-th pass over the experts in order, 128 experts at a time, two a lane
    const int R = (int)a.n_routes, E = (int)a.n_experts;
    int before = 0;
    bool found = false;
    for (int e0 = 0; e0 < E && !found; e0 += 128) {
      int at[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int x = a.offsets[e0 + 2 * lane + i < E ? e0 + 2 * lane + i : E];
        at[i] = x < 0 ? 0 : x < R ? x : R;
      }
      const int n0 = at[1] > at[0] ? at[1] - at[0] : 0, n1 = at[2] > at[1] ? at[2] - at[1] : 0;
      const int p0 = (n0 + ROWS - 1) / ROWS, p1 = (n1 + ROWS - 1) / ROWS;
      const int end = before + wave_sum_upto(p0 + p1), start = end - p0 - p1;
      const uint64_t hit = __ballot(item >= start && item < end);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        const int s = __builtin_amdgcn_readlane(start, l), q = __builtin_amdgcn_readlane(p0, l);
        const bool second = item >= s + q;
        first = __builtin_amdgcn_readlane(second ? at[1] : at[0], l);
        m = __builtin_amdgcn_readlane(second ? n1 : n0, l);
        pass = item - s - (second ? q : 0);
        e = e0 + 2 * l + second;
        found = true;
      }
      before = __builtin_amdgcn_readlane(end, 63);
    }
    if (!found) return 0;
  }
  first += pass * ROWS;
  m -= pass * ROWS;
  if (m > ROWS) m = ROWS;
  if (lane < m) {
    const int r = a.perm ? a.perm[first + lane] : first + lane;
    src[lane] = (const T*)a.x + (a.perm ? r / (int)a.top_k : r) * a.x_stride;
    dst[lane] = (T*)a.y + r * a.rows;
  }
  w4_wave_fence();
  return m > 0 ? m : 0;
}

template <typename T, int SPS, bool S4, bool Z, int MT, int KS, int WR>
__global__ __launch_bounds__(64 * KS * WR) void w4_mfma_kernel(W4Args a, W4Plan p) {
  using O = Operand<T>;
  constexpr int PLANES = std::is_same<T, float>::value ? 3 : 1;
  constexpr int RB = 16 * WR, TH = 64 * KS * WR;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ const T* src[16 * MT];
  __shared__ T* dst[16 * MT];
  __shared__ uint32_t again;  // rows of x whose sums were not all finite, one a bit
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / p.blocks, n0 = (blockIdx.x - item * p.blocks) * p.deep * RB;
  const int rows_left = (int)(a.rows - n0 < RB * p.deep ? a.rows - n0 : RB * p.deep);
  T* y = (T*)a.y;
  int e;
  const int m = find_item<T, MT>(a, item, e, src, dst);

  // rows of no expert are zero: route `item` by its id, or every items-th row outside the segments
  // (of unsorted ids: the routes that the order puts there)
  auto zero_rows = [&]() {
    auto zero = [&](int64_t r) {
      for (int n = threadIdx.x; n < rows_left; n += TH) y[r * a.rows + n0 + n] = (T)0.0f;
    };
    if (a.ids) {
      if (e < 0 || e >= a.n_experts) zero(item);
    } else if (a.offsets) {
      const int items = gridDim.x / p.blocks, begin = a.offsets[0], end = a.offsets[a.n_experts];
      for (int64_t r = item; r < begin && r < a.n_routes; r += items) zero(r);
      for (int64_t r = (end > 0 ? (int64_t)end : 0) + item; r < a.n_routes; r += items) zero(a.perm ? ~a.perm[r] : r);
    }
  };
  if (m == 0) return zero_rows();
  const int mg = (m + 15) / 16;  // groups of 16 activation rows

  const int cols = (int)a.cols, half = (cols + 1) / 2;
  const int row = lane & 15, g = lane >> 4;
  const int kw = wave % KS, rb = 16 * (wave / KS) + row;  // the wave's part of the columns, the lane's weight row
  const int groups = (int)((a.cols + a.group - 1) / a.group);
  const int64_t first_row = e * a.rows + n0;
  const uint32_t neg8 = O::pack(-8.0f, -8.0f);
  // the weights from the block's first row on as buffers. A load's words past a buffer's end return
  // zeros and take no memory access (of a buffer of no bytes: all), so the number of loads in flight
  // is the same for any number of steps.
  auto buffer = [](const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)bytes, 0x00020000);
  };
  constexpr int SS = S4 ? 4 : 2;
  const uint8_t* codes = a.codes + first_row * half;
  const uint8_t* scales = (const uint8_t*)a.scales + first_row * groups * SS;
  const uint8_t* zeros = a.zeros + first_row * groups;
  // scales from there to the last expert's last row, or as many as a buffer reaches
  int64_t rest = (a.n_experts * a.rows - first_row) * groups;
  rest = rest < 0x7FFFFFFF / SS ? rest : 0x7FFFFFFF / SS;
  // the lane's row of tile t (past the last row: the last)
  auto row_of = [&](int t) { return t * RB + rb < rows_left ? t * RB + rb : rows_left - 1; };
  const int total = (cols + W4_STEP - 1) / W4_STEP;  // steps of a row
  // Codes past a row's end meet zeros of x: the next row's, or the zeros that a buffer's end gives for
  // whole words. Rows that do not end with a word take the plain loop, which loads up to their end.
  const bool ragged = half & 3;
  auto group_of = [&](int s) { return SPS > 1 ? SPS * s : a.group == W4_STEP ? s : s / (int)(a.group / W4_STEP); };
  auto pack_zero = [&](uint32_t z) { return O::pack(-(float)z, -(float)z); };
  // The scales and zero points of the W4_RING steps from s on of the row with `at` scales before it,
  // packed as in memory. Where the turn of the wave's last row ends inside the weights, 16 bytes at a
  // time, past the row's end too; there, and for groups of several steps, one by one.
  constexpr int TURN = W4_RING * SPS, PER = 4 / SS;
  struct Turn {
    uint32_t s[TURN / PER], z[TURN / 4];
  };
  auto load_turn = [&](int at, int last_at, int s, bool in) {
    Turn t;
    const auto sb = buffer(scales, in ? rest * SS : 0), zb = buffer(zeros, in ? rest : 0);
    if ((SPS > 1 || a.group == W4_STEP) && last_at + SPS * s + TURN <= rest) {  // uniform
      const int i = at + SPS * s;
#pragma unroll
      for (int j = 0; j < TURN / PER; j += 4) {
        const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(sb, SS * i + 4 * j, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) t.s[j + q] = v[q];
      }
      if constexpr (Z) {
#pragma unroll
        for (int j = 0; j < TURN / 4; j += 2) {
          const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(zb, i + 4 * j, 0, 0);
          t.z[j] = v[0], t.z[j + 1] = v[1];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < TURN; ++j) {
        const int i = at + group_of(s + j / SPS) + j % SPS;
        if constexpr (S4) {
          t.s[j] = __builtin_amdgcn_raw_buffer_load_b32(sb, 4 * i, 0, 0);
        } else {
          const uint32_t u = __builtin_amdgcn_raw_buffer_load_b16(sb, 2 * i, 0, 0);
          t.s[j / 2] = j % 2 ? t.s[j / 2] | u << 16 : u;
        }
        if constexpr (Z) {
          const uint32_t u = __builtin_amdgcn_raw_buffer_load_b8(zb, i, 0, 0);
          t.z[j / 4] = j % 4 ? t.z[j / 4] | u << (8 * (j % 4)) : u;
        }
      }
    }
    return t;
  };
  // element j of a turn in fp32; of a turn that reaches past the row's last group, 0 for those past it
  auto scale_of = [&](const Turn& t, int j) {
    const uint32_t u = t.s[j / PER];
    if constexpr (S4) return __builtin_bit_cast(float, u);
    const uint16_t h = (uint16_t)(u >> 16 * (j % PER));
    return a.scale_dtype == KTMI_F16 ? half_bits_to_float(h) : bf2f(h);
  };
  auto drop_past = [&](Turn& t, int s) {
#pragma unroll
    for (int j = 0; j < TURN; ++j) {
      const int step = s + j / SPS;
      if (step >= total || group_of(step) + j % SPS >= groups)  // uniform
        t.s[j / PER] &= PER == 1 ? 0u : j % 2 ? 0xFFFFu : 0xFFFF0000u;
    }
  };
  // steps a wave of a stage: all, or as many as the activations' room takes
  int per_stage = ((p.x_bytes / (PLANES * m) - 16) / (2 * W4_STEP * KS));
  per_stage = per_stage < p.steps ? per_stage : p.steps;
  const int stage = per_stage * KS * W4_STEP, pitch = 2 * stage + 16, plane = pitch * m;
  int xr[MT];  // the lane's activation row of each group in LDS (one past the last reads the last)
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = (16 * t + row < m ? 16 * t + row : m - 1) * pitch + 2 * x_base<SPS>(g);

  // the activations of the columns from k0, the loads of a batch ahead of its stores
  const int chunks = stage / 8;
  const float chunks_inv = 1.0f / (float)chunks;
  auto put = [&](int r, int c, const u32x4_t& v, int q) {
    *(u32x4_t*)(lds + q * plane + r * pitch + 16 * c) =
        u32x4_t{__builtin_amdgcn_perm(v[1], v[0], 0x05040100), __builtin_amdgcn_perm(v[3], v[2], 0x05040100),
                __builtin_amdgcn_perm(v[1], v[0], 0x07060302), __builtin_amdgcn_perm(v[3], v[2], 0x07060302)};
  };
  // eight fp32 values as three parts; a value that is not finite has one
  auto put3 = [&](int r, int c, const uint32_t (&u)[8]) {
    uint32_t part[3][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool finite = (u[j] & 0x7F800000u) != 0x7F800000u;
      const uint32_t h = finite || !(u[j] & 0x007FFFFFu) ? u[j] & 0xFFFF0000u : 0x7FC00000u;
      const float r1 = finite ? __builtin_bit_cast(float, u[j]) - __builtin_bit_cast(float, h) : 0.0f;
      const uint32_t mid = __builtin_bit_cast(uint32_t, r1) & 0xFFFF0000u;
      const float r2 = r1 - __builtin_bit_cast(float, mid);
      const uint32_t all[3] = {h, mid, __builtin_bit_cast(uint32_t, r2)};
#pragma unroll
      for (int q = 0; q < 3; ++q) part[q][j / 2] = j % 2 ? (all[q] & 0xFFFF0000u) | part[q][j / 2] : all[q] >> 16;
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) put(r, c, u32x4_t{part[q][0], part[q][1], part[q][2], part[q][3]}, q);
  };
  constexpr int XB = PLANES == 1 ? 8 : 4;  // a thread's loads of a batch, the second half only where there are so many
  const int x_all = m * chunks;
  struct Batch {
    u32x4_t v[XB][PLANES == 1 ? 1 : 2];
    int at[XB];  // row and chunk
  };
  // the thread's chunks from i0 on; past the last the last again
  auto fetch = [&](int k0, int i0) {
    Batch b;
    auto part = [&](int j) {
      const int i = i0 + j * TH < x_all ? i0 + j * TH : x_all - 1;
      const int r = (int)(((float)i + 0.5f) * chunks_inv), c = i - r * chunks, k = k0 + 8 * c;
      b.at[j] = r << 16 | c;
      const T* x = src[r] + (k < cols - 8 ? k : cols - 8);
      if constexpr (PLANES == 1) {
        b.v[j][0] = gload<u32x4_a2_t>(x);
      } else {
        b.v[j][0] = gload<u32x4_a4_t>(x);
        b.v[j][1] = gload<u32x4_a4_t>(x + 4);
      }
    };
#pragma unroll
    for (int j = 0; j < XB / 2; ++j) part(j);
    if (x_all > XB / 2 * TH)  // uniform
#pragma unroll
      for (int j = XB / 2; j < XB; ++j) part(j);
    return b;
  };
  auto store = [&](int k0, int i0, const Batch& b) {
    auto part = [&](int j) {
      const int r = b.at[j] >> 16, c = b.at[j] & 0xFFFF, k = k0 + 8 * c;
      if (i0 + j * TH < x_all && (k + 8 <= cols || k >= cols)) {
        const bool in = k < cols;
        if constexpr (PLANES == 1) {
          put(r, c, in ? b.v[j][0] : u32x4_t{0, 0, 0, 0}, 0);
        } else {
          uint32_t u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = in ? b.v[j][i / 4][i % 4] : 0u;
          put3(r, c, u);
        }
      }
    };
#pragma unroll
    for (int j = 0; j < XB / 2; ++j) part(j);
    if (x_all > XB / 2 * TH)
#pragma unroll
      for (int j = XB / 2; j < XB; ++j) part(j);
  };
  auto fill = [&](int k0, const Batch& b) {
    store(k0, threadIdx.x, b);
    for (int i0 = threadIdx.x + XB * TH; i0 < x_all; i0 += XB * TH) {
      store(k0, i0, fetch(k0, i0));
      __builtin_amdgcn_s_waitcnt(W4_VMCNT0);  // lanes without a store too: nothing is in flight past the loop
    }
    // the chunk that the rows end in, element by element
    const int k = cols & ~7;
    if ((cols & 7) && k >= k0 && k < k0 + stage && threadIdx.x < m) {
      const int r = threadIdx.x, c = (k - k0) / 8;
      const T* x = src[r] + k;
      if constexpr (PLANES == 1) {
        uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 7; ++j)
          if (k + j < cols) u[j / 2] |= (uint32_t)gload<uint16_t>(x + j) << (16 * (j % 2));
        put(r, c, u32x4_t{u[0], u[1], u[2], u[3]}, 0);
      } else {
        uint32_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = k + j < cols ? gload<uint32_t>(x + j) : 0u;
        put3(r, c, u);
      }
    }
  };

  f32x4_t acc[MT] = {};
  // step s, the at-th of the stage
  auto compute = [&](auto plain, const u32x4_t& raw, const float* scale, const uint32_t (&zz)[SPS], int at) {
    constexpr bool PLAIN = decltype(plain)::value;
    constexpr int J = 4 / SPS;
    uint32_t w[4] = {raw[0], raw[1], raw[2], raw[3]};
    regroup<SPS>(w);
#pragma unroll
    for (int sub = 0; sub < SPS; ++sub) {
      const u32x4_t zf = {zz[sub], zz[sub], zz[sub], zz[sub]};
      u32x4_t wf[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if constexpr (PLAIN)
          wf[j] = decode_plain<T>(w[sub * J + j], O::low(zz[sub]));
        else
          wf[j] = decode<T>(w[sub * J + j]);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t == 0 || t < mg) {  // uniform
          f32x4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int q = 0; q < PLANES; ++q) {
              const u32x4_t xv = *(const u32x4_t*)(lds + xr[t] + q * plane + 2 * W4_STEP * at + 2 * x_fixed<SPS>(sub * J + j));
              d = O::mfma(xv, wf[j], d);
              if constexpr (!PLAIN) d = O::mfma(xv, zf, d);
            }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(scale[sub], d[i], acc[t][i]);
          // the sums are taken here, in the block of their MFMAs: moved past the branch behind it, the
          // compiler left out the wait states between an MFMA and the reader of its result
          asm volatile("" : "+v"(acc[t]));
        }
      }
    }
  };
  const bool staged = per_stage < p.steps;  // in more than one stage: sums wait in LDS between them
  f32x4_t* sums = (f32x4_t*)(lds + p.x_bytes) + wave * MT * 64 + lane;
  uint32_t only = ~0u;  // rows of x whose sums are the plain run's
  auto out = [&](auto plain, int t) {  // the sums of row tile t
    if (t * RB + rb < rows_left)
#pragma unroll
      for (int q = 0; q < MT; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * q + 4 * g + i;
          if (r < m && (!decltype(plain)::value || (only >> r & 1)))
            *(__attribute__((address_space(1))) T*)(dst[r] + n0 + t * RB + rb) = (T)acc[q][i];  // global: a flat store drains the ring
        }
  };
  uint32_t bad = 0;  // the lane's sums that are not finite: 4 t + i of acc[t][i]
  auto run = [&](auto plain) {
    constexpr bool PLAIN = decltype(plain)::value;
    const int tiles = (rows_left + RB - 1) / RB;
    auto check = [&]() {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= fabsf(acc[t][i]) < __builtin_inff() ? 0u : 1u << (4 * t + i);
    };
    auto clear = [&]() {
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();
    for (int i0 = 0; i0 < p.steps; i0 += per_stage) {
      const int n = p.steps - i0 < per_stage ? p.steps - i0 : per_stage;
      const int first = KS * i0, s0 = first + kw * n;  // the stage's steps; the wave's are s0 .. s0 + n - 1
      // the activations' loads, the first steps', then the activations' stores
      const Batch b = fetch(first * W4_STEP, threadIdx.x);
      __builtin_amdgcn_sched_barrier(0);  // in this order
      const int valid = n < total - s0 ? n : total - s0;  // the wave's steps that the rows have
      // the ring runs on from turn to turn and tile to tile; steps past the valid ones are zeros or
      // others' codes, which no sum takes
      u32x4_t ring[W4_RING];
      auto codes_at = [&](int t, int i) { return row_of(t) * half + 64 * (s0 + i) + 16 * g; };
      auto load_step = [&](int at, int u, bool in) {
        return __builtin_amdgcn_raw_buffer_load_b128(buffer(codes, in ? rows_left * (int64_t)half : 0), at + 64 * u, 0, 0);
      };
      // no load for a step past the wave's part of a stage, but for the second of a pair: one row of 7168 x 2048
      // 7.0 us (7.3 with them), 512 rows of 102 experts of 2048 x 768 25 (27)
      auto wanted = [&](int i, int u) { return i + u < n; };
      auto turn_of = [&](int t, int i) {  // from step i of tile t; past the tile's end: the next tile's first
        const bool on = i >= n;
        t += on;
        const int last = t * RB + RB < rows_left ? t * RB + RB - 1 : rows_left - 1;
        return load_turn(row_of(t) * groups, last * groups, s0 + (on ? 0 : i), t < tiles);
      };
      Turn turn;
      if constexpr (!PLAIN) {
        turn = turn_of(0, 0);
        const int at = codes_at(0, 0);
#pragma unroll
        for (int u = 0; u < W4_RING; ++u) ring[u] = load_step(at, u, wanted(0, u / 2 * 2));
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i0) __syncthreads();  // every wave is done with the stage before
      fill(first * W4_STEP, b);
      __syncthreads();
      for (int t = 0; t < tiles; ++t) {
        if constexpr (PLAIN) {
          for (int i = 0; i < valid; ++i) {
            float sc[SPS];
            uint32_t zz[SPS];
#pragma unroll
            for (int q = 0; q < SPS; ++q) {
              const int gr = group_of(s0 + i) + q;
              const int64_t at = (first_row + row_of(t)) * groups + (gr < groups ? gr : groups - 1);
              sc[q] = gr < groups ? scale_as_float(a.scales, a.scale_dtype, at) : 0.0f;
              zz[q] = Z ? pack_zero(gload<uint8_t>(a.zeros + at)) : neg8;
            }
            const int over = 64 * (s0 + i) + 16 * g - (half - 16);  // bytes of the lane's 16 past the row's end
            u32x4_t raw = load_step(codes_at(t, i) - (over > 0 ? over : 0), 0, true);
            raw = shift_down(raw, over < 0 ? 0 : over < 15 ? over : 15);
            compute(plain, raw, sc, zz, kw * n + i);
          }
        } else {
          for (int i = 0; i < n; i += W4_RING) {
            Turn now = turn;
            turn = turn_of(t, i + W4_RING);
            const bool last = i + W4_RING >= n;
            const int at_next = codes_at(t + last, last ? 0 : i + W4_RING);
            const bool in = t + last < tiles;
            if (s0 + i + W4_RING >= total) drop_past(now, s0 + i);  // uniform
#pragma unroll
            for (int u = 0; u < W4_RING; u += 2) {
              // two steps; the second may be past the wave's last, then with scales of 0
              if (i + u < valid) {  // uniform
                const bool both = i + u + 1 < valid;
#pragma unroll
                for (int v = u; v < u + 2; ++v) {
                  float sc[SPS];
                  uint32_t zz[SPS];
#pragma unroll
                  for (int q = 0; q < SPS; ++q) {
                    const int j = SPS * v + q;
                    sc[q] = v == u || both ? scale_of(now, j) : 0.0f;
                    zz[q] = Z ? pack_zero((now.z[j / 4] >> 8 * (j % 4)) & 255u) : neg8;
                  }
                  compute(plain, ring[v], sc, zz, kw * n + i + (v == u || both ? v : u));
                }
              }
              __builtin_amdgcn_sched_barrier(0);  // the steps' registers take the loads: no copies that wait
              // both halves of each row's 128 bytes at once
              ring[u] = load_step(at_next, u, in && wanted(last ? 0 : i + W4_RING, u));
              ring[u + 1] = load_step(at_next, u + 1, in && wanted(last ? 0 : i + W4_RING, u));
            }
          }
        }
        if constexpr (KS == 1) {
          if (staged) {
#pragma unroll
            for (int q = 0; q < MT; ++q) {
              f32x4_t* at = sums + (t * WR * MT + q) * 64;
              if (i0) acc[q] += *at;
              *at = acc[q];
            }
          }
          if (i0 + n == p.steps) {
            if constexpr (!PLAIN) check();
            out(plain, t);
          }
          clear();
        }
      }
    }
    if constexpr (KS > 1 && !PLAIN) check();
    return __syncthreads_or(bad != 0);
  };
  if (ragged || run(std::false_type{})) {
    f32x4_t first[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) first[t] = acc[t];
    if (!ragged) {
      if (threadIdx.x == 0) again = 0;
      __syncthreads();
      if (bad) atomicOr(&again, (bad & 15u) << (4 * g) | (bad >> 4) << (16 + 4 * g));
      __syncthreads();
      only = again;
    }
    run(std::true_type{});
    if constexpr (KS > 1)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = only >> (16 * t + 4 * g + i) & 1 ? acc[t][i] : first[t][i];
  }

  // the waves' sums over their columns meet in LDS, in the order of the columns' parts
  if constexpr (KS > 1) {
    f32x4_t* part = (f32x4_t*)lds + (wave / KS) * (KS - 1) * MT * 64;
    if (kw > 0)
#pragma unroll
      for (int t = 0; t < MT; ++t) part[((kw - 1) * MT + t) * 64 + lane] = acc[t];
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
        for (int w = 0; w < KS - 1; ++w) acc[t] += part[(w * MT + t) * 64 + lane];
      out(std::false_type{}, 0);
    }
  }
  zero_rows();
}

// Rows shorter than a step: one wave a weight row and route, a byte of codes a lane. 512 rows of 96 bf16 columns,
// 2048 experts of 1024 weight rows: by ids 128 us, sorted 145 (offsets looked at one by one 9.7 ms).
template <typename T>
__global__ __launch_bounds__(256) void w4_short_kernel(W4Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x;
  static_assert(SORT_MAX_EXPERTS + 64 <= 64 * 64, "a step's experts are one a lane");
  int e = 0;
  int64_t xr = r;
  if (a.ids) {
    e = a.ids[r];
    xr = r / a.top_k;
  } else if (a.offsets) {
    // the last expert whose rows begin at r or before, of every step-th first, then of the step's
    const int E = (int)a.n_experts, step = (E + 64) / 64;
    auto begun = [&](int i, bool on) { return __popcll(__ballot(on && i <= E && a.offsets[i <= E ? i : E] <= r)); };
    e = (begun(lane * step, true) - 1) * step;
    if (e >= 0) e += begun(e + lane, lane < step) - 1;  // n_experts: behind the last
  }
  const int half = (int)(a.cols + 1) / 2, groups = (int)((a.cols + a.group - 1) / a.group);
  for (int64_t n = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); n < a.rows; n += (int64_t)gridDim.y * 4) {
    float acc = 0.0f;
    if (e >= 0 && e < a.n_experts) {
      const int64_t row = e * a.rows + n;
      if (lane < half) {
        const int64_t at = row * groups + 2 * lane / (int)a.group;
        const float s = scale_as_float(a.scales, a.scale_dtype, at), z = a.zeros ? (float)a.zeros[at] : 8.0f;
        const T* x = (const T*)a.x + xr * a.x_stride + 2 * lane;
        const uint8_t q = a.codes[row * half + lane];
        acc = ((float)(q & 15) - z) * (float)x[0];
        if (2 * lane + 1 < a.cols) acc = fmaf((float)(q >> 4) - z, (float)x[1], acc);
        acc *= s;
      }
#pragma unroll
      for (int d = 32; d; d >>= 1) acc += __shfl_xor(acc, d);
    }
    if (lane == 0) ((T*)a.y)[r * a.rows + n] = (T)acc;
  }
}

// The launches; with tell, what they would launch instead.
template <typename T, int SPS, bool S4, bool Z, int MT, int KS, int WR>
int launch_as(const W4Args& a, int64_t items, int64_t expected, hipStream_t stream, ktmi_w4_kernel* tell) {
  constexpr int PLANES = std::is_same<T, float>::value ? 3 : 1, RB = 16 * WR, UNIT = W4_STEP * KS;
  const int64_t tiles = (a.rows + RB - 1) / RB;
  W4Plan p;
  p.steps = (int)((a.cols + UNIT - 1) / UNIT);
  const int64_t rows = a.n_routes < 16 * MT ? a.n_routes : 16 * MT;  // at most, of an item
  // room for one step of every row; up to the limit, or all columns of every row
  const int64_t least = PLANES * rows * (2 * UNIT + 16), whole = PLANES * rows * (2 * (int64_t)UNIT * p.steps + 16);
  const int64_t limit = KS > 1 ? W4_X_SPLIT : W4_X_BYTES;
  int64_t x_bytes = whole < limit ? whole : limit;
  if (x_bytes < least) x_bytes = least;
  if (KS > 1 && x_bytes < (KS - 1) * WR * MT * 64 * 16) x_bytes = (KS - 1) * WR * MT * 64 * 16;
  p.x_bytes = (int)((x_bytes + 15) / 16 * 16);
  // row tiles a block: so many that the blocks left are about those that the chip holds at once (three a
  // CU by their registers, fewer by their LDS), whose loads of activations and searches for their item
  // are then fewer; their codes and scales stay within 2^31 bytes
  const int64_t held = W4_CU_LDS / p.x_bytes < 3 ? W4_CU_LDS / p.x_bytes : 3;
  int64_t deep = KS > 1 ? 1 : expected * tiles / (256 * (held < 1 ? 1 : held));
  const int64_t most = 0x7FFFFFFFll / (RB * ((a.cols + 1) / 2));
  deep = deep > 8 ? 8 : deep;
  deep = deep > most ? most : deep;
  p.deep = (int)(deep < 1 ? 1 : deep);
  p.blocks = (int)((tiles + p.deep - 1) / p.deep);
  const int64_t bytes = p.x_bytes + (KS == 1 && whole > x_bytes ? p.deep * WR * MT * 64 * 16 : 0);
  KTMI_REQUIRE(items * p.blocks * 64 * KS * WR < 1ll << 32, KTMI_EINVAL, "w4: a grid of %lld x %d threads (below 2^32)",
               (long long)(items * p.blocks), 64 * KS * WR);
  auto kernel = w4_mfma_kernel<T, SPS, S4, Z, MT, KS, WR>;
  KTMI_REQUIRE(bytes <= W4_LDS_MOST, KTMI_EINVAL, "w4: %lld bytes of LDS", (long long)bytes);
  if (tell) {
    *tell = {16 * MT, KS, 16 * WR, p.deep, whole > x_bytes};
    return KTMI_OK;
  }
  kernel<<<(unsigned)(items * p.blocks), 64 * KS * WR, bytes, stream>>>(a, p);
  return KTMI_OK;
}

template <typename T, int SPS, int MT, int KS, int WR>
int launch_one(const W4Args& a, int64_t items, int64_t expected, hipStream_t stream, ktmi_w4_kernel* tell) {
  if (a.scale_dtype == KTMI_F32)
    return a.zeros ? launch_as<T, SPS, true, true, MT, KS, WR>(a, items, expected, stream, tell)
                   : launch_as<T, SPS, true, false, MT, KS, WR>(a, items, expected, stream, tell);
  return a.zeros ? launch_as<T, SPS, false, true, MT, KS, WR>(a, items, expected, stream, tell)
                 : launch_as<T, SPS, false, false, MT, KS, WR>(a, items, expected, stream, tell);
}

template <typename T, int SPS>
int launch_sps(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell) {
  constexpr bool F32 = std::is_same<T, float>::value;
  // rows of an expert, about: 16 a pass, or 32 where there are more (dense 4096 x 7168, bf16: 32 rows 26 us
  // in one pass of 32, 64 rows 27 in two; in one of 64 with its shorter stages 71)
  const int64_t mean = a.offsets ? a.n_routes / a.n_experts : a.ids ? 1 : a.n_routes;
  const bool many = !F32 && mean > 16;
  const int64_t rows = many ? 32 : 16;
  const int64_t items = a.ids ? a.n_routes
                        : a.offsets ? (a.n_experts < a.n_routes ? a.n_experts : a.n_routes) + a.n_routes / rows
                                    : (a.n_routes + rows - 1) / rows;
  // items that have rows, at most but for passes after an expert's first
  const int64_t expected = !a.ids && !a.offsets ? items : a.n_experts < a.n_routes ? a.n_experts : a.n_routes;
  // Four waves share 16 weight rows (the larger passes' blocks have 32) where whole rows a wave would leave CUs idle:
  // 7168 x 2048 bf16 dense, one row, 7.4 us; 23 experts of 1024 x 2048, 10.8 us without and 20.4 with
  const bool split = expected * ((a.rows + 63) / 64) < 256;
  // Larger passes share it by two, 64 weight rows a block, where blocks of 32, one a CU by their LDS, would
  // be more than the CUs: 7168 x 2048, 64 rows 12.2 us (19.8 of 32); 32 rows, 224 blocks of 32, 11.7 (11.4)
  const bool wide = expected * ((a.rows + 31) / 32) > 256;
  if constexpr (!F32)
    if (many)
      return !split ? launch_one<T, SPS, 2, 1, 4>(a, items, expected, stream, tell)
             : wide ? launch_one<T, SPS, 2, 2, 4>(a, items, expected, stream, tell)
                    : launch_one<T, SPS, 2, 4, 2>(a, items, expected, stream, tell);
  return split ? launch_one<T, SPS, 1, 4, 1>(a, items, expected, stream, tell) : launch_one<T, SPS, 1, 1, 4>(a, items, expected, stream, tell);
}

template <typename T>
int launch_t(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell) {
  W4Args b = a;
  if (a.group >= a.cols) b.group = (a.cols + W4_STEP - 1) / W4_STEP * W4_STEP;  // one group of whole steps
  if (a.cols < W4_STEP) {
    if (tell) {
      *tell = {1, 1, 4, 1, 0};
      return KTMI_OK;
    }
    const int64_t quads = (a.rows + 3) / 4;
    const dim3 grid((unsigned)a.n_routes, (unsigned)(quads < 65535 ? quads : 65535));
    w4_short_kernel<T><<<grid, 256, 0, stream>>>(b);
    return KTMI_OK;
  }
  return b.group == 32   ? launch_sps<T, 4>(b, stream, tell)
         : b.group == 64 ? launch_sps<T, 2>(b, stream, tell)
                         : launch_sps<T, 1>(b, stream, tell);
}

}  // namespace

}  // namespace ktmi
