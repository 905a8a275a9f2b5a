// What the kernels of the products by expert share (prod_tile.h: many rows, prod_rows.h: few rows): the
// element types on the matrix cores, the rows' segments by expert, the gate's activation.
#pragma once
#include <type_traits>

#include "kernels.h"

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
// 16 bytes at any address: global loads take one
typedef uint32_t u32x4_a1_t __attribute__((ext_vector_type(4))) __attribute__((aligned(1)));

namespace ktmi {

// and stores
template <bool STREAM>
__device__ __forceinline__ void gstore(void* p, u32x4_t v) {
  auto* g = (__attribute__((address_space(1))) u32x4_a1_t*)p;
  if constexpr (STREAM) __builtin_nontemporal_store(v, g);
  else *g = v;
}

// An element type: its bytes (ES), elements of a 16-byte chunk (EPC), the fp32 value of one and back, and
// the products of 32 rows by 32 rows (mma32) and 16 by 16 (mma16) over the k of one chunk a lane: lane half
// (quarter) q holds chunk q of its row, so that the sum runs over 2 (4) chunks. fp32 chunks take four
// instructions of one k a lane: the k of an instruction are not neighbours, but the same in both operands.
struct BF16 {
  using S = __bf16;
  static constexpr int ES = 2, EPC = 8;
  static __device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};

struct F16 {
  using S = _Float16;
  static constexpr int ES = 2, EPC = 8;
  static __device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

struct F32 {
  using S = float;
  static constexpr int ES = 4, EPC = 4;
  static __device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
    const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
    return c;
  }
};

template <typename S>
struct vec4_of { typedef S type __attribute__((ext_vector_type(4))); };

// 16 bytes of a row of n elements from element k on, zeros past its end: at any alignment
template <int ES>
__device__ __forceinline__ u32x4_t load_chunk(const uint8_t* row, int64_t k, int64_t n) {
  constexpr int EPC = 16 / ES;
  const uint8_t* p = row + k * ES;
  if (k + EPC <= n) return gload<u32x4_a1_t>(p);
  u32x4_t v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < EPC; ++i) {
    if (k + i >= n) continue;
    uint32_t u;
    if constexpr (ES == 4) u = gload<uint32_t>(p + 4 * i);
    else if constexpr (ES == 2) u = gload<uint16_t>(p + 2 * i);
    else u = gload<uint8_t>(p + i);
    v[i * ES / 4] |= u << (8 * (i * ES % 4));
  }
  return v;
}

// The gate's activation in fp32: silu(g) = g / (1 + e^-g); gelu(g) = g / (1 + e^-2z), z = sqrt(2 / pi)
// (g + 0.044715 g^3), which is the tanh form g (1 + tanh z) / 2: both are g times a sigmoid. Past |g| = 16
// the second's sigmoid is 0 or 1 in fp32, so the cube takes a clamped g, which cannot overflow.
constexpr float GELU_2C = 1.5957691216057308f, GELU_A = 0.044715f;
// S: the type that the values are rounded to. In 16 bits the power is that of v_exp_f32 with the argument's product with log2 e
// rounded (2^-24 |v| of it), far below their rounding; in fp32 it is right to a step.
template <typename S>
__device__ __forceinline__ float sigmoid(float v) {
  return 1.0f / (1.0f + (std::is_same<S, float>::value ? expf(-v) : __expf(-v)));
}
__device__ __forceinline__ float clamp16(float g) { return g > 16.0f ? 16.0f : g < -16.0f ? -16.0f : g; }
template <typename S>
__device__ __forceinline__ float gate_sigmoid(int act, float g) {
  if (act == KTMI_ACT_SILU) return sigmoid<S>(g);
  const float c = clamp16(g);
  return sigmoid<S>(GELU_2C * (c + GELU_A * c * c * c));
}
template <typename S>
__device__ __forceinline__ float act_of(int act, float g) { return g * gate_sigmoid<S>(act, g); }
// act(g) and its derivative
template <typename S>
__device__ __forceinline__ void act_grad(int act, float g, float& f, float& d) {
  const float s = gate_sigmoid<S>(act, g), c = clamp16(g);
  f = g * s;
  d = act == KTMI_ACT_SILU ? s + f * (1.0f - s) : s + c * s * (1.0f - s) * GELU_2C * (1.0f + 3.0f * GELU_A * c * c);
}

// The rows 0 .. R-1 of sorted operands as E + 2 segments: those in front of the first expert's, the
// experts', those behind the last one's. bound(i) is the first row of segment i; segment i is expert i - 1's.
// Offsets that are no rows are clamped to them; a segment that would end before it starts has no rows.
struct Segments {
  const int32_t* offsets;
  int E;
  int R;
  __device__ __forceinline__ int bound(int i) const {
    if (i == 0) return 0;
    if (i > E + 1) return R;
    return min(max(offsets[i - 1], 0), R);
  }
};

struct RowTile {
  int expert;  // -1: rows of no expert, which are zeros
  int row0, rows;
  bool there;
};

// The wave's tile number t when every segment is cut into tiles of bm rows, and the number of all tiles.
// Each lane counts the tiles of a run of segments, the wave adds them up, and the lane that holds tile t
// finds it in its run.
__device__ __forceinline__ int count_tiles(const Segments& s, int bm, int& mine) {
  const int lane = threadIdx.x & 63, n = s.E + 2, per = (n + 63) / 64;
  int sum = 0, at = lane * per;
  int b = s.bound(min(at, n));
  for (int i = 0; i < per && at + i < n; ++i) {
    const int e = s.bound(at + i + 1);
    sum += (max(e - b, 0) + bm - 1) / bm;
    b = e;
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o, 64);
    if (lane >= o) inc += u;
  }
  mine = inc - sum;
  return __builtin_amdgcn_readlane(inc, 63);
}
__device__ __forceinline__ RowTile find_tile(const Segments& s, int bm, int t, int mine) {
  const int n = s.E + 2, per = (n + 63) / 64;
  const uint64_t before = __ballot(mine <= t);
  const int lane = 63 - __builtin_clzll(before);  // the last lane whose run starts at or before t (lane 0's does)
  int left = t - __builtin_amdgcn_readlane(mine, lane);
  const int at = lane * per;
  for (int i = 0; i < per && at + i < n; ++i) {
    const int b = s.bound(at + i), c = max(s.bound(at + i + 1) - b, 0), k = (c + bm - 1) / bm;
    if (left < k)
      return RowTile{at + i >= 1 && at + i <= s.E ? at + i - 1 : -1, b + left * bm, min(bm, c - left * bm), true};
    left -= k;
  }
  return RowTile{-1, 0, 0, false};
}

}  // namespace ktmi
