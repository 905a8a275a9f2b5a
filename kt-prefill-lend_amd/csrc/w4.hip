// Products with 4-bit weights and group scales:
//   y[r, n] = sum_g s[e, n, g] * sum_{c in g} (q[e, n, c] - z[e, n, g]) * x[r, c]
//
// w4_mfma_kernel, for rows of 16 bytes of codes or more, runs the matrix cores for any number of
// activation rows from one: v_mfma_f32_16x16x32 with 16 weight rows as its columns and up to 16
// activation rows as its rows. A wave takes 16 weight rows in steps of 128 columns, 16 bytes of
// codes a lane (lane l: row l % 16, column piece g = l / 16), loaded ahead into a ring of registers.
//
// Codes become operands exactly: an e4m3 byte of value n < 16 is n * 2^-9 (the subnormals run on
// into the first normal binade), so one v_cvt_scalef32_pk turns two masked nibbles into two bf16 or
// f16 integers. The zero point is a second product of the same activations with the constant -z, so
// the group's sum D = sum (q - z) x is exact but for fp32 sums, and acc += s D. Infinite or NaN
// activations (and products past fp32) make that inf - inf: a block whose sums are not all finite
// runs again with q - z as the operand, which gives the plain sum's infinities and NaN.
//
// fp32 activations are three bf16 parts (8 + 8 + 8 bits of the significand, cut, so that nothing
// overflows), each with a product of its own: exact but for parts below bf16's smallest number.
//
// The activations of the block's rows pass through LDS in column stages, values of each eight in the
// order 0 2 4 6 1 3 5 7 in which the nibbles come out; columns past the row's end are zeros there.
// The scales and zero points of the stage are expanded to fp32 and packed -z beside them, SPS for
// each 128 columns, zeros past the last group. What a lane loads past its row's end then meets a zero on either side.
#include <type_traits>

#include "kernels.h"

namespace ktmi {

namespace {

constexpr int W4_THREADS = 256;
constexpr int W4_STEP = 128;       // columns of a step: 16 bytes of codes a lane
constexpr int W4_RING = 4;         // steps of codes in flight a wave
constexpr int W4_IDS = 64;         // routes whose ids a wave holds one a lane
constexpr int W4_X_BYTES = 48 << 10;   // LDS for a stage's activations, about
constexpr int W4_S_BYTES = 16 << 10;   // and for its scales

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// what the MFMA takes: bf16 for bf16 and fp32 activations, f16 for f16
template <typename T>
struct Operand {
  using V8 = bf16x8_t;
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

// the four words of a lane's 16 bytes shifted down by n bytes (0 < n < 16), zeros from above
__device__ __forceinline__ u32x4_t shift_down(const u32x4_t& w, int n) {
  const int words = n >> 2, bits = 8 * (n & 3);
  uint32_t v[5] = {w[0], w[1], w[2], w[3], 0u};
  u32x4_t out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      lo = i + words == j ? v[j] : lo;
      hi = i + words + 1 == j ? v[j] : hi;
    }
    out[i] = (uint32_t)(((uint64_t)hi << 32 | lo) >> bits);
  }
  return out;
}

__device__ __forceinline__ float scale_as_float(const void* s, int dtype, int64_t i) {
  if (dtype == KTMI_F32) return gload<float>((const float*)s + i);
  const uint16_t v = gload<uint16_t>((const uint16_t*)s + i);
  return dtype == KTMI_F16 ? half_bits_to_float(v) : bf2f(v);
}

// One launch's plan: blocks of RB = 64 / KS weight rows (KS waves of a block share their rows and
// split the columns), items (expert, pass of up to 16 MT of its rows), columns a stage.
struct W4Plan {
  int tiles;    // row blocks
  int stage;    // columns of a stage, a multiple of 128 KS
  int x_rows;   // activation rows a stage holds
  int x_pitch;  // bytes between them
  int s_pitch;  // scales between weight rows, odd
  int steps;    // steps a wave, all stages
  uint32_t chunks_inv, scales_inv;  // ceil(2^32 / d) of a stage's 8-column chunks and scales a row
};

// i / d for i, d < 2^16 from inv = ceil(2^32 / d) (0 for d = 1)
__device__ __forceinline__ int divide(int i, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)i, inv) : i; }

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

// The block's item: expert e, its rows of y at list[0 .. m) and of x at from[0 .. m); m = 0: none.
// Every wave of the block writes the same lists.
template <int MT>
__device__ __forceinline__ int find_item(const W4Args& a, int item, int& e, int* list, int* from) {
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
      list[mine] = lane;
      from[mine] = lane / (int)a.top_k;
    }
    const int m = __popcll(same) - rank;
    return m < ROWS ? m : ROWS;
  }
  int first = 0, m = (int)a.n_routes, pass = item;
  e = 0;
  if (a.offsets) {
    // the item-th pass over the experts in order: passes of 64 experts at a time, summed over the lanes
    int before = 0;
    bool found = false;
    for (int64_t e0 = 0; e0 < a.n_experts && !found; e0 += 64) {
      const int64_t i = e0 + lane;
      int lo = 0, n = 0;
      if (i < a.n_experts) {
        const int R = (int)a.n_routes;
        lo = a.offsets[i];
        int hi = a.offsets[i + 1];
        lo = lo < 0 ? 0 : lo < R ? lo : R;
        hi = hi < 0 ? 0 : hi < R ? hi : R;
        n = hi > lo ? hi - lo : 0;
      }
      const int passes = (n + ROWS - 1) / ROWS;
      int sum = passes;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(sum, d);
        if (lane >= d) sum += u;
      }
      const int start = before + sum - passes;
      const uint64_t hit = __ballot(item >= start && item < start + passes);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        first = __shfl(lo, l), m = __shfl(n, l), pass = item - __shfl(start, l), e = (int)e0 + l;
        found = true;
      }
      before = __shfl(before + sum, 63);
    }
    if (!found) return 0;
  }
  first += pass * ROWS;
  m -= pass * ROWS;
  if (m > ROWS) m = ROWS;
  if (lane < m) {
    const int r = a.perm ? a.perm[first + lane] : first + lane;
    list[lane] = r;
    from[lane] = a.perm ? r / (int)a.top_k : r;
  }
  return m > 0 ? m : 0;
}

template <typename T, int SPS, int MT, int KS>
__global__ __launch_bounds__(W4_THREADS) void w4_mfma_kernel(W4Args a, W4Plan p) {
  using O = Operand<T>;
  constexpr int PLANES = std::is_same<T, float>::value ? 3 : 1;
  constexpr int RB = 64 / KS;  // weight rows of the block
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int list[16 * MT], from[16 * MT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / p.tiles, tile = blockIdx.x - item * p.tiles;
  const int n0 = tile * RB;
  T* y = (T*)a.y;
  // rows of no expert are zero: route `item` by its id, or every items-th row past the last segment
  if (a.ids) {
    const int e = a.ids[item];
    if (e < 0 || e >= a.n_experts) {
      for (int n = n0 + threadIdx.x; n < n0 + RB && n < a.rows; n += W4_THREADS) y[item * a.rows + n] = (T)0.0f;
      return;
    }
  } else if (a.offsets) {
    // (of unsorted ids: the routes that the order puts there), and those before the first
    const int items = gridDim.x / p.tiles;
    auto zero = [&](int64_t r, int64_t end) {
      for (r += item; r < end; r += items) {
        const int64_t at = a.perm ? ~a.perm[r] : r;
        for (int n = n0 + threadIdx.x; n < n0 + RB && n < a.rows; n += W4_THREADS) y[at * a.rows + n] = (T)0.0f;
      }
    };
    const int begin = a.offsets[0], end = a.offsets[a.n_experts];
    zero(0, begin < a.n_routes ? begin : a.n_routes);
    zero(end > 0 ? end : 0, a.n_routes);
  }
  int e;
  const int m = find_item<MT>(a, item, e, list, from);
  if (m == 0) return;
  const int mg = (m + 15) / 16;  // groups of 16 activation rows
  __syncthreads();

  const int cols = (int)a.cols, half = (cols + 1) / 2;
  const int row = lane & 15, g = lane >> 4;
  const int rb = KS == 1 ? 16 * wave + row : row;  // the lane's weight row in the block
  const int64_t groups = (a.cols + a.group - 1) / a.group;
  const int64_t first_row = e * a.rows + n0;
  const int rows_left = (int)(a.rows - n0 < RB ? a.rows - n0 : RB);
  const uint8_t* codes = a.codes + (first_row + (rb < rows_left ? rb : rows_left - 1)) * half;
  // 16 bytes of step s, those past the row's end replaced by its last ones
  auto load = [&](int s) {
    const int b = 64 * s + 16 * g;
    return gload<u32x4_a1_t>(codes + (b < half - 16 ? b : half - 16));
  };
  float* scales = (float*)(lds + (size_t)PLANES * p.x_rows * p.x_pitch);
  uint32_t* negz = (uint32_t*)scales + RB * p.s_pitch;
  const uint32_t neg8 = O::pack(-8.0f, -8.0f);

  f32x4_t acc[MT];
  auto run = [&](auto plain) {
    constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int per_stage = p.stage / (W4_STEP * KS);

    // activations, scales and zero points of the columns from k0
    auto stage = [&](int k0) {
      const int chunks = p.stage / 8;
      for (int i = threadIdx.x; i < m * chunks; i += W4_THREADS) {
        const int r = divide(i, p.chunks_inv), c = i - r * chunks, k = k0 + 8 * c;
        const T* x = (const T*)a.x + from[r] * a.x_stride + k;
        uint8_t* out = lds + (size_t)r * p.x_pitch + 16 * c;
        if constexpr (PLANES == 1) {
          u32x4_t v = {0, 0, 0, 0};
          if (k + 8 <= cols) {
            v = gload<u32x4_a2_t>(x);
          } else {
            for (int j = 0; j < 8; ++j)
              if (k + j < cols) {
                const uint32_t u = (uint32_t)gload<uint16_t>(x + j) << (16 * (j & 1));
                if (j < 2) v[0] |= u; else if (j < 4) v[1] |= u; else if (j < 6) v[2] |= u; else v[3] |= u;
              }
          }
          *(u32x4_t*)out = u32x4_t{__builtin_amdgcn_perm(v[1], v[0], 0x05040100), __builtin_amdgcn_perm(v[3], v[2], 0x05040100),
                                   __builtin_amdgcn_perm(v[1], v[0], 0x07060302), __builtin_amdgcn_perm(v[3], v[2], 0x07060302)};
        } else {
          uint32_t part[3][8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float v = k + j < cols ? gload<float>(x + j) : 0.0f;
            const uint32_t u = __builtin_bit_cast(uint32_t, v), h = u & 0xFFFF0000u;
            const bool finite = (u & 0x7F800000u) != 0x7F800000u;
            const float r1 = finite ? v - __builtin_bit_cast(float, h) : 0.0f;
            const uint32_t mid = __builtin_bit_cast(uint32_t, r1) & 0xFFFF0000u;
            const float r2 = r1 - __builtin_bit_cast(float, mid);
            // a NaN whose set bits are all in the low half stays one
            part[0][j] = finite || !(u & 0x007FFFFFu) ? h >> 16 : 0x7FC0u;
            part[1][j] = mid >> 16;
            part[2][j] = __builtin_bit_cast(uint32_t, r2) >> 16;
          }
#pragma unroll
          for (int q = 0; q < 3; ++q)
            *(u32x4_t*)(out + (size_t)q * p.x_rows * p.x_pitch) =
                u32x4_t{part[q][0] | part[q][2] << 16, part[q][4] | part[q][6] << 16, part[q][1] | part[q][3] << 16,
                        part[q][5] | part[q][7] << 16};
        }
      }
      const int n = p.stage / W4_STEP * SPS;
      for (int i = threadIdx.x; i < RB * n; i += W4_THREADS) {
        const int r = divide(i, p.scales_inv), c = i - r * n;
        const int gr = SPS == 1 ? (k0 + W4_STEP * c) / (int)a.group : k0 / (W4_STEP / SPS) + c;
        const bool in = r < rows_left && gr < groups;
        const int64_t at = (first_row + r) * groups + gr;
        scales[r * p.s_pitch + c] = in ? scale_as_float(a.scales, a.scale_dtype, at) : 0.0f;
        if (a.zeros) {
          const float z = in ? -(float)gload<uint8_t>(a.zeros + at) : 0.0f;
          negz[r * p.s_pitch + c] = O::pack(z, z);
        }
      }
    };

    auto compute = [&](u32x4_t raw, int s, int k0) {
      // a row that ends inside these 16 bytes: what was loaded ends with the row
      const int over = 64 * s + 16 * g - (half - 16);
      if (64 * s + 64 > half && (half & 15)) {
        if (over > 0 && over < 16) raw = shift_down(raw, over);
      }
      uint32_t w[4] = {raw[0], raw[1], raw[2], raw[3]};
      regroup<SPS>(w);
      const int k = W4_STEP * s - k0;  // in the stage
      const uint8_t* xp = lds + 2 * (k + x_base<SPS>(g));
      const int gi = rb * p.s_pitch + k / W4_STEP * SPS;
#pragma unroll
      for (int sub = 0; sub < SPS; ++sub) {
        const float sc = scales[gi + sub];
        const uint32_t zz = a.zeros ? negz[gi + sub] : neg8;
        const u32x4_t zf = {zz, zz, zz, zz};
        u32x4_t wf[4 / SPS];
#pragma unroll
        for (int j = 0; j < 4 / SPS; ++j) {
          if constexpr (PLAIN)
            wf[j] = decode_plain<T>(w[sub * (4 / SPS) + j], O::low(zz));
          else
            wf[j] = decode<T>(w[sub * (4 / SPS) + j]);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (t < mg) {  // uniform
            const int r = 16 * t + row < m ? 16 * t + row : m - 1;
            f32x4_t d = {0.0f, 0.0f, 0.0f, 0.0f}, dz = d;
#pragma unroll
            for (int j = 0; j < 4 / SPS; ++j)
#pragma unroll
              for (int q = 0; q < PLANES; ++q) {
                const u32x4_t xv = *(const u32x4_t*)(xp + (size_t)(q * p.x_rows + r) * p.x_pitch +
                                                     2 * x_fixed<SPS>(sub * (4 / SPS) + j));
                d = O::mfma(xv, wf[j], d);
                if constexpr (!PLAIN) dz = O::mfma(xv, zf, dz);
              }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(sc, PLAIN ? d[i] : d[i] + dz[i], acc[t][i]);
          }
        }
      }
    };

    const int first = KS == 1 ? 0 : wave;
    u32x4_t ring[W4_RING];
    int k0 = 0;
#pragma unroll
    for (int u = 0; u < W4_RING; ++u) ring[u] = load(first + KS * u);
    for (int i = 0; i < p.steps; i += W4_RING) {
#pragma unroll
      for (int u = 0; u < W4_RING; ++u) {
        if (i + u < p.steps) {
          if ((i + u) % per_stage == 0) {
            k0 = (i + u) / per_stage * p.stage;
            if (i + u) __syncthreads();
            stage(k0);
            __syncthreads();
          }
          const u32x4_t raw = ring[u];
          ring[u] = load(first + KS * (i + u + W4_RING));
          compute(raw, first + KS * (i + u), k0);
        }
      }
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= !(fabsf(acc[t][i]) < __builtin_inff());
    return __syncthreads_or(bad);
  };
  if (run(std::false_type{})) run(std::true_type{});

  // the waves' sums over their columns meet in LDS, wave 0's first
  if constexpr (KS > 1) {
    f32x4_t* part = (f32x4_t*)lds;
    if (wave > 0)
#pragma unroll
      for (int t = 0; t < MT; ++t) part[((wave - 1) * MT + t) * 64 + lane] = acc[t];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int t = 0; t < MT; ++t)
      for (int w = 0; w < KS - 1; ++w) acc[t] += part[(w * MT + t) * 64 + lane];
  }
  if (rb < rows_left)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * t + 4 * g + i;
        if (r < m) y[list[r] * a.rows + n0 + rb] = (T)acc[t][i];
      }
}

// Rows of fewer than 16 bytes of codes: one wave a weight row and route.
template <typename T>
__global__ __launch_bounds__(W4_THREADS) void w4_short_kernel(W4Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x;
  int e = 0;
  int64_t xr = r;
  if (a.ids) {
    e = a.ids[r];
    xr = r / a.top_k;
  } else if (a.offsets) {
    e = -1;
    for (int i = 0; i < a.n_experts && e < 0; ++i)
      if (r < a.offsets[i + 1] && r >= a.offsets[i]) e = i;
  }
  const int half = (int)(a.cols + 1) / 2;
  for (int64_t n = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); n < a.rows; n += (int64_t)gridDim.y * 4) {
    float acc = 0.0f;
    if (e >= 0 && e < a.n_experts) {
      // below 32 columns there is one group
      const int64_t row = e * a.rows + n;
      const float s = scale_as_float(a.scales, a.scale_dtype, row), z = a.zeros ? (float)a.zeros[row] : 8.0f;
      if (lane < half) {
        const T* x = (const T*)a.x + xr * a.x_stride + 2 * lane;
        const uint8_t q = a.codes[row * half + lane];
        acc = ((float)(q & 15) - z) * (float)x[0];
        if (2 * lane + 1 < a.cols) acc = fmaf((float)(q >> 4) - z, (float)x[1], acc);
      }
#pragma unroll
      for (int d = 8; d; d >>= 1) acc += __shfl_xor(acc, d);
      acc *= s;
    }
    if (lane == 0) ((T*)a.y)[r * a.rows + n] = (T)acc;
  }
}

template <typename T, int SPS, int MT, int KS>
int launch_one(const W4Args& a, int64_t items, hipStream_t stream) {
  constexpr int PLANES = std::is_same<T, float>::value ? 3 : 1, RB = 64 / KS, UNIT = W4_STEP * KS;
  W4Plan p;
  p.tiles = (int)((a.rows + RB - 1) / RB);
  p.x_rows = (int)(a.n_routes < 16 * MT ? a.n_routes : 16 * MT);
  const int64_t whole = (a.cols + UNIT - 1) / UNIT * UNIT;
  int64_t stage = (W4_X_BYTES / (2 * PLANES * p.x_rows) - 8) / UNIT * UNIT;
  const int64_t by_scales = (int64_t)W4_STEP * (W4_S_BYTES / (4 * RB * SPS)) / UNIT * UNIT;
  if (by_scales < stage) stage = by_scales;
  if (stage < UNIT) stage = UNIT;
  if (stage > whole) stage = whole;
  p.stage = (int)stage;
  p.x_pitch = 2 * p.stage + 16;
  const int scales = p.stage / W4_STEP * SPS;
  p.s_pitch = scales | 1;
  p.chunks_inv = (uint32_t)((0x100000000ull + p.stage / 8 - 1) / (p.stage / 8));
  p.scales_inv = scales == 1 ? 0 : (uint32_t)((0x100000000ull + scales - 1) / scales);
  p.steps = (int)(whole / UNIT);
  int64_t bytes = (int64_t)PLANES * p.x_rows * p.x_pitch + (int64_t)RB * p.s_pitch * (a.zeros ? 8 : 4);
  if (KS > 1 && bytes < (KS - 1) * MT * 64 * 16) bytes = (KS - 1) * MT * 64 * 16;
  KTMI_REQUIRE(items * p.tiles <= 0x7FFFFFFF, KTMI_EINVAL, "w4: %lld blocks (below 2^31)", (long long)(items * p.tiles));
  auto kernel = w4_mfma_kernel<T, SPS, MT, KS>;
  static const hipError_t attr =
      hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, W4_LDS_MOST);
  KTMI_HIP_TRY(attr);
  KTMI_REQUIRE(bytes <= W4_LDS_MOST, KTMI_EINVAL, "w4: %lld bytes of LDS", (long long)bytes);
  kernel<<<(unsigned)(items * p.tiles), W4_THREADS, bytes, stream>>>(a, p);
  return KTMI_OK;
}

template <typename T, int SPS>
int launch_sps(const W4Args& a, hipStream_t stream) {
  const int64_t mean = a.offsets ? a.n_routes / a.n_experts : a.ids ? 1 : a.n_routes;  // rows of an expert, about
  const bool many = !std::is_same<T, float>::value && mean > 16;
  const int64_t rows = many ? 64 : 16;
  const int64_t items = a.ids ? a.n_routes
                        : a.offsets ? (a.n_experts < a.n_routes ? a.n_experts : a.n_routes) + a.n_routes / rows
                                    : (a.n_routes + rows - 1) / rows;
  const bool split = items * ((a.rows + 63) / 64) < 1024;
  if constexpr (!std::is_same<T, float>::value)
    if (many) return split ? launch_one<T, SPS, 4, 4>(a, items, stream) : launch_one<T, SPS, 4, 1>(a, items, stream);
  return split ? launch_one<T, SPS, 1, 4>(a, items, stream) : launch_one<T, SPS, 1, 1>(a, items, stream);
}

template <typename T>
int launch_t(const W4Args& a, hipStream_t stream) {
  if (a.cols < 31) {
    const int64_t quads = (a.rows + 3) / 4;
    const dim3 grid((unsigned)a.n_routes, (unsigned)(quads < 65535 ? quads : 65535));
    w4_short_kernel<T><<<grid, W4_THREADS, 0, stream>>>(a);
    return KTMI_OK;
  }
  W4Args b = a;
  if (a.group >= a.cols) b.group = (a.cols + W4_STEP - 1) / W4_STEP * W4_STEP;  // one group of whole steps
  return b.group == 32 ? launch_sps<T, 4>(b, stream) : b.group == 64 ? launch_sps<T, 2>(b, stream) : launch_sps<T, 1>(b, stream);
}

int launch_any(const W4Args& a, hipStream_t stream) {
  return a.x_dtype == KTMI_F32 ? launch_t<float>(a, stream)
         : a.x_dtype == KTMI_F16 ? launch_t<_Float16>(a, stream) : launch_t<__bf16>(a, stream);
}

// workspace of a call with more ids than a wave holds: the routes' order (offsets, perm, pos) and the
// sort's counts
int64_t ints(int64_t n) { return (n + 3) / 4 * 4; }

}  // namespace

int64_t w4_workspace(int64_t tokens, int64_t top_k, int64_t E) {
  const int64_t R = tokens * top_k;
  if (R <= W4_IDS) return 0;
  return 4 * (ints(E + 1) + 2 * ints(R) + ints(moe_sort_chunks(R) * (E + 1)));
}

int launch_w4(const W4Args& a, hipStream_t stream) {
  int rc;
  if (a.ids && a.n_routes > W4_IDS && a.cols >= 31) {
    int* offsets = (int*)a.ws;
    int* perm = offsets + ints(a.n_experts + 1);
    int* pos = perm + ints(a.n_routes);
    rc = launch_moe_sort(nullptr, 2, 0, 0, a.ids, a.n_routes / a.top_k, a.top_k, a.n_experts, nullptr, offsets, perm, pos,
                         pos + ints(a.n_routes), stream);
    if (rc) return rc;
    W4Args b = a;
    b.ids = nullptr, b.offsets = offsets, b.perm = perm;
    rc = launch_any(b, stream);
  } else {
    rc = launch_any(a, stream);
  }
  if (rc) return rc;
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

}  // namespace ktmi
