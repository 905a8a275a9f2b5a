// Tokens sorted by expert and back, with the weights applied, and the gradients of both.
//
// With key(r) = ids[r] for a valid id and E for any other, a route's place is
//   p(r) = #{r' : key(r') < key(r)  or  key(r') = key(r) and r' < r},
// a stable counting sort: a histogram of each chunk of routes, then per chunk the places from the
// totals of the keys below, of the chunks before and of the routes before inside the chunk. The
// row copies, the weighted sums and the gradients then go by token: a token's row is read once
// and its routes' places are wave-uniform.
//
// HBM bounds the long calls and launches the short ones. 16384 tokens of 2048 bf16 columns, 8 routes
// each: the order 17 us (two launches), the copies 102 us for 604 MB (5.9 TB/s; a large copy on this
// card moves 5.0 read and written, a fill 6.9); 4096 tokens, a fifth of the routes without an expert: the sums back
// 23 us, their gradients 42 us for 257 MB (6.1 TB/s). One token: one launch of 4 us. The order could be one launch less with blocks that
// wait for each other's counts; that is left out, as a wait between blocks ends only if all of them run.
#include <type_traits>

#include "kernels.h"

namespace ktmi {

namespace {

constexpr int SORT_THREADS = 256;
constexpr int SORT_MAX_PER = 8;   // routes of a thread of the order's two kernels, at most
// Routes of a call that takes one launch, at most. 2048 bf16 columns, 8 routes a token: 5120 routes 13.0 us in
// one launch and 13.4 in three, 8192 20.0 and 15.2, 16376 43.4 and 21.6 (every block reads all ids).
constexpr int SORT_SMALL = 4096;
// Routes a token of one launch, at most: a block takes its token's all at once. Of more, 16 at a time, the launches of
// the order and the copies won at every size: 17 a token, 60 tokens of 2048 bf16 columns 10.9 and 10.7 us, 240 tokens
// 23.0 and 12.4; 32 a token, one token 13.3 and 9.6.
constexpr int SORT_SMALL_K = 16;
// Comparisons of one launch, at most: every block (a token and 4 KB of its row) holds its token's routes against all
// ids, 8 of them or 16 (which counts double), so few routes a token and wide rows cost it most. Against the launches of
// the order and the copies, us: the order of 4096 routes 7.4 and 7.2 at 8 a token (2^24 comparisons), 12.5 and 7.4 at 2
// (2^26), 20.7 and 7.3 at 1, of 4000 at 10 11.5 and 7.3 (2^25.6), of 2000 7.5 and 7.1 (2^23.6). With 7168 f32 columns 4096
// routes 28.9 and 27.9 at 8 (2^26.8), 119 and 42.3 at 1 (2^29.8); 2048 14.0 and 18.2 at 8 (2^24.8); 1024 at 1 16.8 and 16.8
// (2^25.8). Up to SORT_NO_WS comparisons of the order it is one launch whatever the rows' width, which needs no
// workspace: 512 routes at 1, 7168 f32 columns, 10.3 and 10.8.
constexpr int64_t SORT_ORDER_WORK = 1 << 24, SORT_ROWS_WORK = 1 << 26, SORT_NO_WS = 1 << 22;
constexpr int SORT_PIECE = 4096;  // bytes of a row that a block of the one launch copies
constexpr int64_t SORT_CACHED = 256 << 20;  // the last-level cache
// Chunks up to which every chunk adds up the counts of all by itself; of more they are added up once, in a
// launch of its own (else the work would grow with the routes' square). The order of 256 keys: 64 chunks
// 14.5 us by themselves and 14.9 with the launch, 128 18.8 and 15.4, 256 27.2 and 16.6.
constexpr int SORT_SCAN = 64;
constexpr int SCAN_WAVES = 16;
constexpr int ROW_WAVES = 4;      // waves of a row kernel's block, at most
constexpr int64_t ROW_TOKENS = 1 << 23;  // tokens (blocks) of a row kernel's launch, at most: a grid has below 2^32 threads

__device__ __forceinline__ int key_of(int id, int E) { return id >= 0 && id < E ? id : E; }

__device__ __forceinline__ void sort_wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// counts[chunk][E + 1]: the chunk's routes by key. Bound by LDS atomics on popular keys: 2 routes a
// thread 2.8 us at 16376 routes, 8 a thread 5.4.
template <int PER>
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const int32_t* __restrict__ ids, int R, int E,
                                                                  int* __restrict__ counts) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e <= E; e += SORT_THREADS) hist[e] = 0;
  __syncthreads();
  const int64_t r0 = (int64_t)blockIdx.x * (PER * SORT_THREADS);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * SORT_THREADS + threadIdx.x;
    if (r < R) atomicAdd(&hist[key_of(ids[r], E)], 1);
  }
  __syncthreads();
  int* out = counts + (int64_t)blockIdx.x * (E + 1);
  for (int e = threadIdx.x; e <= E; e += SORT_THREADS) out[e] = hist[e];
}

// exclusive sum over the block of one value a thread (SORT_THREADS threads); tmp: 4 ints of LDS
__device__ __forceinline__ int block_exclusive(int v, int* tmp) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(s, d);
    if (lane >= d) s += u;
  }
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += tmp[w];
  __syncthreads();
  return before + s - v;
}

// counts[c][e] becomes the routes of key e before chunk c, counts[chunks][e] all of them. A block takes 64
// keys, each of its waves a run of chunks: their sum first, then their running sums.
__global__ __launch_bounds__(64 * SCAN_WAVES) void sort_scan_kernel(int* __restrict__ counts, int chunks, int n) {
  __shared__ int part[SCAN_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
  const int span = (chunks + SCAN_WAVES - 1) / SCAN_WAVES, c0 = wave * span;
  const int c1 = c0 + span < chunks ? c0 + span : chunks;
  int v[16], sum = 0;
  for (int c = c0; c < c1; c += 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = e < n && c + i < c1 ? counts[(int64_t)(c + i) * n + e] : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += v[i];
  }
  part[wave][lane] = sum;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < SCAN_WAVES; ++w) {
    before += w < wave ? part[w][lane] : 0;
    all += part[w][lane];
  }
  for (int c = c0; c < c1; c += 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = e < n && c + i < c1 ? counts[(int64_t)(c + i) * n + e] : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (e < n && c + i < c1) counts[(int64_t)(c + i) * n + e] = before;
      before += v[i];
    }
  }
  if (wave == 0 && e < n) counts[(int64_t)chunks * n + e] = all;
}

// The places of a chunk's routes. SCANNED: the counts are as sort_scan_kernel leaves them. LDS: the keys' first places [E + 1], then one running place for
// every key and wave [4][E + 1]. Wave w owns the w-th quarter of the chunk, 64 routes at a time in
// order; the lanes of one key find each other by ballots over the key's bits. 5.2 us at 16376 routes of
// 128 keys, 11.5 at 131072 of 256 (64 chunks, the counts of all chunks, sixteen loads at a time; one by one 29).
template <int PER, bool SCANNED>
__global__ __launch_bounds__(SORT_THREADS) void sort_place_kernel(const int32_t* __restrict__ ids, int R, int E,
                                                                  int key_bits, const int* __restrict__ counts,
                                                                  int chunks, int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ perm,
                                                                  int32_t* __restrict__ pos) {
  extern __shared__ int lds[];
  __shared__ int tmp[4];
  const int n = E + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x;
  int* total = lds;
  int* run = lds + n;
  for (int e = threadIdx.x; e < n; e += SORT_THREADS) {
    int before = 0, all = 0;
    if constexpr (SCANNED) {
      before = counts[(int64_t)c * n + e];
      all = counts[(int64_t)chunks * n + e];
    } else {
      for (int i0 = 0; i0 < chunks; i0 += 16) {  // sixteen loads on their way at once
        int v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = counts[(int64_t)(i0 + i < chunks ? i0 + i : chunks - 1) * n + e];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          all += i0 + i < chunks ? v[i] : 0;
          before += i0 + i < c ? v[i] : 0;
        }
      }
    }
    total[e] = all;
    run[e] = before;
    run[n + e] = run[2 * n + e] = run[3 * n + e] = 0;
  }
  __syncthreads();
  // exclusive sums of the totals: each thread its own consecutive keys
  const int span = (n + SORT_THREADS - 1) / SORT_THREADS;
  const int e0 = threadIdx.x * span;
  int sum = 0;
  for (int e = e0; e < e0 + span && e < n; ++e) sum += total[e];
  int at = block_exclusive(sum, tmp);
  for (int e = e0; e < e0 + span && e < n; ++e) {
    const int v = total[e];
    run[e] += at;
    if (c == 0) offsets[e] = at;
    at += v;
  }
  // the wave's own routes and their counts for the waves after it
  int key[PER];
  const int64_t r0 = ((int64_t)c * 4 + wave) * (64 * PER);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + 64 * i + lane;
    key[i] = r < R ? key_of(ids[r], E) : -1;
    if (key[i] >= 0 && wave < 3) atomicAdd(&run[(wave + 1) * n + key[i]], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += SORT_THREADS) {
    int v = run[e];
#pragma unroll
    for (int w = 1; w < 4; ++w) run[w * n + e] = v += run[w * n + e];
  }
  __syncthreads();
  int* mine = run + wave * n;
  const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = key[i] >= 0;
    uint64_t same = __ballot(in);
    for (int b = 0; b < key_bits; ++b) {
      const bool bit = (key[i] >> b) & 1;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    if (in) {
      const int rank = __popcll(same & below);
      const int first = mine[key[i]];
      sort_wave_fence();
      if (rank == 0) mine[key[i]] = first + __popcll(same);
      const int p = first + rank, r = (int)(r0 + 64 * i + lane);
      const bool valid = key[i] < E;
      perm[p] = valid ? r : ~r;
      pos[r] = valid ? p : ~p;
    }
    sort_wave_fence();
  }
}

// 16 bytes of a row at any alignment of its elements
__device__ __forceinline__ u32x4_t load16(const void* p) { return gload<u32x4_a2_t>(p); }
// Non-temporal, but for the sort's copies of up to SORT_CACHED bytes: of 2048 bf16 columns and 8 routes a
// token, the sort takes 118 us at 16384 tokens (138 with plain stores) and 37.5 at 4096 (34.2), the sums
// back 110 and 23.6 (120 and 24.4), their gradients 223 and 46.4 (229 and 48.9).
template <bool NT = true>
__device__ __forceinline__ void store16(void* p, const u32x4_t& v) {
  if constexpr (NT)
    __builtin_nontemporal_store(v, (u32x4_a2_t*)p);
  else
    *(u32x4_a2_t*)p = v;
}

// A call of few routes (sort_in_one) in one launch: block (token, piece of its row) counts the places of
// the token's routes itself, against all ids, while its part of the row is on its way; the block past
// the last token makes the offsets. G: room for the token's routes. key << 14 | route orders the routes by one comparison.
template <int ES, int G>
__global__ __launch_bounds__(SORT_THREADS) void sort_small_kernel(const uint8_t* __restrict__ x, int64_t x_stride,
                                                                  int64_t bytes, const int32_t* __restrict__ ids,
                                                                  int tokens, int top_k, int E,
                                                                  int32_t* __restrict__ offsets, int32_t* __restrict__ perm,
                                                                  int32_t* __restrict__ pos, uint8_t* __restrict__ rows) {
  static_assert(SORT_PIECE == 16 * SORT_THREADS, "a thread copies 16 bytes");
  static_assert(SORT_SMALL <= 1 << 14 && SORT_MAX_EXPERTS < 1 << 17, "an order fits 31 bits");
  extern __shared__ int lds[];  // the last block's E + 1 counts
  __shared__ int part[4][G];
  const int R = tokens * top_k, t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (t == tokens) {
    if (blockIdx.y) return;
    for (int e = threadIdx.x; e <= E; e += SORT_THREADS) lds[e] = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < R; r += SORT_THREADS) atomicAdd(&lds[key_of(ids[r], E)], 1);
    __syncthreads();
    const int per = (E + SORT_THREADS) / SORT_THREADS, e0 = threadIdx.x * per;
    int sum = 0;
    for (int e = e0; e < e0 + per && e <= E; ++e) sum += lds[e];
    int at = block_exclusive(sum, part[0]);
    for (int e = e0; e < e0 + per && e <= E; ++e) {
      offsets[e] = at;
      at += lds[e];
    }
    return;
  }
  const int64_t at = 16 * ((int64_t)blockIdx.y * SORT_THREADS + threadIdx.x);
  const int64_t b = at < bytes - 16 ? at : bytes - 16;
  u32x4_t v = {0, 0, 0, 0};
  const u32x4_t zero = v;
  if (rows && bytes >= 16 && at < bytes) v = load16(x + t * x_stride + b);
  int mine[G], count[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int r = t * top_k + (j < top_k ? j : top_k - 1);
    mine[j] = key_of(ids[r], E) << 14 | r;
    count[j] = 0;
  }
  for (int r0 = 64 * wave; r0 < R; r0 += 4 * SORT_THREADS) {  // four loads on their way at once
    int id[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = ids[r0 + i * SORT_THREADS + lane < R ? r0 + i * SORT_THREADS + lane : R - 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i * SORT_THREADS + lane;
      const int order = r < R ? key_of(id[i], E) << 14 | r : 0x7FFFFFFF;
#pragma unroll
      for (int j = 0; j < G; ++j) count[j] += __popcll(__ballot(order < mine[j]));
    }
  }
  if (lane == 0)
#pragma unroll
    for (int j = 0; j < G; ++j) part[wave][j] = count[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < G; ++j) {
    if (j < top_k) {
      const int p = part[0][j] + part[1][j] + part[2][j] + part[3][j];
      const bool valid = mine[j] >> 14 < E;
      const int r = t * top_k + j;
      if (blockIdx.y == 0 && threadIdx.x == 0) {
        perm[p] = valid ? r : ~r;
        pos[r] = valid ? p : ~p;
      }
      if (rows && at < bytes) {
        if (bytes >= 16) {
          store16(rows + p * bytes + b, valid ? v : zero);
        } else {
          using U = typename std::conditional<ES == 4, uint32_t, uint16_t>::type;
          for (int64_t i = 0; i < bytes / ES; ++i)
            ((U*)(rows + p * bytes))[i] = valid ? ((const U*)(x + t * x_stride))[i] : (U)0;
        }
      }
    }
  }
}

// A row of `bytes` bytes in 16-byte pieces, lane by lane; the last piece ends with the row and may
// overlap the one before it. Rows below 16 bytes go element by element (ES bytes each).
template <int ES, bool NT>
__global__ __launch_bounds__(64 * ROW_WAVES) void sort_rows_kernel(const uint8_t* __restrict__ x, int64_t x_stride,
                                                                   int64_t bytes, const int32_t* __restrict__ pos,
                                                                   int top_k, uint8_t* __restrict__ rows) {
  const int64_t t = blockIdx.x;
  const int64_t at = 16 * ((int64_t)blockIdx.y * blockDim.x + threadIdx.x);
  if (at >= bytes) return;
  const int32_t* tp = pos + t * top_k;
  if (bytes >= 16) {
    const int64_t b = at < bytes - 16 ? at : bytes - 16;
    const u32x4_t v = load16(x + t * x_stride + b), zero = {0, 0, 0, 0};
    for (int j = 0; j < top_k; ++j) {
      const int p = tp[j];
      store16<NT>(rows + (int64_t)(p >= 0 ? p : ~p) * bytes + b, p >= 0 ? v : zero);
    }
  } else {
    using E = typename std::conditional<ES == 4, uint32_t, uint16_t>::type;
    for (int64_t i = 0; i < bytes / ES; ++i) {
      const E v = ((const E*)(x + t * x_stride))[i];
      for (int j = 0; j < top_k; ++j) {
        const int p = tp[j];
        ((E*)(rows + (int64_t)(p >= 0 ? p : ~p) * bytes))[i] = p >= 0 ? v : (E)0;
      }
    }
  }
}

// V values of a row as loaded, and in fp32: 16 bytes of them, or one (rows shorter than 16 bytes)
template <typename T, int V>
struct Loaded {
  using W = typename std::conditional<V == 1, T, u32x4_t>::type;
  W w;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1)
      w = p[0];
    else
      w = load16(p);
  }
};
template <typename T, int V>
struct Piece {
  float f[V];
  __device__ __forceinline__ void take(const Loaded<T, V>& from) {
    if constexpr (V == 1) {
      f[0] = (float)from.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = from.w[i];  // a bit cast of w[i] itself takes element 0
        if constexpr (sizeof(T) == 4) {
          f[i] = __builtin_bit_cast(float, u);
        } else {
          f[2 * i] = (float)__builtin_bit_cast(T, (uint16_t)u);
          f[2 * i + 1] = (float)__builtin_bit_cast(T, (uint16_t)(u >> 16));
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      p[0] = (T)f[0];
    } else {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4)
          w[i] = __builtin_bit_cast(uint32_t, f[i]);
        else
          w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (T)f[2 * i]) |
                 (uint32_t)__builtin_bit_cast(uint16_t, (T)f[2 * i + 1]) << 16;
      }
      store16(p, w);
    }
  }
};

template <typename T, int V>
__global__ __launch_bounds__(64 * ROW_WAVES) void unsort_kernel(const T* __restrict__ rows, int64_t row_stride,
                                                                int64_t cols, const float* __restrict__ w,
                                                                const int32_t* __restrict__ pos, int top_k, int n_rows,
                                                                T* __restrict__ y) {
  const int64_t t = blockIdx.x;
  const int64_t at = V * ((int64_t)blockIdx.y * blockDim.x + threadIdx.x);
  if (at >= cols) return;
  const int64_t c = at < cols - V ? at : cols - V;
  Piece<T, V> acc;
#pragma unroll
  for (int i = 0; i < V; ++i) acc.f[i] = 0.0f;
  for (int j0 = 0; j0 < top_k; j0 += 8) {  // eight rows on their way at once
    int p[8];
    Loaded<T, V> v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = j0 + j < top_k ? pos[t * top_k + j0 + j] : -1;
      if (p[j] >= n_rows) p[j] = -1;
      if (p[j] >= 0) v[j].load(rows + p[j] * row_stride + c);  // uniform
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (p[j] >= 0) {
        const float wj = w ? w[t * top_k + j0 + j] : 1.0f;
        Piece<T, V> o;
        o.take(v[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) acc.f[i] = fmaf(wj, o.f[i], acc.f[i]);
      }
    }
  }
  acc.store(y + t * cols + c);
}

// One block a token: dy[t] against its routes' rows. The dots are summed a lane's own pieces first,
// then over the wave's lanes and over the waves, always in the same order.
template <typename T, int V>
__global__ __launch_bounds__(64 * ROW_WAVES) void unsort_grad_kernel(const T* __restrict__ dy, int64_t dy_stride,
                                                                     const T* __restrict__ rows, int64_t row_stride,
                                                                     int64_t cols, const float* __restrict__ w,
                                                                     const int32_t* __restrict__ pos, int top_k,
                                                                     int n_rows, T* __restrict__ drows,
                                                                     float* __restrict__ dw) {
  __shared__ float part[ROW_WAVES][8];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int j0 = 0; j0 < top_k; j0 += 8) {
    int p[8];
    float wj[8], dot[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = j0 + j < top_k ? pos[t * top_k + j0 + j] : n_rows;  // n_rows: no row at all
      wj[j] = p[j] >= 0 && p[j] < n_rows ? (w ? w[t * top_k + j0 + j] : 1.0f) : 0.0f;
      dot[j] = 0.0f;
    }
    for (int64_t at = (int64_t)V * threadIdx.x; at < cols; at += (int64_t)V * blockDim.x) {
      const int64_t c = at < cols - V ? at : cols - V;
      const int skip = (int)(at - c);  // values of this piece that the one before holds too
      Loaded<T, V> dl, l[8];
      dl.load(dy + t * dy_stride + c);
      if (dw)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (p[j] >= 0 && p[j] < n_rows) l[j].load(rows + p[j] * row_stride + c);  // uniform
      Piece<T, V> d;
      d.take(dl);
      if (drows)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int q = p[j] >= 0 ? p[j] : ~p[j];
          if (q < n_rows) {
            Piece<T, V> r;
#pragma unroll
            for (int i = 0; i < V; ++i) r.f[i] = p[j] >= 0 ? wj[j] * d.f[i] : 0.0f;
            r.store(drows + q * cols + c);
          }
        }
      if (dw)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (p[j] >= 0 && p[j] < n_rows) {
            Piece<T, V> o;
            o.take(l[j]);
#pragma unroll
            for (int i = 0; i < V; ++i) dot[j] = i < skip ? dot[j] : fmaf(d.f[i], o.f[i], dot[j]);
          }
    }
    if (dw) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int s = 32; s; s >>= 1) dot[j] += __shfl_xor(dot[j], s);
      if (j0) __syncthreads();
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[wave][j] = dot[j];
      __syncthreads();
      const int j = threadIdx.x;
      if (j < 8 && j0 + j < top_k) {
        float all = 0.0f;
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) all += part[i][j];
        dw[t * top_k + j0 + j] = all;  // without a row: its sums are 0
      }
    }
  }
}

int row_threads(int64_t pieces) { return (int)(pieces >= 64 * ROW_WAVES ? 64 * ROW_WAVES : (pieces + 63) / 64 * 64); }

}  // namespace

// Routes a thread: few, for more blocks, as long as the blocks' counts stay few to add up
static int sort_per(int64_t routes) { return routes <= 65536 ? 2 : SORT_MAX_PER; }
static int64_t sort_chunks(int64_t routes) {
  const int64_t chunk = sort_per(routes) * SORT_THREADS;
  return (routes + chunk - 1) / chunk;
}
// Comparisons of the order in one launch; where it does not take the routes, more than any limit
static int64_t sort_work(int64_t tokens, int64_t top_k) {
  if (tokens * top_k > SORT_SMALL || top_k > SORT_SMALL_K) return INT64_MAX;
  return tokens * (tokens * top_k) * (top_k > 8 ? 32 : 8);
}
static bool sort_in_one(int64_t tokens, int64_t top_k, int64_t pieces) {  // pieces of a row, 0: the order alone
  const int64_t work = sort_work(tokens, top_k);
  if (work <= SORT_NO_WS) return true;
  return pieces ? work <= SORT_ROWS_WORK / pieces : work <= SORT_ORDER_WORK;
}
int64_t moe_sort_counts(int64_t tokens, int64_t top_k) {
  if (sort_work(tokens, top_k) <= SORT_NO_WS) return 0;
  const int64_t chunks = sort_chunks(tokens * top_k);
  return chunks + 1;  // and their totals, of many chunks
}

int launch_moe_sort(const uint8_t* x, int es, int64_t x_stride, int64_t cols, const int32_t* ids, int64_t tokens,
                    int64_t top_k, int64_t E, uint8_t* rows, int32_t* offsets, int32_t* perm, int32_t* pos, int* counts,
                    hipStream_t stream) {
  const int R = (int)(tokens * top_k), n = (int)E + 1;
  int bits = 0;
  while ((n - 1) >> bits) ++bits;
  const int64_t row_pieces = rows ? (cols * es + SORT_PIECE - 1) / SORT_PIECE : 0;
  if (sort_in_one(tokens, top_k, row_pieces)) {
    const int64_t bytes = rows ? cols * es : 1;
    dim3 grid((unsigned)tokens + 1, rows ? (unsigned)row_pieces : 1);
    auto kernel = es == 4 ? (top_k > 8 ? sort_small_kernel<4, 16> : sort_small_kernel<4, 8>)
                          : (top_k > 8 ? sort_small_kernel<2, 16> : sort_small_kernel<2, 8>);
    kernel<<<grid, SORT_THREADS, n * sizeof(int), stream>>>(x, x_stride * es, bytes, ids, (int)tokens, (int)top_k, (int)E,
                                                            offsets, perm, pos, rows);
    KTMI_HIP_TRY(hipGetLastError());
    return KTMI_OK;
  }
  const int chunks = (int)sort_chunks(R);
  const bool few = sort_per(R) == 2, scan = !few && chunks > SORT_SCAN;
  auto count = few ? sort_count_kernel<2> : sort_count_kernel<SORT_MAX_PER>;
  auto place = few ? sort_place_kernel<2, false> : scan ? sort_place_kernel<SORT_MAX_PER, true> : sort_place_kernel<SORT_MAX_PER, false>;
  count<<<chunks, SORT_THREADS, n * sizeof(int), stream>>>(ids, R, (int)E, counts);
  if (scan) sort_scan_kernel<<<(n + 63) / 64, 64 * SCAN_WAVES, 0, stream>>>(counts, chunks, n);
  place<<<chunks, SORT_THREADS, 5 * n * sizeof(int), stream>>>(ids, R, (int)E, bits, counts, chunks, offsets, perm, pos);
  if (rows) {
    const int64_t bytes = cols * es, pieces = (bytes + 15) / 16;
    const int th = row_threads(pieces);
    const bool nt = (int64_t)R * bytes > SORT_CACHED;
    auto kernel = es == 4 ? (nt ? sort_rows_kernel<4, true> : sort_rows_kernel<4, false>)
                          : (nt ? sort_rows_kernel<2, true> : sort_rows_kernel<2, false>);
    for (int64_t t = 0; t < tokens; t += ROW_TOKENS) {
      dim3 grid((unsigned)(tokens - t < ROW_TOKENS ? tokens - t : ROW_TOKENS), (unsigned)((pieces + th - 1) / th));
      kernel<<<grid, th, 0, stream>>>(x + t * x_stride * es, x_stride * es, bytes, pos + t * top_k, (int)top_k, rows);
    }
  }
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

namespace {

template <typename T>
void unsort_of(const void* rows, int64_t row_stride, int64_t cols, const float* w, const int32_t* pos, int64_t tokens,
               int64_t top_k, void* y, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int v = cols >= V ? V : 1;
  const int64_t pieces = (cols + v - 1) / v;
  const int th = row_threads(pieces), R = (int)(tokens * top_k);
  auto kernel = v == V ? unsort_kernel<T, V> : unsort_kernel<T, 1>;
  for (int64_t t = 0; t < tokens; t += ROW_TOKENS) {
    dim3 grid((unsigned)(tokens - t < ROW_TOKENS ? tokens - t : ROW_TOKENS), (unsigned)((pieces + th - 1) / th));
    kernel<<<grid, th, 0, stream>>>((const T*)rows, row_stride, cols, w ? w + t * top_k : w, pos + t * top_k, (int)top_k, R,
                                    (T*)y + t * cols);
  }
}

template <typename T>
void unsort_grad_of(const void* dy, int64_t dy_stride, const void* rows, int64_t row_stride, int64_t cols, const float* w,
                    const int32_t* pos, int64_t tokens, int64_t top_k, void* drows, float* dw, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int v = cols >= V ? V : 1;
  const int th = row_threads((cols + v - 1) / v), R = (int)(tokens * top_k);
  auto kernel = v == V ? unsort_grad_kernel<T, V> : unsort_grad_kernel<T, 1>;
  for (int64_t t = 0; t < tokens; t += ROW_TOKENS)
    kernel<<<(unsigned)(tokens - t < ROW_TOKENS ? tokens - t : ROW_TOKENS), th, 0, stream>>>(
        (const T*)dy + t * dy_stride, dy_stride, (const T*)rows, row_stride, cols, w ? w + t * top_k : w, pos + t * top_k,
        (int)top_k, R, (T*)drows, dw ? dw + t * top_k : dw);
}

}  // namespace

int launch_moe_unsort(const void* rows, int dtype, int64_t row_stride, int64_t cols, const float* w, const int32_t* pos,
                      int64_t tokens, int64_t top_k, void* y, hipStream_t stream) {
  switch (dtype) {
    case KTMI_F32: unsort_of<float>(rows, row_stride, cols, w, pos, tokens, top_k, y, stream); break;
    case KTMI_F16: unsort_of<_Float16>(rows, row_stride, cols, w, pos, tokens, top_k, y, stream); break;
    default: unsort_of<__bf16>(rows, row_stride, cols, w, pos, tokens, top_k, y, stream); break;
  }
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

int launch_moe_unsort_grad(const void* dy, int64_t dy_stride, const void* rows, int64_t row_stride, int dtype,
                           int64_t cols, const float* w, const int32_t* pos, int64_t tokens, int64_t top_k, void* drows,
                           float* dw, hipStream_t stream) {
  switch (dtype) {
    case KTMI_F32:
      unsort_grad_of<float>(dy, dy_stride, rows, row_stride, cols, w, pos, tokens, top_k, drows, dw, stream);
      break;
    case KTMI_F16:
      unsort_grad_of<_Float16>(dy, dy_stride, rows, row_stride, cols, w, pos, tokens, top_k, drows, dw, stream);
      break;
    default: unsort_grad_of<__bf16>(dy, dy_stride, rows, row_stride, cols, w, pos, tokens, top_k, drows, dw, stream); break;
  }
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

}  // namespace ktmi
