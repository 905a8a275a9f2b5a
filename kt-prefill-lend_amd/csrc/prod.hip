// The products by expert: which kernel a call takes (prod_tile.h: tiles of rows, prod_rows.h: few rows a matrix).
#include "prod_rows.h"

namespace ktmi {

namespace {

ProdTable table(int dtype) {
  return dtype == KTMI_F32 ? prod_table_f32() : dtype == KTMI_F16 ? prod_table_f16() : prod_table_bf16();
}

int size_of(int dtype) { return dtype == KTMI_F32 ? 4 : 2; }

// bytes of rows; whole words, as buffer loads count them (a word that holds the last 16 bits is there as a whole)
int64_t bytes_of(int64_t rows, int64_t stride, int64_t width) { return rows > 0 ? ((rows - 1) * stride + width + 3) / 4 * 4 : 0; }

int64_t mean_rows(int64_t rows, int64_t n_experts) { return (rows + n_experts - 1) / n_experts; }

int64_t ints(int64_t n) { return (n + 3) / 4 * 4; }

// Whether the kernel for few rows runs: up to 32 a matrix, where tiles of 128 of its rows would be too few blocks to keep
// the CUs' loads on their way, the fewer the more rows of x there are to read for each. One limit for all types. us by 4096
// columns, weights from HBM, in this kernel and in tiles: e4m3 one row by 16384 17 / 21, 65280 59 / 67, 131072 111 / 128; 16 rows by
// 8192 13 / 17, 16384 20 / 21, 32768 38 / 31; 32 rows by 4096 15 / 16, 7168 27 / 18. bf16 one row by 16384 27 / 30, 65280 104 / 99,
// 131072 195 / 174; 16 rows by 8192 21 / 21, 16384 40 / 30, 32768 60 / 65; 32 rows by 4096 15 / 15, 7168 26 / 20. So at
// 32 rows the limit is late: from about 6000 rows of w on tiles take less.
bool few_rows(int64_t mean, int64_t parts, int64_t n) {
  return mean <= 32 && parts * ((n + 127) / 128) < (mean <= 4 ? 512 : mean <= 16 ? 256 : 64);
}

// A product's tiles and the blocks that share a tile's k.
struct TilePlan {
  int size, splits;
};

// The splits of a tile's `steps` that take the least time by this count, and that time in us: a step takes 0.5 us in a
// block of four waves that has its CU to itself, 0.3 us for each that shares it, 1 us in one of eight (in fp32 twice that);
// a slice of sums is written and read at 4 TB/s, and adding them up is a launch more (3 us). (512 rows by 4096 x 7168 bf16: 61 us,
// with three splits 46; by 7168 x 2048: 25 us, with two 40.)
TilePlan split_tiles(int size, int es, int64_t tiles, int64_t steps, int64_t values, double* us) {
  const bool four = size == TILE_LOW || size == TILE_SMALL;
  const int64_t slots = size == TILE_LOW && es != 2 ? 768 : four ? 512 : 256;
  TilePlan best = {size, 1};
  for (int64_t s = 1; s <= 16 && (s == 1 || (tiles * s <= slots && steps >= 8 * s)); ++s) {
    const int64_t blocks = tiles * s, rounds = (blocks + slots - 1) / slots, shared = (blocks + 255) / 256;
    const double step = (four ? (shared > 1 ? 0.3 * (shared < slots / 256 ? shared : slots / 256) : 0.5) : 1.0) * (es == 4 ? 2 : 1);
    const double t = (double)rounds * (double)((steps + s - 1) / s) * step + (s > 1 ? 3 + 2e-6 * (double)(s * values) : 0);
    if (s == 1 || t < *us) *us = t, best.splits = (int)s;
  }
  return best;
}

// m: rows of a matrix (gradient of w: of its rows), parts matrices.
TilePlan plan_tiles(int mode, int es, int64_t m, int64_t n, int64_t steps, int64_t parts) {
  auto tiles = [&](int size) { return parts * ((m + tile_m(size) - 1) / tile_m(size)) * ((n + tile_n(size) - 1) / tile_n(size)); };
  auto split = [&](int size, double* us) { return split_tiles(size, es, tiles(size), steps, parts * m * n, us); };
  double us, other;
  if (mode == PROD_DW) {
    const TilePlan small = split(TILE_SMALL, &us), large = split(TILE_LARGE, &other);
    return es == 2 && (tiles(TILE_LARGE) >= 192 || other < us) ? large : small;
  }
  if (m <= (es == 4 ? 256 : 64) || tiles(TILE_SMALL) < 192) return split(TILE_LOW, &us);
  // (8-bit, 64 experts of 1024 x 2048, us in tiles of 128 / 256 rows: each 256 rows 67 / 62, 300 94 / 99, 400 125 / 108, 512 143 / 124; uneven
  // ones of such a mean 86 / 93, 101 / 103, 125 / 139, 155 / 153, of 600 183 / 169)
  if (m >= 512 && tiles(TILE_LARGE) >= 192) return {TILE_LARGE, 1};
  if (mode == PROD_FWD && es != 1 && tiles(TILE_DEEP) >= 192) return {TILE_DEEP, 1};
  return split(TILE_SMALL, &us);
}

int64_t slice_of(int64_t values) { return ints(values); }

struct ProdPlan {
  bool few;
  TilePlan tiles;
  int64_t rows, width;  // of the sums that splits keep
};
ProdPlan plan_prod(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows) {
  const int es = size_of(dtype);
  const int64_t mean = mean_rows(n_rows, n_experts), parts = n_experts < n_rows ? n_experts : n_rows, bk = STEP_BYTES / es;
  auto steps = [&](int64_t k) { return (k + bk - 1) / bk; };
  ProdPlan p = {};
  switch (what) {
    case KTMI_PROD_GATED:
    case KTMI_PROD_LINEAR: {
      const int64_t n = what == KTMI_PROD_GATED ? 2 * rows : rows;
      p.few = few_rows(mean, parts, n);
      p.tiles = plan_tiles(PROD_FWD, es, mean, n, steps(cols), parts);
      p.rows = n_rows, p.width = n;
      break;
    }
    case KTMI_PROD_GRAD_X:
      p.tiles = plan_tiles(PROD_DX, es, mean, cols, steps(rows), parts);
      p.rows = n_rows, p.width = cols;
      break;
    default:
      p.tiles = plan_tiles(PROD_DW, es, rows, cols, steps(mean), n_experts);
      p.rows = n_experts * rows, p.width = cols;
  }
  if (p.few || n_rows == 0) p.tiles.splits = 1;
  return p;
}

}  // namespace

int64_t prod_workspace(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows) {
  const ProdPlan p = plan_prod(what, dtype, rows, cols, n_experts, n_rows);
  return p.tiles.splits > 1 ? 4 * p.tiles.splits * slice_of(p.rows * p.width) : 0;
}

static ktmi_prod_kernel told(bool few, const TilePlan& p) {
  if (few) return {0, 0, 1};
  return {tile_m(p.size), tile_n(p.size), p.splits};
}

ktmi_prod_kernel prod_kernel_of(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows) {
  const ProdPlan p = plan_prod(what, dtype, rows, cols, n_experts, n_rows);
  return told(p.few, p.tiles);
}

int launch_prod(int what, const ProdArgs& a, hipStream_t stream) {
  const int es = size_of(a.dtype);
  const Segments seg = {a.offsets, (int)a.n_experts, (int)a.n_rows};
  const ProdPlan p = plan_prod(what, a.dtype, a.rows, a.cols, a.n_experts, a.n_rows);
  const bool gated = what == KTMI_PROD_GATED;
  const int64_t w_rows = gated ? 2 * a.rows : a.rows;
  const ProdTable ops = table(a.dtype);
  if (p.few) {
    RowsArgs r = {};
    r.x = a.x, r.x_stride = a.x_stride, r.w = (const uint8_t*)a.w, r.y = a.y, r.w_expert = w_rows * a.cols * es;
    r.N = (int)a.rows, r.K = (int)a.cols, r.R = (int)a.n_rows, r.act = a.act, r.gu = a.sums, r.top_k = 1, r.seg = seg;
    return ops.rows(false, gated, r, (int)mean_rows(a.n_rows, a.n_experts), stream);
  }
  TileArgs t = {};
  const uint8_t *x = (const uint8_t*)a.x, *dy = (const uint8_t*)a.dy;
  const int64_t x_stride = a.x_stride * es, dy_stride = a.dy_stride * es;
  const int64_t x_bytes = bytes_of(a.n_rows, x_stride, a.cols * es), dy_bytes = bytes_of(a.n_rows, dy_stride, a.rows * es);
  t.seg = seg, t.c = a.y, t.gu = a.sums, t.act = a.act;
  t.splits = p.tiles.splits, t.part = a.part, t.slice = slice_of(p.rows * p.width);
  t.q = (const uint8_t*)a.w, t.q_stride = a.cols * es, t.q_bytes = t.q_expert = w_rows * a.cols * es;
  int mode = PROD_FWD;
  if (what == KTMI_PROD_GRAD_X) {
    mode = PROD_DX;
    t.p = dy, t.p_stride = dy_stride, t.p_bytes = dy_bytes;
    t.c_stride = a.cols, t.M = (int)a.n_rows, t.N = (int)a.cols, t.K = (int)a.rows;
  } else if (what == KTMI_PROD_GRAD_W) {
    mode = PROD_DW;
    t.p = dy, t.p_stride = dy_stride, t.p_bytes = dy_bytes;
    t.q = x, t.q_stride = x_stride, t.q_bytes = x_bytes, t.q_expert = 0;
    t.c_stride = a.cols, t.c_expert = a.rows * a.cols, t.M = (int)a.rows, t.N = (int)a.cols, t.K = (int)a.n_rows;
  } else {
    t.p = x, t.p_stride = x_stride, t.p_bytes = x_bytes;
    t.c_stride = a.rows, t.M = (int)a.n_rows, t.N = (int)a.rows, t.K = (int)a.cols;
  }
  const int rc = ops.tile(mode, gated, t, p.tiles.size, stream);
  if (rc || t.splits == 1) return rc;
  return ops.sum(gated, t.part, t.splits, t.slice, p.rows, gated ? a.rows : p.width, a.act, a.y, a.sums, stream);
}

int launch_gated_grad(const float* sums, const void* dh, int dtype, int64_t dh_stride, int64_t inter, int64_t n_rows, int act,
                      void* dsums, hipStream_t stream) {
  return table(dtype).gated_grad(sums, dh, dh_stride, inter, n_rows, act, dsums, stream);
}

// ---- 8-bit floating point. Workspace of many rows: their codes and scales; of routes past 64: their order.
static int64_t fp8_order_bytes(int64_t tokens, int64_t top_k, int64_t E) {
  const int64_t R = tokens * top_k;
  return R <= 64 ? 0 : 4 * (ints(E + 1) + 2 * ints(R) + ints(moe_sort_counts(tokens, top_k) * (E + 1)));
}

namespace {
struct Fp8Plan {
  bool few;
  TilePlan tiles;
};
Fp8Plan plan_fp8(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids) {
  const int64_t R = x_rows * top_k, mean = mean_rows(R, n_experts), parts = n_experts < R ? n_experts : R;
  Fp8Plan p = {};
  // Up to 64 routes are taken as they come, without the order's and the quantisation's launches. (64 routes by 4096 x 7168 of 4
  // experts 33 us, in tiles, that is of 65 routes, 35; of 8 experts 53 / 53. Where many of them share an expert tiles take less: of one
  // or two experts 58 / 25, by 65280 x 2048 338 / 41.)
  p.few = (ids && R <= 64) || few_rows(mean, parts, rows);
  p.tiles = plan_tiles(PROD_FWD, 1, mean, rows, (cols + 127) / 128, parts);
  if (cols % 16 && p.tiles.size == TILE_LARGE) p.tiles.size = TILE_SMALL;  // codes through registers: no tiles of 256 rows
  if (cols > (1 << 22)) p.tiles.size = TILE_LOW;  // 32-bit offsets reach the codes of 64 rows of 2^24, of 256 of 2^22
  if (p.few) p.tiles.splits = 1;
  return p;
}
}  // namespace

ktmi_prod_kernel fp8_kernel_of(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids) {
  const Fp8Plan p = plan_fp8(rows, cols, x_rows, n_experts, top_k, ids);
  return told(p.few, p.tiles);
}

static int64_t fp8_slice_workspace(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids) {
  const int64_t blocks = (cols + 127) / 128;
  const int64_t order = ids ? fp8_order_bytes(x_rows, top_k, n_experts) : 0;
  const Fp8Plan p = plan_fp8(rows, cols, x_rows, n_experts, top_k, ids);
  if (p.few) return order;
  return order + 4 * ints(blocks * x_rows) + x_rows * blocks * 128 +
         (p.tiles.splits > 1 ? 4 * p.tiles.splits * slice_of(x_rows * top_k * rows) : 0);
}

static int launch_fp8_slice(const Fp8Args& a, hipStream_t stream) {
  const int64_t R = a.x_rows * a.top_k, mean = mean_rows(R, a.n_experts), blocks = (a.cols + 127) / 128;
  Segments seg = {a.offsets, (int)a.n_experts, (int)R};
  const int32_t *perm = nullptr, *ids = a.ids;
  const Fp8Plan plan = plan_fp8(a.rows, a.cols, a.x_rows, a.n_experts, a.top_k, ids);
  uint8_t* ws = a.ws;
  if (!plan.few) {  // before the first launch: what fp8_tile's grid would be refused for
    const int bm = tile_m(plan.tiles.size);
    const int64_t grid = (R / bm + a.n_experts + 2) * ((a.rows + 127) / 128) * plan.tiles.splits;
    KTMI_REQUIRE(grid < 0xffffffffll / 256, KTMI_EINVAL, "a grid of %lld blocks (below 2^32 threads)", (long long)grid);
  }
  if (ids && R > 64) {
    int* offsets = (int*)ws;
    int* p = offsets + ints(a.n_experts + 1);
    int* pos = p + ints(R);
    const int rc = launch_moe_sort(nullptr, 2, 0, 0, ids, a.x_rows, a.top_k, a.n_experts, nullptr, offsets, p, pos,
                                   pos + ints(R), stream);
    if (rc) return rc;
    ws += fp8_order_bytes(a.x_rows, a.top_k, a.n_experts);
    seg.offsets = offsets, perm = p, ids = nullptr;
  }
  const ProdTable t = table(a.dtype);
  if (plan.few) {
    RowsArgs r = {};
    r.x = a.x, r.x_stride = a.x_stride, r.w = a.w, r.ws = a.scales, r.y = a.y, r.w_expert = a.rows * a.cols;
    r.N = (int)a.rows, r.K = (int)a.cols, r.R = (int)R, r.ids = ids, r.top_k = (int)a.top_k, r.seg = seg, r.perm = perm;
    return t.rows(true, false, r, (int)mean, stream);
  }
  float* xs = (float*)ws;
  uint8_t* codes = ws + 4 * ints(blocks * a.x_rows);
  int rc = t.quantise(a.x, a.x_stride, a.cols, a.x_rows, a.offsets ? a.offsets + a.n_experts : nullptr, codes, xs, stream);
  if (rc) return rc;
  Fp8TileArgs f = {};
  f.x = codes, f.xs = xs, f.x_stride = blocks * 128, f.xs_stride = a.x_rows, f.x_rows = a.x_rows;
  f.w = a.w, f.ws = a.scales, f.y = a.y, f.M = (int)R, f.N = (int)a.rows, f.K = (int)a.cols, f.seg = seg;
  f.perm = perm, f.top_k = (int)a.top_k;
  f.splits = plan.tiles.splits, f.part = (float*)(codes + a.x_rows * blocks * 128), f.slice = slice_of(R * a.rows);
  rc = t.fp8_tile(f, plan.tiles.size, stream);
  if (rc || f.splits == 1) return rc;
  return t.sum(false, f.part, f.splits, f.slice, R, a.rows, 0, a.y, nullptr, stream);
}

// Routes past 64 gather their tokens' codes by 32-bit offsets: tokens in slices of less than 2 GiB of codes.
static int64_t fp8_slice_rows(int64_t cols) { return 0x7fffffff / ((cols + 127) / 128 * 128); }

int64_t fp8_workspace(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids) {
  const int64_t most = fp8_slice_rows(cols);
  if (!ids || x_rows <= most) return fp8_slice_workspace(rows, cols, x_rows, n_experts, top_k, ids);
  const int64_t rest = x_rows % most, a = fp8_slice_workspace(rows, cols, most, n_experts, top_k, ids);
  const int64_t b = rest ? fp8_slice_workspace(rows, cols, rest, n_experts, top_k, ids) : 0;
  return a > b ? a : b;
}

int launch_fp8(const Fp8Args& a, hipStream_t stream) {
  const int64_t most = fp8_slice_rows(a.cols);
  if (!a.ids || a.x_rows <= most) return launch_fp8_slice(a, stream);
  const int es = size_of(a.dtype);
  for (int64_t t0 = 0; t0 < a.x_rows; t0 += most) {
    Fp8Args b = a;
    b.x = (const uint8_t*)a.x + t0 * a.x_stride * es;
    b.x_rows = a.x_rows - t0 < most ? a.x_rows - t0 : most;
    b.ids = a.ids + t0 * a.top_k;
    b.y = (uint8_t*)a.y + t0 * a.top_k * a.rows * es;
    const int rc = launch_fp8_slice(b, stream);
    if (rc) return rc;
  }
  return KTMI_OK;
}

}  // namespace ktmi
