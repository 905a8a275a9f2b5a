// The products by expert: which kernel a call takes (prod_tile.h: tiles of rows, prod_rows.h: few rows a matrix).
#include "prod_rows.h"

namespace ktmi {

namespace {

ProdTable table(int dtype) {
  return dtype == KTMI_F32 ? prod_table_f32() : dtype == KTMI_F16 ? prod_table_f16() : prod_table_bf16();
}

int size_of(int dtype) { return dtype == KTMI_F32 ? 4 : 2; }

int64_t bytes_of(int64_t rows, int64_t stride, int64_t width) { return rows > 0 ? (rows - 1) * stride + width : 0; }

// rows a matrix up to which the kernels for few rows run
constexpr int64_t FEW_ROWS = 64;

int64_t mean_rows(int64_t rows, int64_t n_experts) { return (rows + n_experts - 1) / n_experts; }

int64_t ints(int64_t n) { return (n + 3) / 4 * 4; }

}  // namespace

int launch_prod_fwd(const ProdArgs& a, bool gated, hipStream_t stream) {
  const int es = size_of(a.dtype);
  const Segments seg = {a.offsets, (int)a.n_experts, (int)a.n_rows};
  const int64_t w_rows = gated ? 2 * a.rows : a.rows, mean = mean_rows(a.n_rows, a.n_experts);
  if (mean <= FEW_ROWS) {
    RowsArgs r = {};
    r.x = a.x, r.x_stride = a.x_stride, r.w = (const uint8_t*)a.w, r.y = a.y, r.w_expert = w_rows * a.cols * es;
    r.N = (int)a.rows, r.K = (int)a.cols, r.R = (int)a.n_rows, r.act = a.act, r.gu = a.sums, r.top_k = 1, r.seg = seg;
    return table(a.dtype).rows(false, gated, r, (int)mean, stream);
  }
  TileArgs t = {};
  t.p = (const uint8_t*)a.x, t.p_stride = a.x_stride * es, t.p_bytes = bytes_of(a.n_rows, a.x_stride * es, a.cols * es);
  t.q = (const uint8_t*)a.w, t.q_stride = a.cols * es, t.q_bytes = t.q_expert = w_rows * a.cols * es;
  t.c = a.y, t.c_stride = a.rows, t.M = (int)a.n_rows, t.N = (int)a.rows, t.K = (int)a.cols, t.seg = seg;
  t.gu = a.sums, t.act = a.act;
  return table(a.dtype).tile(PROD_FWD, gated, t, stream);
}

int launch_prod_dx(const ProdArgs& a, hipStream_t stream) {
  const int es = size_of(a.dtype);
  TileArgs t = {};
  t.p = (const uint8_t*)a.dy, t.p_stride = a.dy_stride * es, t.p_bytes = bytes_of(a.n_rows, a.dy_stride * es, a.rows * es);
  t.q = (const uint8_t*)a.w, t.q_stride = a.cols * es, t.q_bytes = t.q_expert = a.rows * a.cols * es;
  t.c = a.y, t.c_stride = a.cols, t.M = (int)a.n_rows, t.N = (int)a.cols, t.K = (int)a.rows;
  t.seg = {a.offsets, (int)a.n_experts, (int)a.n_rows};
  return table(a.dtype).tile(PROD_DX, false, t, stream);
}

int launch_prod_dw(const ProdArgs& a, hipStream_t stream) {
  const int es = size_of(a.dtype);
  TileArgs t = {};
  t.p = (const uint8_t*)a.dy, t.p_stride = a.dy_stride * es, t.p_bytes = bytes_of(a.n_rows, a.dy_stride * es, a.rows * es);
  t.q = (const uint8_t*)a.x, t.q_stride = a.x_stride * es, t.q_bytes = bytes_of(a.n_rows, a.x_stride * es, a.cols * es);
  t.c = a.y, t.c_stride = a.cols, t.c_expert = a.rows * a.cols, t.M = (int)a.rows, t.N = (int)a.cols, t.K = (int)a.n_rows;
  t.seg = {a.offsets, (int)a.n_experts, (int)a.n_rows};
  return table(a.dtype).tile(PROD_DW, false, t, stream);
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

int64_t fp8_workspace(int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids) {
  const int64_t blocks = (cols + 127) / 128, mean = mean_rows(x_rows * top_k, n_experts);
  const int64_t order = ids ? fp8_order_bytes(x_rows, top_k, n_experts) : 0;
  if (mean <= FEW_ROWS) return order;
  return order + 4 * ints(blocks * x_rows) + x_rows * blocks * 128;
}

static int launch_fp8_slice(const Fp8Args& a, hipStream_t stream) {
  const int64_t R = a.x_rows * a.top_k, mean = mean_rows(R, a.n_experts), blocks = (a.cols + 127) / 128;
  Segments seg = {a.offsets, (int)a.n_experts, (int)R};
  const int32_t *perm = nullptr, *ids = a.ids;
  uint8_t* ws = a.ws;
  if (mean > FEW_ROWS && !(ids && R <= 64)) {  // before the first launch: what fp8_tile's grid would be refused for
    const int64_t grid = (R / 128 + a.n_experts + 2) * ((a.rows + 127) / 128);
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
  if (mean <= FEW_ROWS || ids) {
    RowsArgs r = {};
    r.x = a.x, r.x_stride = a.x_stride, r.w = a.w, r.ws = a.scales, r.y = a.y, r.w_expert = a.rows * a.cols;
    r.N = (int)a.rows, r.K = (int)a.cols, r.R = (int)R, r.ids = ids, r.top_k = (int)a.top_k, r.seg = seg, r.perm = perm;
    return t.rows(true, false, r, (int)mean, stream);
  }
  float* xs = (float*)ws;
  uint8_t* codes = ws + 4 * ints(blocks * a.x_rows);
  const int rc = t.quantise(a.x, a.x_stride, a.cols, a.x_rows, a.offsets ? a.offsets + a.n_experts : nullptr, codes, xs, stream);
  if (rc) return rc;
  Fp8TileArgs f = {};
  f.x = codes, f.xs = xs, f.x_stride = blocks * 128, f.xs_stride = a.x_rows, f.x_rows = a.x_rows;
  f.w = a.w, f.ws = a.scales, f.y = a.y, f.M = (int)R, f.N = (int)a.rows, f.K = (int)a.cols, f.seg = seg;
  f.perm = perm, f.top_k = (int)a.top_k;
  return t.fp8_tile(f, stream);
}

// Routes past 64 gather their tokens' codes by 32-bit offsets: tokens in slices of less than 2 GiB of codes.
int launch_fp8(const Fp8Args& a, hipStream_t stream) {
  const int64_t most = 0x7fffffff / ((a.cols + 127) / 128 * 128);
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
