// extern "C" entry points of libktmi.so: argument checks, workspace carve-up, dispatch.
#include <mutex>

#include <stdarg.h>
#include <stdio.h>

#include "kernels.h"

namespace ktmi {

static thread_local char g_err[512] = "";

void clear_error() { g_err[0] = 0; }

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof g_err, fmt, ap);
  va_end(ap);
}

static bool type_ok(int t) { return t == GGML_Q8_0 || t == GGML_Q4_K || t == GGML_Q6_K || t == GGML_IQ3_S; }
static bool dtype_ok(int d) { return d == KTMI_F32 || d == KTMI_F16 || d == KTMI_BF16; }
static bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

static thread_local hipEvent_t g_stage_events[KTMI_STAGE_EVENTS];
static thread_local int g_stage_on = 0;

void record_stage(int i, hipStream_t stream) {
  if (g_stage_on && i >= 0 && i < KTMI_STAGE_EVENTS && g_stage_events[i]) (void)hipEventRecord(g_stage_events[i], stream);
}

// routes per call above which KTMI_MODE_AUTO takes the grouped MFMA path
static const int64_t kGemvMaxRoutes = 256;

}  // namespace ktmi

using namespace ktmi;

extern "C" {

const char* ktmi_last_error(void) { return g_err; }

int ktmi_version(void) { return 100; }

int ktmi_set_stage_events(void* const* events, int n) {
  g_err[0] = 0;
  if (n == 0 || events == nullptr) {
    g_stage_on = 0;
    return KTMI_OK;
  }
  KTMI_REQUIRE(n == KTMI_STAGE_EVENTS, KTMI_EINVAL, "set_stage_events: %d events (need %d)", n, KTMI_STAGE_EVENTS);
  for (int i = 0; i < n; ++i) g_stage_events[i] = (hipEvent_t)events[i];
  g_stage_on = 1;
  return KTMI_OK;
}

int ktmi_type_supported(int ggml_type) { return type_ok(ggml_type) ? 1 : 0; }

int64_t ktmi_row_bytes(int64_t cols, int ggml_type) {
  if (!type_ok(ggml_type) || cols <= 0 || cols % blck_size(ggml_type)) return 0;
  return row_bytes(cols, ggml_type);
}

int64_t ktmi_q8_1_row_bytes(int64_t cols) { return cols > 0 ? q8_1_row_bytes(cols) : 0; }

int ktmi_quantize_q8_1(const void* x, int x_dtype, int64_t cols, int64_t tokens, void* out, void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(dtype_ok(x_dtype), KTMI_EINVAL, "quantize_q8_1: dtype %d", x_dtype);
  KTMI_REQUIRE(cols > 0 && tokens >= 0, KTMI_EINVAL, "quantize_q8_1: cols %lld tokens %lld", (long long)cols,
               (long long)tokens);
  KTMI_REQUIRE(tokens == 0 || (x && out && aligned(out, 4)), KTMI_EINVAL, "quantize_q8_1: null or misaligned pointer");
  return launch_quantize_q8_1(x, x_dtype, cols, tokens, (uint8_t*)out, (hipStream_t)stream);
}

int64_t ktmi_moe_a8_vec_workspace(int64_t cols, int64_t tokens) {
  if (cols <= 0 || tokens < 0) return 0;
  return q8_1_row_bytes(cols) * tokens;
}

int ktmi_moe_a8_vec(const void* X, int x_dtype, int64_t cols, const void* W, int w_is_table, const int32_t* ids,
                    int64_t top_k, int ggml_type, int64_t rows, int64_t tokens, int per_route, void* Y,
                    void* workspace, int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(type_ok(ggml_type), KTMI_ETYPE, "moe_a8_vec: ggml type %d has no kernel", ggml_type);
  KTMI_REQUIRE(dtype_ok(x_dtype), KTMI_EINVAL, "moe_a8_vec: dtype %d", x_dtype);
  KTMI_REQUIRE(cols > 0 && cols % blck_size(ggml_type) == 0, KTMI_EINVAL,
               "moe_a8_vec: cols %lld not a multiple of the block size %lld", (long long)cols,
               (long long)blck_size(ggml_type));
  KTMI_REQUIRE(rows > 0 && top_k > 0 && tokens >= 0, KTMI_EINVAL, "moe_a8_vec: rows %lld top_k %lld tokens %lld",
               (long long)rows, (long long)top_k, (long long)tokens);
  KTMI_REQUIRE(tokens * top_k <= 65535, KTMI_EINVAL, "moe_a8_vec: %lld routes (at most 65535 per call)",
               (long long)(tokens * top_k));
  if (tokens == 0) return KTMI_OK;
  const int64_t need = ktmi_moe_a8_vec_workspace(cols, tokens);
  KTMI_REQUIRE(workspace && ws_bytes >= need, KTMI_ESPACE, "moe_a8_vec: workspace %lld < %lld bytes",
               (long long)ws_bytes, (long long)need);
  KTMI_REQUIRE(X && W && ids && Y, KTMI_EINVAL, "moe_a8_vec: null pointer");
  KTMI_REQUIRE(aligned(W, 16) && aligned(workspace, 16), KTMI_EINVAL, "moe_a8_vec: W and workspace must be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  int rc = launch_quantize_q8_1(X, x_dtype, cols, tokens, (uint8_t*)workspace, s);
  if (rc) return rc;
  const int64_t rb = row_bytes(cols, ggml_type);
  return launch_moe_gemv((const uint8_t*)workspace, q8_1_row_bytes(cols), W, w_is_table, rows * rb, ids, top_k,
                         tokens * top_k, ggml_type, rows, cols, Y, x_dtype, per_route, 0x7FFFFFFF, s);
}

int ktmi_dequant_experts(const void* raw, int64_t raw_stride, int ggml_type, int64_t n, int64_t rows, int64_t cols,
                         void* out_bf16, int64_t out_stride, void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(type_ok(ggml_type), KTMI_ETYPE, "dequant: no GPU dequantizer for ggml type %d", ggml_type);
  KTMI_REQUIRE(n >= 0 && rows >= 0 && cols > 0 && cols % blck_size(ggml_type) == 0, KTMI_EINVAL,
               "dequant: n %lld rows %lld cols %lld (block %lld)", (long long)n, (long long)rows, (long long)cols,
               (long long)blck_size(ggml_type));
  KTMI_REQUIRE(n <= 65535, KTMI_EINVAL, "dequant: %lld experts per call (at most 65535)", (long long)n);
  if (n == 0 || rows == 0) return KTMI_OK;
  KTMI_REQUIRE(raw_stride >= rows * row_bytes(cols, ggml_type) && raw_stride % 2 == 0, KTMI_EINVAL,
               "dequant: raw_stride %lld (expert bytes %lld, must be even)", (long long)raw_stride,
               (long long)(rows * row_bytes(cols, ggml_type)));
  KTMI_REQUIRE(out_stride >= rows * cols && out_stride % 8 == 0, KTMI_EINVAL,
               "dequant: out_stride %lld must be >= rows*cols and a multiple of 8", (long long)out_stride);
  KTMI_REQUIRE(raw && out_bf16 && aligned(raw, 16) && aligned(out_bf16, 16), KTMI_EINVAL,
               "dequant: raw and out must be 16-byte aligned device pointers");
  KTMI_REQUIRE(ggml_type != GGML_Q4_K || raw_stride % 16 == 0, KTMI_EINVAL, "dequant: Q4_K raw_stride must be a multiple of 16");
  return launch_dequant((const uint8_t*)raw, raw_stride, ggml_type, n, rows, cols, (uint16_t*)out_bf16, out_stride,
                        (hipStream_t)stream);
}

int ktmi_hot_route(const int32_t* ids, int64_t n, const int32_t* log2slot, const int32_t* log2cpu, float* counts,
                   int32_t* slot_ids, int32_t* cpu_ids, void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(n >= 0, KTMI_EINVAL, "hot_route: n %lld", (long long)n);
  if (n == 0) return KTMI_OK;
  KTMI_REQUIRE(ids && log2slot && log2cpu && slot_ids && cpu_ids, KTMI_EINVAL, "hot_route: null pointer");
  return launch_route(ids, n, log2slot, log2cpu, counts, slot_ids, cpu_ids, (hipStream_t)stream);
}

int ktmi_silu_and_mul(const void* h, int dtype, int64_t R, int64_t N, void* out, void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(dtype_ok(dtype), KTMI_EINVAL, "silu_and_mul: dtype %d", dtype);
  KTMI_REQUIRE(R >= 0 && N > 0, KTMI_EINVAL, "silu_and_mul: R %lld N %lld", (long long)R, (long long)N);
  if (R == 0) return KTMI_OK;
  KTMI_REQUIRE(h && out, KTMI_EINVAL, "silu_and_mul: null pointer");
  return launch_silu_and_mul(h, dtype, R, N, out, (hipStream_t)stream);
}

int ktmi_combine(const void* out, int dtype, const float* w, int64_t T, int64_t top_k, int64_t K, void* res,
                 void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(dtype_ok(dtype), KTMI_EINVAL, "combine: dtype %d", dtype);
  KTMI_REQUIRE(T >= 0 && top_k > 0 && K > 0, KTMI_EINVAL, "combine: T %lld top_k %lld K %lld", (long long)T,
               (long long)top_k, (long long)K);
  if (T == 0) return KTMI_OK;
  KTMI_REQUIRE(out && w && res, KTMI_EINVAL, "combine: null pointer");
  return launch_combine(out, dtype, w, T, top_k, K, res, (hipStream_t)stream);
}

// ---- tokens sorted by expert and back

// the shape of a sort's or unsort's routes: the grids take a token a block, the places are int32
static int check_routes(const char* what, int dtype, int64_t cols, int64_t tokens, int64_t top_k) {
  KTMI_REQUIRE(dtype_ok(dtype), KTMI_EINVAL, "%s: dtype %d", what, dtype);
  KTMI_REQUIRE(cols > 0 && cols <= (1 << 24) && tokens >= 0 && top_k > 0, KTMI_EINVAL,
               "%s: cols %lld (at most 2^24) tokens %lld top_k %lld", what, (long long)cols, (long long)tokens,
               (long long)top_k);
  KTMI_REQUIRE(top_k <= 65535 && tokens <= 0x7FFFFFFF / top_k, KTMI_EINVAL,
               "%s: %lld tokens x top-%lld (at most 65535 a token, below 2^31 routes in all)", what, (long long)tokens,
               (long long)top_k);
  return KTMI_OK;
}

int64_t ktmi_moe_sort_workspace(int64_t tokens, int64_t top_k, int64_t n_experts) {
  if (tokens <= 0 || top_k <= 0 || n_experts <= 0 || tokens > 0x7FFFFFFF / top_k) return 0;
  return moe_sort_counts(tokens, top_k) * (n_experts + 1) * (int64_t)sizeof(int);
}

int ktmi_moe_sort(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const int32_t* ids, int64_t tokens,
                  int64_t top_k, int64_t n_experts, void* rows, int32_t* offsets, int32_t* perm, int32_t* pos,
                  void* workspace, int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  int rc = check_routes("moe_sort", x_dtype, cols, tokens, top_k);
  if (rc) return rc;
  KTMI_REQUIRE(n_experts > 0 && n_experts <= SORT_MAX_EXPERTS, KTMI_EINVAL, "moe_sort: %lld experts (1 to %lld)",
               (long long)n_experts, (long long)SORT_MAX_EXPERTS);
  KTMI_REQUIRE(offsets && (tokens == 0 || (ids && perm && pos && (!rows || x))), KTMI_EINVAL, "moe_sort: null pointer");
  const int es = x_dtype == KTMI_F32 ? 4 : 2;
  KTMI_REQUIRE(aligned(x, es) && aligned(rows, es), KTMI_EINVAL, "moe_sort: x and rows must be aligned to their type");
  KTMI_REQUIRE(!rows || x_stride >= cols || tokens <= 1, KTMI_EINVAL, "moe_sort: x_stride %lld below cols %lld",
               (long long)x_stride, (long long)cols);
  const int64_t need = ktmi_moe_sort_workspace(tokens, top_k, n_experts);
  KTMI_REQUIRE(need == 0 || (workspace && ws_bytes >= need && aligned(workspace, 4)), KTMI_ESPACE,
               "moe_sort: workspace %lld < %lld bytes", (long long)ws_bytes, (long long)need);
  return launch_moe_sort((const uint8_t*)x, es, x_stride, cols, ids, tokens, top_k, n_experts, (uint8_t*)rows, offsets,
                         perm, pos, (int*)workspace, (hipStream_t)stream);
}

int ktmi_moe_unsort(const void* rows, int dtype, int64_t row_stride, int64_t cols, const float* w, const int32_t* pos,
                    int64_t tokens, int64_t top_k, void* y, void* stream) {
  g_err[0] = 0;
  int rc = check_routes("moe_unsort", dtype, cols, tokens, top_k);
  if (rc) return rc;
  if (tokens == 0) return KTMI_OK;
  const int es = dtype == KTMI_F32 ? 4 : 2;
  KTMI_REQUIRE(rows && pos && y && aligned(rows, es) && aligned(y, es), KTMI_EINVAL,
               "moe_unsort: null pointer, or one not aligned to its type");
  KTMI_REQUIRE(row_stride >= cols || tokens * top_k <= 1, KTMI_EINVAL, "moe_unsort: row_stride %lld below cols %lld",
               (long long)row_stride, (long long)cols);
  return launch_moe_unsort(rows, dtype, row_stride, cols, w, pos, tokens, top_k, y, (hipStream_t)stream);
}

int ktmi_moe_unsort_grad(const void* dy, int64_t dy_stride, const void* rows, int64_t row_stride, int dtype,
                         int64_t cols, const float* w, const int32_t* pos, int64_t tokens, int64_t top_k, void* drows,
                         float* dw, void* stream) {
  g_err[0] = 0;
  int rc = check_routes("moe_unsort_grad", dtype, cols, tokens, top_k);
  if (rc) return rc;
  if (tokens == 0 || (!drows && !dw)) return KTMI_OK;
  const int es = dtype == KTMI_F32 ? 4 : 2;
  KTMI_REQUIRE(dy && pos && (!dw || rows) && aligned(dy, es) && aligned(rows, es) && aligned(drows, es), KTMI_EINVAL,
               "moe_unsort_grad: null pointer, or one not aligned to its type");
  KTMI_REQUIRE(dy_stride >= cols || tokens <= 1, KTMI_EINVAL, "moe_unsort_grad: dy_stride %lld below cols %lld",
               (long long)dy_stride, (long long)cols);
  KTMI_REQUIRE(!dw || row_stride >= cols || tokens * top_k <= 1, KTMI_EINVAL,
               "moe_unsort_grad: row_stride %lld below cols %lld", (long long)row_stride, (long long)cols);
  return launch_moe_unsort_grad(dy, dy_stride, rows, row_stride, dtype, cols, w, pos, tokens, top_k, drows, dw,
                                (hipStream_t)stream);
}

// ---- products with 4-bit weights

// n: rows of x, routes: rows of y
static int check_w4(const char* what, const W4Args& a, int64_t n) {
  KTMI_REQUIRE(dtype_ok(a.x_dtype) && dtype_ok(a.scale_dtype), KTMI_EINVAL, "%s: x dtype %d scale dtype %d", what,
               a.x_dtype, a.scale_dtype);
  KTMI_REQUIRE(a.cols > 0 && a.cols <= (1 << 24) && a.rows > 0 && a.rows <= (1 << 24), KTMI_EINVAL,
               "%s: cols %lld rows %lld (1 to 2^24)", what, (long long)a.cols, (long long)a.rows);
  KTMI_REQUIRE(a.n_experts > 0 && a.n_experts <= SORT_MAX_EXPERTS, KTMI_EINVAL, "%s: %lld experts (1 to %lld)", what,
               (long long)a.n_experts, (long long)SORT_MAX_EXPERTS);
  KTMI_REQUIRE(a.group == 32 || a.group == 64 || (a.group > 0 && (a.group % 128 == 0 || a.group >= a.cols)), KTMI_EINVAL,
               "%s: group %lld (32, 64, a multiple of 128, or at least cols)", what, (long long)a.group);
  KTMI_REQUIRE(n >= 0 && a.top_k > 0 && a.n_routes >= 0, KTMI_EINVAL, "%s: %lld rows of x, top_k %lld", what, (long long)n,
               (long long)a.top_k);
  KTMI_REQUIRE(a.n_routes <= W4_ROUTES, KTMI_EINVAL, "%s: %lld rows of y (at most 2^23)", what, (long long)a.n_routes);
  if (a.n_routes == 0) return KTMI_OK;
  const int es = a.x_dtype == KTMI_F32 ? 4 : 2, ss = a.scale_dtype == KTMI_F32 ? 4 : 2;
  KTMI_REQUIRE(a.x && a.codes && a.scales && a.y, KTMI_EINVAL, "%s: null pointer", what);
  KTMI_REQUIRE(aligned(a.x, es) && aligned(a.y, es) && aligned(a.scales, ss), KTMI_EINVAL,
               "%s: x, y and scales must be aligned to their types", what);
  KTMI_REQUIRE(a.x_stride >= a.cols || n <= 1, KTMI_EINVAL, "%s: x_stride %lld below cols %lld", what, (long long)a.x_stride,
               (long long)a.cols);
  return KTMI_OK;
}

int ktmi_w4_vec(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const void* codes, const void* scales,
                int scale_dtype, const void* zeros, int64_t group, int64_t rows, int64_t tokens, void* y, void* stream) {
  g_err[0] = 0;
  const W4Args a = {x, x_stride, cols, (const uint8_t*)codes, scales, (const uint8_t*)zeros, group, rows, 1, nullptr, nullptr,
                    1, tokens, y, nullptr, x_dtype, scale_dtype, nullptr};
  int rc = check_w4("w4_vec", a, tokens);
  if (rc || tokens == 0) return rc;
  return launch_w4(a, (hipStream_t)stream);
}

int64_t ktmi_moe_w4_vec_workspace(int64_t tokens, int64_t top_k, int64_t n_experts) {
  if (tokens <= 0 || top_k <= 0 || n_experts <= 0 || tokens > 0x7FFFFFFF / top_k) return 0;
  return w4_workspace(tokens, top_k, n_experts);
}

int ktmi_moe_w4_vec(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const void* codes, const void* scales,
                    int scale_dtype, const void* zeros, int64_t group, int64_t rows, int64_t n_experts,
                    const int32_t* ids, int64_t top_k, int64_t tokens, void* y, void* workspace, int64_t ws_bytes,
                    void* stream) {
  g_err[0] = 0;
  KTMI_REQUIRE(tokens >= 0 && top_k > 0 && top_k <= 65535 && tokens <= 0x7FFFFFFF / top_k, KTMI_EINVAL,
               "moe_w4_vec: %lld tokens x top-%lld (at most 65535 a token, 2^31 in all)", (long long)tokens, (long long)top_k);
  const W4Args a = {x, x_stride, cols, (const uint8_t*)codes, scales, (const uint8_t*)zeros, group, rows, n_experts, ids,
                    nullptr, top_k, tokens * top_k, y, (uint8_t*)workspace, x_dtype, scale_dtype, nullptr};
  int rc = check_w4("moe_w4_vec", a, tokens);
  if (rc || tokens == 0) return rc;
  KTMI_REQUIRE(ids, KTMI_EINVAL, "moe_w4_vec: null pointer");
  const int64_t need = w4_workspace(tokens, top_k, n_experts);
  KTMI_REQUIRE(need == 0 || (workspace && ws_bytes >= need && aligned(workspace, 16)), KTMI_ESPACE,
               "moe_w4_vec: workspace %lld < %lld bytes", (long long)ws_bytes, (long long)need);
  return launch_w4(a, (hipStream_t)stream);
}

int ktmi_moe_w4_sorted(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const void* codes,
                       const void* scales, int scale_dtype, const void* zeros, int64_t group, int64_t rows,
                       int64_t n_experts, const int32_t* offsets, int64_t n_rows, void* y, void* stream) {
  g_err[0] = 0;
  const W4Args a = {x, x_stride, cols, (const uint8_t*)codes, scales, (const uint8_t*)zeros, group, rows, n_experts, nullptr,
                    offsets, 1, n_rows, y, nullptr, x_dtype, scale_dtype, nullptr};
  int rc = check_w4("moe_w4_sorted", a, n_rows);
  if (rc || n_rows == 0) return rc;
  KTMI_REQUIRE(offsets, KTMI_EINVAL, "moe_w4_sorted: null pointer");
  return launch_w4(a, (hipStream_t)stream);
}

int ktmi_w4_kernel_of(int by, int x_dtype, int64_t cols, int64_t group, int64_t rows, int64_t n_experts, int64_t n_rows,
                      ktmi_w4_kernel* kernel) {
  g_err[0] = 0;
  KTMI_REQUIRE(by >= KTMI_W4_DENSE && by <= KTMI_W4_SORTED && kernel && n_rows > 0, KTMI_EINVAL,
               "w4_kernel_of: by %d, %lld rows, or a null pointer", by, (long long)n_rows);
  static const int32_t named = 0;  // stands in for the tensors, which the choice does not read
  const W4Args a = {&named, cols, cols, (const uint8_t*)&named, &named, nullptr, group, rows, by == KTMI_W4_DENSE ? 1 : n_experts,
                    by == KTMI_W4_IDS ? &named : nullptr, by == KTMI_W4_SORTED ? &named : nullptr, 1, n_rows, (void*)&named,
                    (uint8_t*)&named, x_dtype, KTMI_F32, nullptr};
  int rc = check_w4("w4_kernel_of", a, n_rows);
  return rc ? rc : launch_w4(a, nullptr, kernel);
}

// ---- products in 8-bit floating point

static constexpr int64_t MAX_ROWS = 0x7fffff00;  // of x or y: 31 bits hold a row past the last tile's

static int check_fp8(const char* what, const Fp8Args& a, int64_t need, int64_t ws_bytes) {
  KTMI_REQUIRE(dtype_ok(a.dtype), KTMI_EINVAL, "%s: x dtype %d", what, a.dtype);
  KTMI_REQUIRE(a.cols > 0 && a.cols <= (1 << 24) && a.rows > 0 && a.rows <= (1 << 24), KTMI_EINVAL,
               "%s: cols %lld rows %lld (1 to 2^24)", what, (long long)a.cols, (long long)a.rows);
  KTMI_REQUIRE(a.n_experts > 0 && a.n_experts <= SORT_MAX_EXPERTS, KTMI_EINVAL, "%s: %lld experts (1 to %lld)", what,
               (long long)a.n_experts, (long long)SORT_MAX_EXPERTS);
  KTMI_REQUIRE(a.x_rows >= 0 && a.top_k > 0 && a.top_k <= 65535 && a.x_rows <= MAX_ROWS / a.top_k, KTMI_EINVAL,
               "%s: %lld rows of x, top_k %lld (at most 65535, and %lld rows of y)", what, (long long)a.x_rows,
               (long long)a.top_k, (long long)MAX_ROWS);
  if (a.x_rows == 0) return KTMI_OK;
  const int es = a.dtype == KTMI_F32 ? 4 : 2;
  KTMI_REQUIRE(a.x && a.w && a.scales && a.y, KTMI_EINVAL, "%s: null pointer", what);
  KTMI_REQUIRE(aligned(a.x, es) && aligned(a.y, es) && aligned(a.scales, 4), KTMI_EINVAL,
               "%s: x, y and scales must be aligned to their types", what);
  KTMI_REQUIRE(a.x_stride >= a.cols || a.x_rows <= 1, KTMI_EINVAL, "%s: x_stride %lld below cols %lld", what,
               (long long)a.x_stride, (long long)a.cols);
  KTMI_REQUIRE(need == 0 || (a.ws && ws_bytes >= need && aligned(a.ws, 16)), KTMI_ESPACE,
               "%s: workspace %lld < %lld bytes, or not aligned to 16", what, (long long)ws_bytes, (long long)need);
  return KTMI_OK;
}

static bool fp8_shape(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k) {
  return rows > 0 && rows <= (1 << 24) && cols > 0 && cols <= (1 << 24) && x_rows > 0 && n_experts > 0 && n_experts <= SORT_MAX_EXPERTS && top_k > 0 &&
         top_k <= 65535 && x_rows <= MAX_ROWS / top_k;
}

int64_t ktmi_fp8_linear_workspace(int64_t rows, int64_t cols, int64_t tokens) {
  return fp8_shape(rows, cols, tokens, 1, 1) ? fp8_workspace(rows, cols, tokens, 1, 1, false) : 0;
}

int ktmi_fp8_linear(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const void* w, const float* scales,
                    int64_t rows, int64_t tokens, void* y, void* workspace, int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  const Fp8Args a = {x_dtype, x, x_stride, tokens, (const uint8_t*)w, scales, rows, cols, 1, nullptr, 1, nullptr, y,
                     (uint8_t*)workspace};
  int rc = check_fp8("fp8_linear", a, ktmi_fp8_linear_workspace(rows, cols, tokens), ws_bytes);
  return rc || tokens == 0 ? rc : launch_fp8(a, (hipStream_t)stream);
}

int64_t ktmi_moe_fp8_vec_workspace(int64_t rows, int64_t cols, int64_t tokens, int64_t top_k, int64_t n_experts) {
  return fp8_shape(rows, cols, tokens, n_experts, top_k) ? fp8_workspace(rows, cols, tokens, n_experts, top_k, true) : 0;
}

int ktmi_moe_fp8_vec(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const void* w, const float* scales,
                     int64_t rows, int64_t n_experts, const int32_t* ids, int64_t top_k, int64_t tokens, void* y,
                     void* workspace, int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  const Fp8Args a = {x_dtype, x, x_stride, tokens, (const uint8_t*)w, scales, rows, cols, n_experts, ids, top_k, nullptr, y,
                     (uint8_t*)workspace};
  int rc = check_fp8("moe_fp8_vec", a, ktmi_moe_fp8_vec_workspace(rows, cols, tokens, top_k, n_experts), ws_bytes);
  if (rc || tokens == 0) return rc;
  KTMI_REQUIRE(ids, KTMI_EINVAL, "moe_fp8_vec: null pointer");
  return launch_fp8(a, (hipStream_t)stream);
}

int64_t ktmi_moe_fp8_sorted_workspace(int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows) {
  return fp8_shape(rows, cols, n_rows, n_experts, 1) ? fp8_workspace(rows, cols, n_rows, n_experts, 1, false) : 0;
}

int ktmi_moe_fp8_sorted(const void* x, int x_dtype, int64_t x_stride, int64_t cols, const void* w, const float* scales,
                        int64_t rows, int64_t n_experts, const int32_t* offsets, int64_t n_rows, void* y, void* workspace,
                        int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  const Fp8Args a = {x_dtype, x, x_stride, n_rows, (const uint8_t*)w, scales, rows, cols, n_experts, nullptr, 1, offsets, y,
                     (uint8_t*)workspace};
  int rc = check_fp8("moe_fp8_sorted", a, ktmi_moe_fp8_sorted_workspace(rows, cols, n_experts, n_rows), ws_bytes);
  if (rc || n_rows == 0) return rc;
  KTMI_REQUIRE(offsets, KTMI_EINVAL, "moe_fp8_sorted: null pointer");
  return launch_fp8(a, (hipStream_t)stream);
}

int ktmi_fp8_kernel_of(int routed, int64_t rows, int64_t cols, int64_t n_experts, int64_t top_k, int64_t x_rows,
                       ktmi_prod_kernel* kernel) {
  g_err[0] = 0;
  KTMI_REQUIRE(fp8_shape(rows, cols, x_rows, n_experts, top_k) && kernel, KTMI_EINVAL, "fp8_kernel_of: a shape, or a null pointer");
  *kernel = fp8_kernel_of(rows, cols, x_rows, n_experts, top_k, routed != 0);
  return KTMI_OK;
}

// ---- gated and linear products with gradients

static int check_prod(const char* what, const ProdArgs& a) {
  KTMI_REQUIRE(dtype_ok(a.dtype), KTMI_EINVAL, "%s: dtype %d", what, a.dtype);
  KTMI_REQUIRE(a.cols > 0 && a.cols <= (1 << 24) && a.rows > 0 && a.rows <= (1 << 24), KTMI_EINVAL,
               "%s: cols %lld rows %lld (1 to 2^24)", what, (long long)a.cols, (long long)a.rows);
  KTMI_REQUIRE(a.n_experts > 0 && a.n_experts <= SORT_MAX_EXPERTS && (a.offsets || a.n_experts == 1), KTMI_EINVAL,
               "%s: %lld experts (1 to %lld; without offsets 1)", what, (long long)a.n_experts, (long long)SORT_MAX_EXPERTS);
  KTMI_REQUIRE(a.n_rows >= 0 && a.n_rows <= MAX_ROWS, KTMI_EINVAL, "%s: %lld rows (at most %lld)", what, (long long)a.n_rows,
               (long long)MAX_ROWS);
  const int es = a.dtype == KTMI_F32 ? 4 : 2;
  KTMI_REQUIRE(aligned(a.x, es) && aligned(a.dy, es) && aligned(a.w, es) && aligned(a.y, es) && aligned(a.sums, 16), KTMI_EINVAL,
               "%s: tensors must be aligned to their types, sums to 16 bytes", what);
  return KTMI_OK;
}

static int check_stride(const char* what, const char* name, int64_t stride, int64_t width, int64_t rows) {
  KTMI_REQUIRE(stride >= width || rows <= 1, KTMI_EINVAL, "%s: %s %lld below the row's %lld", what, name, (long long)stride,
               (long long)width);
  return KTMI_OK;
}

int64_t ktmi_linear_workspace(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows) {
  if (what < KTMI_PROD_GATED || what > KTMI_PROD_GRAD_W || !dtype_ok(dtype) || rows <= 0 || rows > (1 << 24) || cols <= 0 ||
      cols > (1 << 24) || n_experts <= 0 || n_experts > SORT_MAX_EXPERTS || n_rows <= 0 || n_rows > MAX_ROWS)
    return 0;
  return prod_workspace(what, dtype, rows, cols, n_experts, n_rows);
}

int ktmi_linear_kernel_of(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows,
                          ktmi_prod_kernel* kernel) {
  g_err[0] = 0;
  KTMI_REQUIRE(what >= KTMI_PROD_GATED && what <= KTMI_PROD_GRAD_W && dtype_ok(dtype) && rows > 0 && rows <= (1 << 24) && cols > 0 &&
                   cols <= (1 << 24) && n_experts > 0 && n_experts <= SORT_MAX_EXPERTS && n_rows > 0 && n_rows <= MAX_ROWS && kernel,
               KTMI_EINVAL, "linear_kernel_of: a shape, or a null pointer");
  *kernel = prod_kernel_of(what, dtype, rows, cols, n_experts, n_rows);
  return KTMI_OK;
}

// the call's workspace is there; then it runs
static int run_prod(const char* name, int what, const ProdArgs& a, int64_t ws_bytes, void* stream) {
  const int64_t need = ktmi_linear_workspace(what, a.dtype, a.rows, a.cols, a.n_experts, a.n_rows);
  KTMI_REQUIRE(need == 0 || (a.part && ws_bytes >= need && aligned(a.part, 16)), KTMI_ESPACE,
               "%s: workspace %lld < %lld bytes, or not aligned to 16", name, (long long)ws_bytes, (long long)need);
  return launch_prod(what, a, (hipStream_t)stream);
}

static int check_act(const char* what, int act) {
  KTMI_REQUIRE(act == KTMI_ACT_SILU || act == KTMI_ACT_GELU_TANH, KTMI_EINVAL, "%s: act %d", what, act);
  return KTMI_OK;
}

int ktmi_gated(const void* x, int dtype, int64_t x_stride, int64_t cols, const void* w13, int64_t inter, int64_t n_experts,
               const int32_t* offsets, int64_t n_rows, int act, void* h, float* sums, void* workspace, int64_t ws_bytes,
               void* stream) {
  g_err[0] = 0;
  const ProdArgs a = {dtype, x, x_stride, nullptr, 0, w13, inter, cols, n_experts, offsets, n_rows, act, h, sums, (float*)workspace};
  int rc = check_prod("gated", a);
  if (!rc) rc = check_act("gated", act);
  if (!rc) rc = check_stride("gated", "x_stride", x_stride, cols, n_rows);
  KTMI_REQUIRE(rc || inter <= (1 << 23), KTMI_EINVAL, "gated: inter %lld (at most 2^23)", (long long)inter);
  if (rc || n_rows == 0) return rc;
  KTMI_REQUIRE(x && w13 && h, KTMI_EINVAL, "gated: null pointer");
  return run_prod("gated", KTMI_PROD_GATED, a, ws_bytes, stream);
}

int ktmi_gated_grad(const float* sums, const void* dh, int dtype, int64_t dh_stride, int64_t inter, int64_t n_rows, int act,
                    void* dsums, void* stream) {
  g_err[0] = 0;
  const ProdArgs a = {dtype, nullptr, 0, dh, dh_stride, nullptr, inter, 1, 1, nullptr, n_rows, act, dsums, (float*)sums,
                      nullptr};
  int rc = check_prod("gated_grad", a);
  if (!rc) rc = check_act("gated_grad", act);
  if (!rc) rc = check_stride("gated_grad", "dh_stride", dh_stride, inter, n_rows);
  KTMI_REQUIRE(rc || inter <= (1 << 23), KTMI_EINVAL, "gated_grad: inter %lld (at most 2^23)", (long long)inter);
  if (rc || n_rows == 0) return rc;
  KTMI_REQUIRE(sums && dh && dsums, KTMI_EINVAL, "gated_grad: null pointer");
  return launch_gated_grad(sums, dh, dtype, dh_stride, inter, n_rows, act, dsums, (hipStream_t)stream);
}

int ktmi_linear(const void* x, int dtype, int64_t x_stride, int64_t cols, const void* w, int64_t rows, int64_t n_experts,
                const int32_t* offsets, int64_t n_rows, void* y, void* workspace, int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  const ProdArgs a = {dtype, x, x_stride, nullptr, 0, w, rows, cols, n_experts, offsets, n_rows, 0, y, nullptr,
                      (float*)workspace};
  int rc = check_prod("linear", a);
  if (!rc) rc = check_stride("linear", "x_stride", x_stride, cols, n_rows);
  if (rc || n_rows == 0) return rc;
  KTMI_REQUIRE(x && w && y, KTMI_EINVAL, "linear: null pointer");
  return run_prod("linear", KTMI_PROD_LINEAR, a, ws_bytes, stream);
}

int ktmi_linear_grad_x(const void* dy, int dtype, int64_t dy_stride, int64_t rows, const void* w, int64_t cols,
                       int64_t n_experts, const int32_t* offsets, int64_t n_rows, void* dx, void* workspace, int64_t ws_bytes,
                       void* stream) {
  g_err[0] = 0;
  const ProdArgs a = {dtype, nullptr, 0, dy, dy_stride, w, rows, cols, n_experts, offsets, n_rows, 0, dx, nullptr,
                      (float*)workspace};
  int rc = check_prod("linear_grad_x", a);
  if (!rc) rc = check_stride("linear_grad_x", "dy_stride", dy_stride, rows, n_rows);
  if (rc || n_rows == 0) return rc;
  KTMI_REQUIRE(dy && w && dx, KTMI_EINVAL, "linear_grad_x: null pointer");
  return run_prod("linear_grad_x", KTMI_PROD_GRAD_X, a, ws_bytes, stream);
}

int ktmi_linear_grad_w(const void* dy, int dtype, int64_t dy_stride, int64_t rows, const void* x, int64_t x_stride,
                       int64_t cols, int64_t n_experts, const int32_t* offsets, int64_t n_rows, void* dw, void* workspace,
                       int64_t ws_bytes, void* stream) {
  g_err[0] = 0;
  const ProdArgs a = {dtype, x, x_stride, dy, dy_stride, nullptr, rows, cols, n_experts, offsets, n_rows, 0, dw, nullptr,
                      (float*)workspace};
  int rc = check_prod("linear_grad_w", a);
  if (!rc) rc = check_stride("linear_grad_w", "dy_stride", dy_stride, rows, n_rows);
  if (!rc) rc = check_stride("linear_grad_w", "x_stride", x_stride, cols, n_rows);
  if (rc) return rc;
  KTMI_REQUIRE(dw && (n_rows == 0 || (dy && x)), KTMI_EINVAL, "linear_grad_w: null pointer");
  return run_prod("linear_grad_w", KTMI_PROD_GRAD_W, a, ws_bytes, stream);
}

// ---- scratch for ktmi_moe_layer_noalloc
// A file-scope device array that stands in for the caller's workspace. In host code its
// name is a host-side stand-in, not a device address: the address on each device comes
// from hipGetSymbolAddress, taken once per device with that device current, and only that
// address is ever handed to kernels. Each GPU holds its own copy until the process ends.
static __device__ __align__(256) uint8_t scratch[KTMI_NOALLOC_SCRATCH_BYTES];
static constexpr int kMaxDevices = 64;
static std::mutex g_scratch_mu;
static void* g_scratch_ptr[kMaxDevices] = {};

static int scratch_of_current_device(void** out) {
  int dev = 0;
  KTMI_HIP_TRY(hipGetDevice(&dev));
  KTMI_REQUIRE(dev >= 0 && dev < kMaxDevices, KTMI_EINVAL, "moe_layer_noalloc: device %d (at most %d)", dev,
               kMaxDevices);
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    KTMI_HIP_TRY(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
    KTMI_REQUIRE(p != nullptr, KTMI_EHIP, "moe_layer_noalloc: no device address for the scratch array on device %d",
                 dev);
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return KTMI_OK;
}

// Below 64 routes the GEMV mode's two launches keep the reference kernels' int8 numerics at about
// the decode mode's speed or better (graph-replayed 2048 x 512 layers with 32 hot slots, us a layer
// GEMV / decode: Q4_K 12.7 / 13.9 at 8 routes, 19.9 / 19.1 at 32, 24.6 / 21.3 at 48; Q8_0 15.1 /
// 17.2, 22.7 / 24.1, 28.1 / 27.6); from 64 routes the decode mode's MFMAs win (Q4_K 27.7 / 22.4 at
// 64, 38.4 / 25.8 at 128; Q8_0 29.8 / 29.0, 39.2 / 34.7).
// Where the rows are too long for those two launches, the decode mode starts at one route: its
// alternative is the stage-by-stage GEMV (7168 x 2048 Q4_K/Q6_K, 7 tokens: 164 against 60 us).
// With hardly a route a slot on long rows of Q8_0 both are bound by the weights' bytes, which the
// GEMV's loads bring at 6.9 TB/s and the decode mode's ring at 5.3: there the GEMV stays (2048 x 512,
// 128 slots all hot, 16 tokens 62 against 75 us; 256 slots, 32 tokens 104 against 147; 1024 rows of
// Q4_K down, 128 slots, 24 tokens 118 against 148), up to a mean of one route a slot at 512 rows:
// past it (42 against 50 us at 128 routes on 72 slots, equal at 4 routes a slot) the decode mode has the
// smaller error, 0.005 against 0.0125 (relative, against 64 bits).
constexpr int64_t kDecodeMinRoutes = 64;

int ktmi_moe_layer_mode(const ktmi_layer* L, int64_t tokens, int64_t top_k) {
  if (tokens * top_k > kGemvMaxRoutes) return KTMI_MODE_GROUPED;
  if (!L || !decode_mfma_fits(L, tokens, top_k)) return KTMI_MODE_GEMV;
  if (!decode_layer_fits(L, tokens, top_k)) return KTMI_MODE_DECODE;
  const int64_t R = tokens * top_k;
  const bool few = L->type13 == GGML_Q8_0 && L->hidden > 1024 && 512 * R <= L->inter * L->n_slots;
  return R >= kDecodeMinRoutes && !few ? KTMI_MODE_DECODE : KTMI_MODE_GEMV;
}

static int64_t gemv_layer_workspace(const ktmi_layer* L, int64_t tokens, int64_t top_k) {
  // q8_1(x) | h13 bf16 [R, 2N] | h bf16 [R, N] | q8_1(h) | out bf16 [R, K]
  const int64_t R = tokens * top_k;
  auto al = [](int64_t v) { return (v + 255) & ~(int64_t)255; };
  return al(q8_1_row_bytes(L->hidden) * tokens) + al(R * 2 * L->inter * 2) + al(R * L->inter * 2) +
         al(q8_1_row_bytes(L->inter) * R) + al(R * L->hidden * 2);
}

static int check_layer(const ktmi_layer* L) {
  KTMI_REQUIRE(L, KTMI_EINVAL, "moe_layer: null layer");
  KTMI_REQUIRE(type_ok(L->type13) && type_ok(L->type2), KTMI_ETYPE, "moe_layer: ggml types %d/%d", L->type13, L->type2);
  KTMI_REQUIRE(L->hidden > 0 && L->inter > 0 && L->n_slots > 0, KTMI_EINVAL, "moe_layer: hidden %lld inter %lld slots %lld",
               (long long)L->hidden, (long long)L->inter, (long long)L->n_slots);
  KTMI_REQUIRE(L->hidden % blck_size(L->type13) == 0 && L->inter % blck_size(L->type2) == 0, KTMI_EINVAL,
               "moe_layer: hidden %lld / inter %lld not multiples of the block sizes", (long long)L->hidden,
               (long long)L->inter);
  KTMI_REQUIRE(L->w13 && L->w2 && aligned(L->w13, 16) && aligned(L->w2, 16), KTMI_EINVAL,
               "moe_layer: weights must be 16-byte aligned device pointers");
  return KTMI_OK;
}

// Tokens per pass of the grouped mode. Its kernels address x [T, K], H [R, N] and Y [R, K]
// (bf16, R = T top_k) with 32-bit buffer offsets, and an offset at 0xFFFFFFF0 marks a store
// to drop; a pass keeps every one of them under 4 GiB - 64 KiB. A token's output depends only
// on its own routes, so a longer layer runs as consecutive passes over token slices, each
// with the whole workspace.
static int64_t grouped_pass_tokens(const ktmi_layer* L, int64_t top_k) {
  const int64_t limit = 0xFFFF0000ll;
  const int64_t per_token = 2 * top_k * (L->hidden > L->inter ? L->hidden : L->inter);
  const int64_t t = limit / per_token;
  return t >= 256 ? t / 256 * 256 : (t > 0 ? t : 1);
}

int64_t ktmi_moe_layer_pass_tokens(const ktmi_layer* L, int64_t top_k) {
  if (!L || top_k <= 0 || L->hidden <= 0 || L->inter <= 0) return 0;
  return grouped_pass_tokens(L, top_k);
}

int64_t ktmi_moe_layer_workspace(const ktmi_layer* L, int64_t tokens, int64_t top_k, int mode) {
  if (!L || tokens < 0 || top_k <= 0) return 0;
  if (mode == KTMI_MODE_AUTO) mode = ktmi_moe_layer_mode(L, tokens, top_k);
  if (mode == KTMI_MODE_DECODE) return decode_mfma_fits(L, tokens, top_k) ? decode_mfma_workspace(L, tokens, top_k) : 0;
  if (mode == KTMI_MODE_GEMV)
    return decode_layer_fits(L, tokens, top_k) ? decode_layer_workspace(L, tokens, top_k)
                                               : gemv_layer_workspace(L, tokens, top_k);
  const int64_t pass = grouped_pass_tokens(L, top_k);
  return grouped_plan(tokens < pass ? tokens : pass, top_k, L->n_slots, L->hidden, L->inter).total;
}

int ktmi_moe_layer(const ktmi_layer* L, const void* x, const float* topk_w, const int32_t* slot_ids, int64_t tokens,
                   int64_t top_k, void* y, void* workspace, int64_t ws_bytes, int mode, void* stream) {
  g_err[0] = 0;
  int rc = check_layer(L);
  if (rc) return rc;
  KTMI_REQUIRE(tokens >= 0 && top_k > 0, KTMI_EINVAL, "moe_layer: tokens %lld top_k %lld", (long long)tokens,
               (long long)top_k);
  if (tokens == 0) return KTMI_OK;
  KTMI_REQUIRE(x && topk_w && slot_ids && y && workspace, KTMI_EINVAL, "moe_layer: null pointer");
  KTMI_REQUIRE(aligned(x, 16) && aligned(y, 16) && aligned(workspace, 256), KTMI_EINVAL,
               "moe_layer: x, y 16-byte and workspace 256-byte aligned");
  if (mode == KTMI_MODE_AUTO) mode = ktmi_moe_layer_mode(L, tokens, top_k);
  const int64_t need = ktmi_moe_layer_workspace(L, tokens, top_k, mode);
  KTMI_REQUIRE(ws_bytes >= need, KTMI_ESPACE, "moe_layer: workspace %lld < %lld bytes", (long long)ws_bytes,
               (long long)need);
  hipStream_t s = (hipStream_t)stream;
  const int64_t R = tokens * top_k;
  const int64_t K = L->hidden, N = L->inter;
  if (mode == KTMI_MODE_DECODE) {
    KTMI_REQUIRE(decode_mfma_fits(L, tokens, top_k), KTMI_EINVAL,
                 "moe_layer: the decode mode takes at most %d routes of %d tokens, at most 512 slots, hidden and "
                 "intermediate sizes that are multiples of 256, and slot matrices under 4 GiB",
                 DM_MAX_ROUTES, DM_MAX_TOKENS);
    return launch_decode_mfma(L, (const uint16_t*)x, topk_w, slot_ids, tokens, top_k, (uint16_t*)y, (uint8_t*)workspace,
                              s);
  }
  if (mode == KTMI_MODE_GEMV && decode_layer_fits(L, tokens, top_k))
    return launch_decode_layer(L, (const uint16_t*)x, topk_w, slot_ids, tokens, top_k, (uint16_t*)y,
                               (uint8_t*)workspace, s);
  if (mode == KTMI_MODE_GEMV) {
    KTMI_REQUIRE(R <= 65535, KTMI_EINVAL, "moe_layer: GEMV mode takes at most 65535 routes");
    auto al = [](int64_t v) { return (v + 255) & ~(int64_t)255; };
    uint8_t* p = (uint8_t*)workspace;
    uint8_t* xq = p; p += al(q8_1_row_bytes(K) * tokens);
    uint16_t* h13 = (uint16_t*)p; p += al(R * 2 * N * 2);
    uint16_t* h = (uint16_t*)p; p += al(R * N * 2);
    uint8_t* hq = p; p += al(q8_1_row_bytes(N) * R);
    uint16_t* out = (uint16_t*)p;
    // the slot ids are the per-route expert ids of the GEMV (cold = -1)
    record_stage(0, s);
    rc = launch_quantize_q8_1(x, KTMI_BF16, K, tokens, xq, s);
    if (rc) return rc;
    record_stage(1, s);
    rc = launch_moe_gemv(xq, q8_1_row_bytes(K), L->w13, L->w_is_table, 2 * N * row_bytes(K, L->type13), slot_ids,
                         top_k, R, L->type13, 2 * N, K, h13, KTMI_BF16, 0, (int)L->n_slots, s);
    if (rc) return rc;
    record_stage(2, s);
    rc = launch_silu_and_mul(h13, KTMI_BF16, R, N, h, s);
    if (rc) return rc;
    rc = launch_quantize_q8_1(h, KTMI_BF16, N, R, hq, s);
    if (rc) return rc;
    record_stage(3, s);
    rc = launch_moe_gemv(hq, q8_1_row_bytes(N), L->w2, L->w_is_table, K * row_bytes(N, L->type2), slot_ids, 1, R,
                         L->type2, K, N, out, KTMI_BF16, 0, (int)L->n_slots, s);
    if (rc) return rc;
    record_stage(4, s);
    rc = launch_combine(out, KTMI_BF16, topk_w, tokens, top_k, K, y, s);
    record_stage(5, s);
    return rc;
  }
  KTMI_REQUIRE(mode == KTMI_MODE_GROUPED, KTMI_EINVAL, "moe_layer: mode %d", mode);
  const int64_t pass = grouped_pass_tokens(L, top_k);
  const bool window = tokens <= pass && window_fits(L, tokens, top_k);
  for (int64_t t0 = 0; t0 < tokens; t0 += pass) {
    const int64_t nt = tokens - t0 < pass ? tokens - t0 : pass;
    const GroupedPlan P = grouped_plan(nt, top_k, L->n_slots, K, N);
    rc = launch_grouped_layer(L, (const uint16_t*)x + t0 * K, topk_w + t0 * top_k, slot_ids + t0 * top_k, nt, top_k,
                              (uint16_t*)y + t0 * K, (uint8_t*)workspace, P, window, s);
    if (rc) return rc;
  }
  return KTMI_OK;
}

int ktmi_moe_layer_noalloc(const ktmi_layer* L, const void* x, const float* topk_w, const int32_t* slot_ids,
                           int64_t tokens, int64_t top_k, void* y, int mode, void* stream) {
  g_err[0] = 0;
  int rc = check_layer(L);
  if (rc) return rc;
  KTMI_REQUIRE(tokens >= 0 && top_k > 0, KTMI_EINVAL, "moe_layer_noalloc: tokens %lld top_k %lld", (long long)tokens,
               (long long)top_k);
  if (tokens == 0) return KTMI_OK;
  if (mode == KTMI_MODE_AUTO) mode = ktmi_moe_layer_mode(L, tokens, top_k);
  const int64_t need = ktmi_moe_layer_workspace(L, tokens, top_k, mode);
  KTMI_REQUIRE(need <= KTMI_NOALLOC_SCRATCH_BYTES, KTMI_ESPACE,
               "moe_layer_noalloc: %lld tokens x top-%lld need %lld bytes of scratch, more than the %lld bytes the "
               "library holds per GPU (call ktmi_moe_layer with a workspace instead)",
               (long long)tokens, (long long)top_k, (long long)need, (long long)KTMI_NOALLOC_SCRATCH_BYTES);
  void* ws = nullptr;
  rc = scratch_of_current_device(&ws);
  if (rc) return rc;
  return ktmi_moe_layer(L, x, topk_w, slot_ids, tokens, top_k, y, ws, KTMI_NOALLOC_SCRATCH_BYTES, mode, stream);
}

}  // extern "C"
