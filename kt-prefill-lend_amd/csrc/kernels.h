// Host-side launchers shared between the kernel files and the C entry points.
#pragma once
#include "ktmi_common.h"

namespace ktmi {

int launch_dequant(const uint8_t* raw, int64_t raw_stride, int type, int64_t n, int64_t rows, int64_t cols,
                   uint16_t* out, int64_t out_stride, hipStream_t stream);
int launch_route(const int32_t* ids, int64_t n, const int32_t* log2slot, const int32_t* log2cpu, float* counts,
                 int32_t* slot_ids, int32_t* cpu_ids, hipStream_t stream);
int launch_quantize_q8_1(const void* x, int dtype, int64_t cols, int64_t tokens, uint8_t* out, hipStream_t stream);
int launch_silu_and_mul(const void* h, int dtype, int64_t R, int64_t N, void* out, hipStream_t stream);
int launch_combine(const void* out, int dtype, const float* w, int64_t T, int64_t top_k, int64_t K, void* res,
                   hipStream_t stream);

// Tokens sorted by expert and back (moe_sort.hip). x_stride, row_stride, dy_stride in elements, es
// the bytes of one; counts: moe_sort_counts(tokens, top_k) * (E + 1) ints; rows = NULL: the order alone.
constexpr int64_t SORT_MAX_EXPERTS = 2048;
int64_t moe_sort_counts(int64_t tokens, int64_t top_k);
int launch_moe_sort(const uint8_t* x, int es, int64_t x_stride, int64_t cols, const int32_t* ids, int64_t tokens,
                    int64_t top_k, int64_t E, uint8_t* rows, int32_t* offsets, int32_t* perm, int32_t* pos, int* counts,
                    hipStream_t stream);
int launch_moe_unsort(const void* rows, int dtype, int64_t row_stride, int64_t cols, const float* w, const int32_t* pos,
                      int64_t tokens, int64_t top_k, void* y, hipStream_t stream);
int launch_moe_unsort_grad(const void* dy, int64_t dy_stride, const void* rows, int64_t row_stride, int dtype,
                           int64_t cols, const float* w, const int32_t* pos, int64_t tokens, int64_t top_k, void* drows,
                           float* dw, hipStream_t stream);

// Products with 4-bit weights (w4.hip). Route r's activation row is r / top_k and its expert ids[r]; with
// offsets instead, row r and the expert whose segment holds it; with neither, row r and the one matrix.
struct W4Args {
  const void* x;
  int64_t x_stride, cols;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  int64_t group, rows, n_experts;
  const int32_t* ids;
  const int32_t* offsets;
  int64_t top_k, n_routes;
  void* y;
  uint8_t* ws;
  int x_dtype, scale_dtype;
  const int32_t* perm;  // with offsets: the route at each place (set by launch_w4 alone)
};
constexpr int W4_LDS_MOST = 152 << 10;
int64_t w4_workspace(int64_t tokens, int64_t top_k, int64_t n_experts);
// tell: takes what the call would launch, and nothing is launched
int launch_w4(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell = nullptr);
// by activation type: one pass without a sort
int launch_w4_bf16(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell);
int launch_w4_f16(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell);
int launch_w4_f32(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell);
constexpr int W4_STEP = 128;  // columns of a step: 16 bytes of codes a lane
constexpr int64_t W4_ROUTES = 1 << 23;  // rows of y of a call, at most: a grid has below 2^32 threads
constexpr int W4_IDS = 64;    // routes whose ids a wave holds one a lane

// Products by expert (prod.hip): rows of x or dy by the matrix of their expert, w [n_experts, rows, cols] (gated: [2 rows,
// cols]); offsets NULL: one matrix. y: the products, or the gradient asked for. Strides in elements.
struct ProdArgs {
  int dtype;
  const void* x;
  int64_t x_stride;
  const void* dy;
  int64_t dy_stride;
  const void* w;
  int64_t rows, cols, n_experts;
  const int32_t* offsets;
  int64_t n_rows;
  int act;
  void* y;
  float* sums;
  float* part;  // workspace
};
int64_t prod_workspace(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows);
ktmi_prod_kernel prod_kernel_of(int what, int dtype, int64_t rows, int64_t cols, int64_t n_experts, int64_t n_rows);
int launch_prod(int what, const ProdArgs& a, hipStream_t stream);
int launch_gated_grad(const float* sums, const void* dh, int dtype, int64_t dh_stride, int64_t inter, int64_t n_rows, int act,
                      void* dsums, hipStream_t stream);
// Products in 8-bit floating point: x [x_rows, cols] by e4m3 matrices with a scale for each block of 128 x 128; route r's
// row of x is r / top_k and its expert ids[r], or that of the segment that holds row r, or the one matrix.
struct Fp8Args {
  int dtype;
  const void* x;
  int64_t x_stride, x_rows;
  const uint8_t* w;
  const float* scales;
  int64_t rows, cols, n_experts;
  const int32_t* ids;
  int64_t top_k;
  const int32_t* offsets;
  void* y;
  uint8_t* ws;
};
int64_t fp8_workspace(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids);
ktmi_prod_kernel fp8_kernel_of(int64_t rows, int64_t cols, int64_t x_rows, int64_t n_experts, int64_t top_k, bool ids);
int launch_fp8(const Fp8Args& a, hipStream_t stream);

// GEMV over raw GGUF rows against q8_1 activations (the decode-window kernel).
// xq: q8_1 rows of the tokens, xq_stride bytes apart. W: slot tensor (w_is_table = 0,
// experts w_expert_stride bytes apart) or int64 table of per-slot addresses. Expert ids
// outside [0, n_experts) give zero rows like ids < 0.
int launch_moe_gemv(const uint8_t* xq, int64_t xq_stride, const void* W, int w_is_table, int64_t w_expert_stride,
                    const int32_t* ids, int64_t top_k, int64_t n_routes, int type, int64_t rows, int64_t cols,
                    void* Y, int y_dtype, int per_route, int n_experts, hipStream_t stream);

// Optional stage timing: when set (ktmi_set_stage_events), the layer records events[i]
// on its stream at each stage boundary (KTMI_STAGE_EVENTS of them).
void record_stage(int i, hipStream_t stream);

// Fused decode-sized layer (decode_layer.hip): two launches, for up to DEC_MAX_ROUTES
// routes, DEC_MAX_SLOTS slots and hidden sizes whose q8_1 rows fit DEC_MAX_XQ_LDS; the
// stage-by-stage GEMV sequence covers the rest.
constexpr int DEC_MAX_ROUTES = 256;
constexpr int DEC_MAX_SLOTS = 512;
constexpr int DEC_MAX_XQ_LDS = 48 * 1024;
bool decode_layer_fits(const ktmi_layer* L, int64_t tokens, int64_t top_k);
int64_t decode_layer_workspace(const ktmi_layer* L, int64_t tokens, int64_t top_k);
int launch_decode_layer(const ktmi_layer* L, const uint16_t* x, const float* topk_w, const int32_t* slot_ids,
                        int64_t tokens, int64_t top_k, uint16_t* y, uint8_t* ws, hipStream_t stream);

// Decode-sized layer on the matrix cores (decode_mfma.hip): three launches. The decode mode
// takes up to DM_MAX_ROUTES routes of at most DM_MAX_TOKENS tokens; the grouped mode runs the
// same kernels on its shortest chunks (window_fits), with h [R, inter] and yv [R, hidden] in
// its own workspace.
constexpr int DM_MAX_ROUTES = 256;
constexpr int DM_MAX_TOKENS = 64;
bool window_fits(const ktmi_layer* L, int64_t tokens, int64_t top_k);
int launch_window(const ktmi_layer* L, const uint16_t* x, const float* topk_w, const int32_t* slot_ids, int64_t tokens,
                  int64_t top_k, uint16_t* y, uint16_t* hbuf, uint16_t* yv, hipStream_t stream);
bool decode_mfma_fits(const ktmi_layer* L, int64_t tokens, int64_t top_k);
int64_t decode_mfma_workspace(const ktmi_layer* L, int64_t tokens, int64_t top_k);
int launch_decode_mfma(const ktmi_layer* L, const uint16_t* x, const float* topk_w, const int32_t* slot_ids,
                       int64_t tokens, int64_t top_k, uint16_t* y, uint8_t* ws, hipStream_t stream);

// Grouped prefill path (moe_gemm.hip).
struct GroupedPlan {
  int64_t routes;      // tokens * top_k
  int64_t n_slots;
  int64_t max_tiles;   // upper bound of M tiles over all slots
  int fj;              // route fragments of 32 per wave (the kernel's FJ)
  int64_t bm;          // routes per M tile (32 fj)
  // workspace carve-up (byte offsets)
  int64_t off_counts, off_seg, off_tseg, off_tinfo, off_perm, off_tok, off_h, off_y, total;
};
GroupedPlan grouped_plan(int64_t tokens, int64_t top_k, int64_t n_slots, int64_t hidden, int64_t inter);
// window: run the decode-sized kernels (window_fits of the whole call, so that every pass of a
// longer one sums in the GEMMs' order, whatever its number of tokens).
int launch_grouped_layer(const ktmi_layer* L, const uint16_t* x, const float* topk_w, const int32_t* slot_ids,
                         int64_t tokens, int64_t top_k, uint16_t* y, uint8_t* ws, const GroupedPlan& P, bool window,
                         hipStream_t stream);

}  // namespace ktmi
