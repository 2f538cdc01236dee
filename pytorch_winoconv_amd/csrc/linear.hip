// Entry points of linear layers and of activations in 8 bits: argument checks, what goes where in the workspace, the launches.
#include "linear.h"

#include <algorithm>

using namespace wc;

namespace {

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
bool known(int dtype) { return dtype == WC_F32 || dtype == WC_F16 || dtype == WC_BF16; }
int size_of(int dtype) { return dtype == WC_F32 ? 4 : 2; }

// extents whose products stay far inside 63 bits and whose launches inside 31
int check_extents(long long rows, int C, int K, int dtype, const char* who) {
  WC_CHECK_ARG(rows >= 0 && C > 0 && K > 0 && known(dtype), "%s: rows %lld, C %d, K %d, dtype %d", who, rows, C, K, dtype);
  if (rows > (1ll << 31) - 1 || C > (1 << 24) || K > (1 << 24))
    return fail(WC_ERR_UNSUPPORTED, "%s: rows %lld, C %d, K %d (at most 2^31 - 1, 2^24 and 2^24)", who, rows, C, K);
  return WC_OK;
}

int check_desc(const wc_linear_desc* d, const char* who) {
  WC_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  if (int rc = check_extents(d->rows, d->C, d->K, d->dtype, who)) return rc;
  WC_CHECK_ARG(d->activation >= WC_ACT_NONE && d->activation <= WC_ACT_SILU, "%s: activation %d", who, d->activation);
  return WC_OK;
}

int check_workspace(const void* ws, size_t have, size_t need, const char* who) {
  if (need == 0) return WC_OK;
  if (!ws || have < need) return fail(WC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, ws ? have : (size_t)0, need);
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0) return fail(WC_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
  return WC_OK;
}

LinearProduct forward_product(const wc_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y, void* z) {
  return {x, w, d->C, d->C, false, false, d->rows, d->K, d->C, {bias, res, y, z, d->activation, d->residual_after != 0, 0}};
}

// What a backward pass launches, and where its scratch lies
struct Backward {
  LinearSlope slope;
  LinearProduct dx, dw;
  bool run_slope, unpack_x;
  size_t dz_at, x_at, scratch_at, bytes;
};

Backward backward_plan(const wc_linear_desc* d, const wc_linear_gradients* g, char* ws) {
  Backward b;
  const size_t es = size_of(d->dtype);
  const bool acts = d->activation != WC_ACT_NONE;
  size_t at = 0;
  const void* dz = g->dy;
  void* dz_out = nullptr;
  b.dz_at = at;
  if (acts && (g->dx || g->dw || g->dz)) {
    dz_out = g->dz ? g->dz : ws + at;
    dz = dz_out;
    if (!g->dz) at += rounded((size_t)d->rows * d->K * es);
  } else if (!acts) {
    dz_out = g->dz;                              // a copy of dy
  }
  b.unpack_x = g->dw && g->x_exponents;
  b.x_at = at;
  const void* x = g->x;
  if (b.unpack_x) {
    x = ws + at;
    at += rounded((size_t)d->rows * d->C * es);
  }
  b.scratch_at = at;
  b.run_slope = dz_out || g->db;
  b.slope = {g->dy, acts ? g->z : nullptr, acts ? g->z_exponents : nullptr, dz_out, g->db, d->activation, g->db_dtype == WC_F32, d->rows, d->K};
  b.dx = {dz, g->w, d->K, d->C, false, true, d->rows, d->C, d->K, {nullptr, nullptr, g->dx, nullptr, WC_ACT_NONE, 0, 0}};
  b.dw = {dz, x, d->K, d->C, true, true, d->K, d->C, d->rows, {nullptr, nullptr, g->dw, nullptr, WC_ACT_NONE, 0, g->dw_dtype == WC_F32}};
  size_t scratch = b.run_slope ? linear_slope_bytes(b.slope, d->dtype) : 0;
  if (g->dx) scratch = std::max(scratch, linear_product_bytes(b.dx, d->dtype));
  if (g->dw) scratch = std::max(scratch, linear_product_bytes(b.dw, d->dtype));
  b.bytes = at + rounded(scratch);
  return b;
}

}  // namespace

extern "C" {

int wc_linear_workspace_bytes(const wc_linear_desc* d, size_t* bytes) {
  WC_CHECK_ARG(bytes != nullptr, "wc_linear_workspace_bytes: null output");
  if (int rc = check_desc(d, "wc_linear_workspace_bytes")) return rc;
  *bytes = d->rows == 0 ? 0 : linear_product_bytes(forward_product(d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr), d->dtype);
  return WC_OK;
}

int wc_linear_forward(const wc_linear_desc* d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z,
                      void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = wc_linear_workspace_bytes(d, &need)) return rc;
  if (d->rows == 0) return WC_OK;
  WC_CHECK_ARG(x && w && y, "wc_linear_forward: null pointer");
  if (int rc = check_workspace(workspace, workspace_bytes, need, "wc_linear_forward")) return rc;
  return linear_product(forward_product(d, x, w, bias, residual, y, z), d->dtype, workspace, stream);
}

int wc_linear_backward_workspace_bytes(const wc_linear_desc* d, const wc_linear_gradients* g, size_t* bytes) {
  WC_CHECK_ARG(bytes != nullptr && g != nullptr, "wc_linear_backward_workspace_bytes: null pointer");
  if (int rc = check_desc(d, "wc_linear_backward_workspace_bytes")) return rc;
  *bytes = d->rows == 0 ? 0 : backward_plan(d, g, nullptr).bytes;
  return WC_OK;
}

int wc_linear_backward(const wc_linear_desc* d, const wc_linear_gradients* g, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = wc_linear_backward_workspace_bytes(d, g, &need)) return rc;
  WC_CHECK_ARG(d->rows > 0, "wc_linear_backward: no rows (the gradients of the parameters are zero)");
  WC_CHECK_ARG(g->dy, "wc_linear_backward: dy is null");
  WC_CHECK_ARG(!g->dx || g->w, "wc_linear_backward: dx needs w");
  WC_CHECK_ARG(!g->dw || g->x, "wc_linear_backward: dw needs x");
  WC_CHECK_ARG(d->activation == WC_ACT_NONE || g->z, "wc_linear_backward: an activation's gradient needs z");
  WC_CHECK_ARG(!g->dw || g->dw_dtype == WC_F32 || g->dw_dtype == d->dtype, "wc_linear_backward: dw of type %d", g->dw_dtype);
  WC_CHECK_ARG(!g->db || g->db_dtype == WC_F32 || g->db_dtype == d->dtype, "wc_linear_backward: db of type %d", g->db_dtype);
  if (int rc = check_workspace(workspace, workspace_bytes, need, "wc_linear_backward")) return rc;
  char* const ws = static_cast<char*>(workspace);
  const Backward b = backward_plan(d, g, ws);
  void* const scratch = ws + b.scratch_at;
  if (b.run_slope)
    if (int rc = linear_slope(b.slope, d->dtype, scratch, stream)) return rc;
  if (g->dx)
    if (int rc = linear_product(b.dx, d->dtype, scratch, stream)) return rc;
  if (!g->dw) return WC_OK;
  if (b.unpack_x)
    if (int rc = unpack8(static_cast<const signed char*>(g->x), g->x_exponents, ws + b.x_at, d->rows, d->C, d->dtype, stream)) return rc;
  return linear_product(b.dw, d->dtype, scratch, stream);
}

int wc_pack8(const void* x, signed char* codes, signed char* exponents, long long rows, int C, int dtype, int keep_sign, void* stream) {
  if (int rc = check_extents(rows, C, 1, dtype, "wc_pack8")) return rc;
  if (rows == 0) return WC_OK;
  WC_CHECK_ARG(x && codes && exponents, "wc_pack8: null pointer");
  if (rows * pack_groups(C) >= (1ll << 36)) return fail(WC_ERR_UNSUPPORTED, "wc_pack8: rows %lld, C %d", rows, C);
  return pack8(x, codes, exponents, rows, C, keep_sign != 0, dtype, stream);
}

int wc_unpack8(const signed char* codes, const signed char* exponents, void* x, long long rows, int C, int dtype, void* stream) {
  if (int rc = check_extents(rows, C, 1, dtype, "wc_unpack8")) return rc;
  if (rows == 0) return WC_OK;
  WC_CHECK_ARG(x && codes && exponents, "wc_unpack8: null pointer");
  if (rows * pack_groups(C) >= (1ll << 36)) return fail(WC_ERR_UNSUPPORTED, "wc_unpack8: rows %lld, C %d", rows, C);
  return unpack8(codes, exponents, x, rows, C, dtype, stream);
}

}  // extern "C"
