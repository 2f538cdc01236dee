// Entry points of linear layers and of activations in 8 bits: argument checks, what goes where in the workspace, the launches.
#include "linear.h"

#include <algorithm>

using namespace wc;

namespace {

constexpr double kWidenPays = 1e8;      // multiplications

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
bool known(int dtype) { return dtype == WC_F32 || dtype == WC_F16 || dtype == WC_BF16; }
int size_of(int dtype) { return dtype == WC_F32 ? 4 : 2; }

// extents whose products stay far inside 63 bits
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

// (a plan never has more parts than the workspace was sized for; checked all the same, since they would be written behind it)
bool parts_fit(const LinearProduct& p, const ProductPlan& plan, size_t at, size_t end) {
  return plan.s == 1 || at + (size_t)plan.s * p.M * p.N * 4 <= end;
}

// Rows that are no multiple of 16 bytes are copied to ones that are, for the kernel that brings them to LDS without registers, where the product is
// worth it: the copy is a launch and a pass over the operands.
bool widen_pays(long long M, long long N, long long R) { return (double)M * N * R >= kWidenPays; }

struct Forward {
  LinearProduct p;
  WideCopy copies[2];
  bool widen;
  size_t scratch_at, bytes;
};

Forward forward_plan(const wc_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y, void* z, char* ws) {
  Forward f;
  const long long ld = wide_row(d->C, d->dtype);
  const size_t es = size_of(d->dtype);
  size_t at = 0;
  f.widen = ld != d->C && widen_pays(d->rows, d->K, d->C);
  if (f.widen) {
    f.copies[0] = {x, ws, d->rows, d->C, ld};
    at = rounded((size_t)d->rows * ld * es);
    f.copies[1] = {w, ws + at, d->K, d->C, ld};
    at += rounded((size_t)d->K * ld * es);
    x = f.copies[0].to;
    w = f.copies[1].to;
  }
  f.p = {x, w, f.widen ? ld : d->C, f.widen ? ld : d->C, false, false, d->rows, d->K, d->C, {bias, res, y, z, d->activation, d->residual_after != 0, 0}};
  f.scratch_at = at;
  f.bytes = at + rounded(product_parts_bytes(f.p, d->dtype, nullptr));
  return f;
}

// What a backward pass launches, and where its scratch lies
struct Backward {
  LinearPrepare before;
  LinearProduct dx, dw;
  size_t sums_at, dx_at, dw_at, bytes;
};

Backward backward_plan(const wc_linear_desc* d, const wc_linear_gradients* g, char* ws) {
  Backward b = {};
  const size_t es = size_of(d->dtype);
  const bool acts = d->activation != WC_ACT_NONE, products = g->dx || g->dw;
  // (either product reads what the other does, so they are widened together)
  const long long ldc = wide_row(d->C, d->dtype), ldk = wide_row(d->K, d->dtype);
  const bool widen = products && widen_pays(d->rows, d->K, d->C), wide_c = widen && ldc != d->C, wide_k = widen && ldk != d->K;
  size_t at = 0;
  auto take = [&](size_t n) { void* const p = ws + at; at += rounded(n); return p; };
  LinearPrepare& f = b.before;
  const void* dz = g->dy;
  void *dz_out = g->dz, *dz_wide = nullptr;       // without an activation: copies of dy
  long long ld_dz = d->K;
  if (products && wide_k) {
    dz = dz_wide = take((size_t)d->rows * ldk * es);
    ld_dz = ldk;
  } else if (products && acts) {
    if (!dz_out) dz_out = take((size_t)d->rows * d->K * es);
    dz = dz_out;
  }
  const long long ld = wide_c ? ldc : d->C;
  const void *w = g->w, *x = g->x;
  if (g->dx && wide_c) {
    f.copies[f.n_copies++] = {w, take((size_t)d->K * ldc * es), d->K, d->C, ldc};
    w = f.copies[0].to;
  }
  if (g->dw && (g->x_exponents || wide_c)) {
    void* const to = take((size_t)d->rows * ld * es);
    if (g->x_exponents) {
      f.codes = static_cast<const signed char*>(g->x);
      f.exps = g->x_exponents;
      f.x = to;
      f.x_rows = d->rows; f.x_ld = ld; f.x_C = d->C;
    } else {
      f.copies[f.n_copies++] = {x, to, d->rows, d->C, ldc};
    }
    x = to;
  }
  f.run_slope = dz_out || dz_wide || g->db;
  f.slope = {g->dy, acts ? g->z : nullptr, acts ? g->z_exponents : nullptr, dz_out, g->db, dz_wide, ldk, d->activation, g->db_dtype == WC_F32, d->rows, d->K};
  b.dx = {dz, w, ld_dz, ld, false, true, d->rows, d->C, d->K, {nullptr, nullptr, g->dx, nullptr, WC_ACT_NONE, 0, 0}};
  b.dw = {dz, x, ld_dz, ld, true, true, d->K, d->C, d->rows, {nullptr, nullptr, g->dw, nullptr, WC_ACT_NONE, 0, g->dw_dtype == WC_F32}};
  b.sums_at = at;
  at += rounded(linear_sums_bytes(f.slope));
  b.dx_at = at;
  if (g->dx) at += rounded(product_parts_bytes(b.dx, d->dtype, nullptr));
  b.dw_at = at;
  if (g->dw) at += rounded(product_parts_bytes(b.dw, d->dtype, &b.dx));
  b.bytes = at;
  return b;
}

}  // namespace

extern "C" {

int wc_linear_workspace_bytes(const wc_linear_desc* d, size_t* bytes) {
  WC_CHECK_ARG(bytes != nullptr, "wc_linear_workspace_bytes: null output");
  if (int rc = check_desc(d, "wc_linear_workspace_bytes")) return rc;
  *bytes = d->rows == 0 ? 0 : forward_plan(d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr).bytes;
  return WC_OK;
}

int wc_linear_forward(const wc_linear_desc* d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z,
                      void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = wc_linear_workspace_bytes(d, &need)) return rc;
  if (d->rows == 0) return WC_OK;
  WC_CHECK_ARG(x && w && y, "wc_linear_forward: null pointer");
  if (int rc = check_workspace(workspace, workspace_bytes, need, "wc_linear_forward")) return rc;
  char* const ws = static_cast<char*>(workspace);
  const Forward f = forward_plan(d, x, w, bias, residual, y, z, ws);
  float* const parts = reinterpret_cast<float*>(ws + f.scratch_at);
  const ProductPlan plan = product_plan(f.p, d->dtype, nullptr);
  if (!parts_fit(f.p, plan, f.scratch_at, need)) return fail(WC_ERR_WORKSPACE, "wc_linear_forward: %d parts do not fit the workspace", plan.s);
  if (f.widen) {
    LinearPrepare before = {};
    before.copies[0] = f.copies[0];
    before.copies[1] = f.copies[1];
    before.n_copies = 2;
    if (int rc = linear_prepare(before, d->dtype, nullptr, stream)) return rc;
  }
  if (int rc = product_run(f.p, plan, parts, d->dtype, stream)) return rc;
  const LinearJoin join = {f.p.e, parts, plan.s, f.p.M, f.p.N};
  return linear_join(&join, 1, nullptr, nullptr, d->dtype, stream);
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
  auto at = [&](size_t n) { return reinterpret_cast<float*>(ws + n); };
  LinearJoin joins[2];
  int n = 0;
  const ProductPlan dx = product_plan(b.dx, d->dtype, nullptr), dw = product_plan(b.dw, d->dtype, &b.dx);      // dw's bits do not hang on whether dx is asked for
  if ((g->dx && !parts_fit(b.dx, dx, b.dx_at, b.dw_at)) || (g->dw && !parts_fit(b.dw, dw, b.dw_at, need)))
    return fail(WC_ERR_WORKSPACE, "wc_linear_backward: %d and %d parts do not fit the workspace", dx.s, dw.s);
  if (int rc = linear_prepare(b.before, d->dtype, at(b.sums_at), stream)) return rc;
  if (g->dx) joins[n++] = {b.dx.e, at(b.dx_at), dx.s, b.dx.M, b.dx.N};
  if (g->dw) joins[n++] = {b.dw.e, at(b.dw_at), dw.s, b.dw.M, b.dw.N};
  int rc = WC_OK;
  if (n == 2) rc = product_run_pair(b.dx, dx, at(b.dx_at), b.dw, dw, at(b.dw_at), d->dtype, stream);
  else if (g->dx) rc = product_run(b.dx, dx, at(b.dx_at), d->dtype, stream);
  else if (g->dw) rc = product_run(b.dw, dw, at(b.dw_at), d->dtype, stream);
  if (rc) return rc;
  return linear_join(joins, n, g->db ? &b.before.slope : nullptr, at(b.sums_at), d->dtype, stream);
}

int wc_pack8(const void* x, signed char* codes, signed char* exponents, long long rows, int C, int dtype, int keep_sign, void* stream) {
  if (int rc = check_extents(rows, C, 1, dtype, "wc_pack8")) return rc;
  if (rows == 0) return WC_OK;
  WC_CHECK_ARG(x && codes && exponents, "wc_pack8: null pointer");
  if (rows * pack_groups(C) >= (1ll << 36)) return fail(WC_ERR_UNSUPPORTED, "wc_pack8: rows %lld, C %d", rows, C);
  return pack8(x, codes, exponents, rows, C, keep_sign == kPackGates ? kPackGates : keep_sign ? kPackSigns : 0, dtype, stream);
}

int wc_unpack8(const signed char* codes, const signed char* exponents, void* x, long long rows, int C, int dtype, void* stream) {
  if (int rc = check_extents(rows, C, 1, dtype, "wc_unpack8")) return rc;
  if (rows == 0) return WC_OK;
  WC_CHECK_ARG(x && codes && exponents, "wc_unpack8: null pointer");
  if (rows * pack_groups(C) >= (1ll << 36)) return fail(WC_ERR_UNSUPPORTED, "wc_unpack8: rows %lld, C %d", rows, C);
  return unpack8(codes, exponents, x, rows, C, dtype, stream);
}

}  // extern "C"
