// Entry points of linear layers with operands in 4 bits (packed4.h): argument checks, which kernel, what goes where in the workspace.
#include "packed4.h"

#include <algorithm>

using namespace wc;

namespace {

bool known(int dtype) { return dtype == WC_F32 || dtype == WC_F16 || dtype == WC_BF16; }

int check_extents4(long long rows, int C, int dtype, const char* who) {
  WC_CHECK_ARG(rows >= 0 && C > 0 && known(dtype), "%s: rows %lld, C %d, dtype %d", who, rows, C, dtype);
  if (rows > (1ll << 31) - 1 || C > kMostChannels4)
    return fail(WC_ERR_UNSUPPORTED, "%s: rows %lld, C %d (at most 2^31 - 1 and 2^22)", who, rows, C);
  return WC_OK;
}

// (codes are read and written by words and 16 bytes)
int check_starts(const unsigned char* codes, const unsigned char* scales, const char* who) {
  WC_CHECK_ARG(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0, "%s: codes and scales must start at multiples of 16 bytes", who);
  return WC_OK;
}

int check_packed(const wc_packed4* t, const char* what, const char* who) {
  WC_CHECK_ARG(t && t->codes && t->scales, "%s: %s is null", who, what);
  return check_starts(t->codes, t->scales, who);
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

int check_desc4(const wc_linear_desc* d, const char* who) {
  WC_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  if (int rc = check_extents4(d->rows, d->C, d->dtype, who)) return rc;
  WC_CHECK_ARG(d->K > 0 && d->activation >= WC_ACT_NONE && d->activation <= WC_ACT_SILU, "%s: K %d, activation %d", who, d->K, d->activation);
  if (d->K > kMostChannels4) return fail(WC_ERR_UNSUPPORTED, "%s: K %d (at most 2^22)", who, d->K);
  return WC_OK;
}

LinearProduct product_of(const wc_linear_desc* d, const void* x, const void* bias, const void* res, void* y) {
  return {x, nullptr, d->C, padded4(d->C), false, false, d->rows, d->K, d->C, {bias, res, y, nullptr, d->activation, d->residual_after != 0, 0}};
}

// A pass over the packed weight, whose workgroups read x anew for every 16 of its rows, up to 8 rows, and up to 16 over a weight of up to 2^25 values.  us, fp16, the pass | tiles:
// 16 x 4096 -> 4096 7.6 | 10, 16 x 8192 -> 8192 23.8 | 20.2, 16 x 25088 -> 4096 33 | 26
// fp32 rows, whose other way widens the weight and multiplies fp32 operands, are taken 16 at a time beside each other (us, passes | widened: 16 x 8192 -> 8192
// 42 | 179, 128 298 | 382, 128 x 25088 -> 4096 413 | 590, 256 x 512 -> 2048 29 | 22)
bool few(const wc_linear_desc* d, bool packed) {
  return d->rows <= 8 || (d->rows <= 16 && (long long)d->C * d->K <= 1ll << 25) || (!packed && d->dtype == WC_F32 && d->rows <= kMostFew4);
}
// Tiles that widen the codes in the registers, up to 2048 rows; above, and for fp32 and rows of x that are no whole 16 bytes, the weight is widened first, a launch and
// a pass over it, for the product of its own type.  us, fp16 8192 -> 8192, tiles | widened first: 64 rows 23 | 64, 1024 128 | 182, 2048 247 | 270, 4096 509 | 499
bool wide(const wc_linear_desc* d) { return d->rows <= kMostWide4 && linear4_wide_fits(nullptr, d->C, d->dtype); }

// the product of two packed operands, its reduction padded
LinearProduct tiled(LinearProduct p) {
  p.R = padded4(p.R);
  return p;
}

// What a backward pass leaves to wc_linear_backward, and what goes where in the workspace.  Up to most_gradient4 rows dx is passes over the packed weight, and dz and all
// else are the other's; above, the weight is widened first
// (dz of gelu and silu is rounded to the operands' type before dx, as in linear_gradient.hip and for its reason: the matrix cores take it so, and as a sum of two parts it
// would take twice the products, 256 of 320 us of bf16 8192 x 2048 <- 8192.  The 2-norm of dx's error there is 0.0023, of an unrounded dz 0.0017, of dx's own rounding 0.0017)
struct Backward4 { bool few, inner; wc_linear_gradients g; const void* dz; void* wide; float* parts; size_t inner_at, bytes; };
int backward4_plan(const wc_linear_desc* d, const wc_linear_gradients* g, void* workspace, Backward4* b) {
  // (sizes go by which pointers are null)
  char* const ws = workspace ? static_cast<char*>(workspace) : reinterpret_cast<char*>(256);
  const size_t size = d->dtype == WC_F32 ? 4 : 2;
  size_t at = 0;
  auto take = [&](size_t n) { char* p = ws + at; at += rounded(n); return p; };
  *b = {};
  b->g = *g;
  b->few = g->dx && d->rows <= most_gradient4(d->dtype);
  if (b->few) {
    b->g.dx = nullptr;
    b->g.w = nullptr;
    if (d->activation != WC_ACT_NONE && !g->dz) b->g.dz = take((size_t)d->rows * d->K * size);
    b->dz = d->activation != WC_ACT_NONE ? b->g.dz : g->dy;
    const int s = linear4_gradient_parts(d->rows, d->K, d->C, d->dtype);
    if (s > 1) b->parts = reinterpret_cast<float*>(take((size_t)s * d->rows * d->C * 4));
  } else if (g->dx) {
    b->wide = take((size_t)d->K * d->C * size);
    b->g.w = b->wide;
  }
  b->inner = b->g.dx || b->g.dw || b->g.db || b->g.dz;
  b->inner_at = b->bytes = at;
  if (!b->inner) return WC_OK;
  size_t inner = 0;
  if (int rc = wc_linear_backward_workspace_bytes(d, &b->g, &inner)) return rc;
  b->bytes += inner;
  return WC_OK;
}

}  // namespace

extern "C" {

int wc_packed4_bytes(long long rows, int C, size_t* codes, size_t* scales) {
  WC_CHECK_ARG(codes && scales, "wc_packed4_bytes: null output");
  if (int rc = check_extents4(rows, C, WC_F32, "wc_packed4_bytes")) return rc;
  *codes = (size_t)(rows * (padded4(C) / 2));
  *scales = (size_t)scale_bytes4(rows, C);
  return WC_OK;
}

int wc_pack4(const void* x, unsigned char* codes, unsigned char* scales, long long rows, int C, int dtype, void* stream) {
  if (int rc = check_extents4(rows, C, dtype, "wc_pack4")) return rc;
  if (rows == 0) return WC_OK;
  WC_CHECK_ARG(x && codes && scales, "wc_pack4: null pointer");
  if (int rc = check_starts(codes, scales, "wc_pack4")) return rc;
  return pack4(x, codes, scales, rows, C, dtype, stream);
}

int wc_unpack4(const unsigned char* codes, const unsigned char* scales, void* x, long long rows, int C, int dtype, void* stream) {
  if (int rc = check_extents4(rows, C, dtype, "wc_unpack4")) return rc;
  if (rows == 0) return WC_OK;
  WC_CHECK_ARG(x && codes && scales, "wc_unpack4: null pointer");
  if (int rc = check_starts(codes, scales, "wc_unpack4")) return rc;
  return unpack4(codes, scales, x, rows, C, dtype, stream);
}

int wc_linear4_workspace_bytes(const wc_linear_desc* d, int x_packed, size_t* bytes) {
  WC_CHECK_ARG(bytes != nullptr, "wc_linear4_workspace_bytes: null output");
  if (int rc = check_desc4(d, "wc_linear4_workspace_bytes")) return rc;
  *bytes = 0;
  if (d->rows == 0 || few(d, x_packed != 0)) return WC_OK;
  if (x_packed) {
    // (a plan goes by whether the epilogue is heavy: the larger of both)
    LinearProduct p = tiled(product_of(d, nullptr, nullptr, nullptr, nullptr));
    int s = 1;
    for (const int after : {0, 1}) {
      p.e.res = after ? d : nullptr;
      s = std::max(s, product4_plan(p).s);
    }
    *bytes = s > 1 ? rounded((size_t)s * d->rows * d->K * 4) : 0;
    return WC_OK;
  }
  if (wide(d)) {
    const LinearProduct p = product_of(d, nullptr, nullptr, nullptr, nullptr);
    const int s = linear4_wide_plan(p).s;
    *bytes = s > 1 ? rounded((size_t)s * d->rows * d->K * 4) : 0;
    return WC_OK;
  }
  size_t inner = 0;
  if (int rc = wc_linear_workspace_bytes(d, &inner)) return rc;
  *bytes = rounded((size_t)d->K * d->C * (d->dtype == WC_F32 ? 4 : 2)) + inner;
  return WC_OK;
}

int wc_linear4_forward(const wc_linear_desc* d, const void* x, const wc_packed4* x4, const wc_packed4* w4, const void* bias, const void* residual, void* y,
                       void* z, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = wc_linear4_workspace_bytes(d, x4 != nullptr, &need)) return rc;
  if (d->rows == 0) return WC_OK;
  WC_CHECK_ARG((x != nullptr) != (x4 != nullptr) && y, "wc_linear4_forward: x is given as it is or packed, and y");
  if (int rc = check_packed(w4, "w", "wc_linear4_forward")) return rc;
  if (x4)
    if (int rc = check_packed(x4, "x", "wc_linear4_forward")) return rc;
  if (need && (!workspace || workspace_bytes < need))
    return fail(WC_ERR_WORKSPACE, "wc_linear4_forward: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return fail(WC_ERR_WORKSPACE, "wc_linear4_forward: workspace must be 256-byte aligned");
  WC_CHECK_ARG(!z || !x4, "wc_linear4_forward: no z of an x in 4 bits, which has no gradient");
  LinearProduct p = product_of(d, x, bias, residual, y);
  p.e.z = z;
  const Operand4 w = {w4->codes, w4->scales};
  if (few(d, x4 != nullptr)) {
    const Operand4 xp = x4 ? Operand4{x4->codes, x4->scales} : Operand4{nullptr, nullptr};
    return product4_few(p, x4 ? &xp : nullptr, w, d->dtype, stream);
  }
  if (x4) {
    const LinearProduct t = tiled(p);
    const ProductPlan plan = product4_plan(t);
    if (plan.s > 1 && (size_t)plan.s * t.M * t.N * 4 > need) return fail(WC_ERR_WORKSPACE, "wc_linear4_forward: %d parts do not fit the workspace", plan.s);
    float* const parts = static_cast<float*>(workspace);
    if (int rc = product4_dma(t, {x4->codes, x4->scales}, w, plan, parts, d->dtype, stream)) return rc;
    const LinearJoin join = {t.e, parts, plan.s, t.M, t.N};
    return linear_join(&join, 1, nullptr, nullptr, d->dtype, stream);
  }
  if (wide(d)) {
    const ProductPlan plan = linear4_wide_plan(p);
    float* const parts = static_cast<float*>(workspace);
    if (plan.s > 1 && (size_t)plan.s * p.M * p.N * 4 > need) return fail(WC_ERR_WORKSPACE, "wc_linear4_forward: %d parts do not fit the workspace", plan.s);
    WC_CHECK_ARG(linear4_wide_fits(x, d->C, d->dtype), "wc_linear4_forward: x must start at a multiple of 16 bytes");
    if (int rc = linear4_wide(p, w, plan, parts, d->dtype, stream)) return rc;
    const LinearJoin join = {p.e, parts, plan.s, p.M, p.N};
    return linear_join(&join, 1, nullptr, nullptr, d->dtype, stream);
  }
  char* const ws = static_cast<char*>(workspace);
  const size_t wide_bytes = rounded((size_t)d->K * d->C * (d->dtype == WC_F32 ? 4 : 2));
  if (int rc = unpack4(w.codes, w.scales, ws, d->K, d->C, d->dtype, stream)) return rc;
  return wc_linear_forward(d, x, ws, bias, residual, y, z, ws + wide_bytes, need - wide_bytes, stream);
}

int wc_linear4_backward_workspace_bytes(const wc_linear_desc* d, const wc_linear_gradients* g, size_t* bytes) {
  WC_CHECK_ARG(bytes != nullptr && g != nullptr, "wc_linear4_backward_workspace_bytes: null pointer");
  if (int rc = check_desc4(d, "wc_linear4_backward_workspace_bytes")) return rc;
  *bytes = 0;
  if (d->rows == 0) return WC_OK;
  Backward4 b;
  if (int rc = backward4_plan(d, g, nullptr, &b)) return rc;
  *bytes = b.bytes;
  return WC_OK;
}

int wc_linear4_backward(const wc_linear_desc* d, const wc_linear_gradients* g, const wc_packed4* w4, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = wc_linear4_backward_workspace_bytes(d, g, &need)) return rc;
  WC_CHECK_ARG(d->rows > 0, "wc_linear4_backward: no rows (the gradients of the parameters are zero)");
  WC_CHECK_ARG(g->dy, "wc_linear4_backward: dy is null");
  WC_CHECK_ARG(!g->w, "wc_linear4_backward: w is given packed");
  WC_CHECK_ARG(d->activation == WC_ACT_NONE || g->z, "wc_linear4_backward: an activation's gradient needs z");
  if (g->dx)
    if (int rc = check_packed(w4, "w", "wc_linear4_backward")) return rc;
  if (need && (!workspace || workspace_bytes < need))
    return fail(WC_ERR_WORKSPACE, "wc_linear4_backward: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return fail(WC_ERR_WORKSPACE, "wc_linear4_backward: workspace must be 256-byte aligned");
  Backward4 b;
  if (int rc = backward4_plan(d, g, workspace, &b)) return rc;
  if (b.wide)
    if (int rc = unpack4(w4->codes, w4->scales, b.wide, d->K, d->C, d->dtype, stream)) return rc;
  if (b.inner)
    if (int rc = wc_linear_backward(d, &b.g, need ? static_cast<char*>(workspace) + b.inner_at : nullptr, need - b.inner_at, stream)) return rc;
  if (!b.few) return WC_OK;
  return linear4_gradient(b.dz, {w4->codes, w4->scales}, g->dx, b.parts, d->rows, d->K, d->C, d->dtype, stream);
}

}  // extern "C"
