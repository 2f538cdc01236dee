// Entry points of the joins of blocks to their stream: argument checks, the workspace, the launches.
#include "residual.h"

#include <cmath>

using namespace wc;

namespace {

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

int check_norm(const wc_norm& n, int dtype, const char* what, const char* who) {
  WC_CHECK_ARG(n.kind >= WC_NORM_NONE && n.kind <= WC_NORM_LAYER, "%s: %s of kind %d", who, what, n.kind);
  if (n.kind == WC_NORM_NONE) return WC_OK;
  WC_CHECK_ARG(n.eps >= 0 && std::isfinite(n.eps), "%s: eps %g of %s", who, (double)n.eps, what);
  WC_CHECK_ARG(n.dtype == WC_F32 || n.dtype == dtype, "%s: parameters of %s of type %d", who, what, n.dtype);
  return WC_OK;
}

int check_desc(const wc_join_desc* d, const char* who) {
  WC_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  WC_CHECK_ARG(d->rows >= 0 && d->C > 0 && (d->dtype == WC_F32 || d->dtype == WC_F16 || d->dtype == WC_BF16), "%s: rows %lld, C %d, dtype %d", who, d->rows, d->C, d->dtype);
  if (d->rows > (1ll << 31) - 1 || d->C > (1 << 24)) return fail(WC_ERR_UNSUPPORTED, "%s: rows %lld, C %d (at most 2^31 - 1 and 2^24)", who, d->rows, d->C);
  WC_CHECK_ARG(d->samples >= 1 && d->rows % d->samples == 0, "%s: %lld rows of %lld samples", who, d->rows, d->samples);
  WC_CHECK_ARG(d->gate_rows == 0 || d->gate_rows == 1 || d->gate_rows == d->samples, "%s: a gate of %lld rows, %lld samples", who, d->gate_rows, d->samples);
  WC_CHECK_ARG(d->gate_rows == 0 || d->gate_dtype == WC_F32 || d->gate_dtype == d->dtype, "%s: a gate of type %d", who, d->gate_dtype);
  WC_CHECK_ARG(d->drop_level >= 0 && d->drop_level <= 65536, "%s: drop level %d of 65536", who, d->drop_level);
  if (int rc = check_norm(d->post, d->dtype, "post", who)) return rc;
  return check_norm(d->pre, d->dtype, "pre", who);
}

// (a row's two are one access)
int check_stats(const void* a, const void* b, const char* who) {
  WC_CHECK_ARG(reinterpret_cast<uintptr_t>(a) % 8 == 0 && reinterpret_cast<uintptr_t>(b) % 8 == 0, "%s: statistics must start at multiples of 8 bytes", who);
  return WC_OK;
}

Norm norm_of(const wc_norm& n) { return {n.kind, n.eps, n.weight, n.bias, n.dtype == WC_F32}; }
Dropout drop_of(const wc_join_desc* d) {
  return {(unsigned)d->drop_level, d->drop_per_sample != 0, d->drop_level == 0 ? 1.f : d->drop_level == 65536 ? 0.f : 65536.f / (float)(65536 - d->drop_level), d->drop_seed,
          d->drop_offset, reinterpret_cast<const unsigned long long*>(d->drop_state)};
}
int gate_of(const wc_join_desc* d) {
  if (d->gate_rows == 0) return kNoGate;
  if (d->gate_rows == 1) return kGateChannel;
  return d->gate_rows == d->rows ? kGateRow : kGateSample;
}

struct Backward {
  JoinGradients g;
  JoinSum sums[5];
  int n;
  size_t bytes;
};

Backward backward_plan(const wc_join_desc* d, const wc_join_gradients* q, char* ws) {
  Backward b = {};
  JoinGradients& g = b.g;
  g = {d->rows, d->rows / d->samples, d->C, q->ds, q->dy, q->f, q->s, q->x, q->gate, gate_of(d), d->gate_dtype == WC_F32, d->stream_scale, d->block_scale, norm_of(d->post),
       norm_of(d->pre), drop_of(d), q->post_stats, q->pre_stats, q->df, q->dx, nullptr, {}, 1, 1, 1};
  if (!q->dy) g.pre.kind = WC_NORM_NONE;
  if (d->dtype != WC_F32 && g.f) g.s = nullptr;
  if (g.gate_rows == kGateRow) g.dgate_rows = q->dgate;
  void* const to[5] = {q->dpre_weight, q->dpre_bias, q->dpost_weight, q->dpost_bias, g.dgate_rows ? nullptr : q->dgate};
  join_plan(&g);
  size_t at = 0;
  for (int k = 0; k < 5; ++k) {
    g.part[k] = nullptr;
    if (!to[k]) continue;
    const long long rows = k == kGateSum ? g.segments * g.parts : g.blocks;
    g.part[k] = reinterpret_cast<float*>(ws + at);
    at += rounded((size_t)rows * d->C * 4);
    const int dtype = k == kGateSum ? d->gate_dtype : k < kPostWeight ? d->pre.dtype : d->post.dtype;
    b.sums[b.n++] = {g.part[k], to[k], dtype == WC_F32, k == kGateSum ? g.segments : 1, (int)(k == kGateSum ? g.parts : g.blocks)};
  }
  b.bytes = at;
  return b;
}

}  // namespace

extern "C" {

int wc_join_forward(const wc_join_desc* d, const void* f, const void* x, const void* gate, void* s, void* y, float* post_stats, float* pre_stats, void* stream) {
  if (int rc = check_desc(d, "wc_join_forward")) return rc;
  WC_CHECK_ARG(d->pre.kind != WC_NORM_NONE || !y, "wc_join_forward: y without its norm");
  if (d->rows == 0) return WC_OK;
  WC_CHECK_ARG(f && (s || y), "wc_join_forward: null pointer");
  WC_CHECK_ARG(!d->gate_rows == !gate, "wc_join_forward: a gate and its rows go together");
  if (int rc = check_stats(post_stats, pre_stats, "wc_join_forward")) return rc;
  JoinArgs a = {d->rows, d->rows / d->samples, d->C, f, x, gate, gate_of(d), d->gate_dtype == WC_F32, d->stream_scale, d->block_scale, norm_of(d->post), norm_of(d->pre),
                drop_of(d), s, y, post_stats, pre_stats};
  if (!y) a.pre.kind = WC_NORM_NONE;
  return join_forward(a, d->dtype, stream);
}

int wc_join_backward_workspace_bytes(const wc_join_desc* d, const wc_join_gradients* q, size_t* bytes) {
  WC_CHECK_ARG(bytes != nullptr && q != nullptr, "wc_join_backward_workspace_bytes: null pointer");
  if (int rc = check_desc(d, "wc_join_backward_workspace_bytes")) return rc;
  *bytes = d->rows == 0 ? 0 : backward_plan(d, q, nullptr).bytes;
  return WC_OK;
}

int wc_join_backward(const wc_join_desc* d, const wc_join_gradients* q, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = wc_join_backward_workspace_bytes(d, q, &need)) return rc;
  WC_CHECK_ARG(d->rows > 0, "wc_join_backward: no rows (the gradients of the parameters are zero)");
  const bool pre = d->pre.kind != WC_NORM_NONE && q->dy, post = d->post.kind != WC_NORM_NONE;
  WC_CHECK_ARG(q->ds || pre, "wc_join_backward: neither ds nor dy with its norm");
  WC_CHECK_ARG(!pre || ((q->s || (q->f && d->dtype != WC_F32)) && q->pre_stats), "wc_join_backward: pre's gradient needs s, or in 16-bit types f, and its statistics");
  WC_CHECK_ARG(!d->gate_rows == !q->gate, "wc_join_backward: a gate and its rows go together");
  WC_CHECK_ARG((!q->dpre_weight && !q->dpre_bias) || pre, "wc_join_backward: gradients of a norm that is not there");
  WC_CHECK_ARG((!q->dpost_weight && !q->dpost_bias) || post, "wc_join_backward: gradients of a norm that is not there");
  WC_CHECK_ARG(!q->dgate || q->gate, "wc_join_backward: the gradient of a gate that is not there");
  WC_CHECK_ARG(!post || q->post_stats, "wc_join_backward: post's gradient needs its statistics");
  WC_CHECK_ARG((!post && !q->dgate) || q->f, "wc_join_backward: post's gradient and the gate's need f");
  if (int rc = check_stats(q->post_stats, q->pre_stats, "wc_join_backward")) return rc;
  if (need && (!workspace || workspace_bytes < need))
    return fail(WC_ERR_WORKSPACE, "wc_join_backward: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return fail(WC_ERR_WORKSPACE, "wc_join_backward: workspace must be 256-byte aligned");
  const Backward b = backward_plan(d, q, static_cast<char*>(workspace));
  if (int rc = join_backward(b.g, d->dtype, stream)) return rc;
  return join_sums(b.sums, b.n, d->C, d->dtype, stream);
}

}  // extern "C"
