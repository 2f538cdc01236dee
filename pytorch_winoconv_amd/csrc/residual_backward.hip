// What a backward pass of residual.h launches: how its rows are shared out, the kernels (residual_backward.inc, a source a type), and the sums of the
// workgroups' parts.
#include "residual.h"

#include <algorithm>

namespace wc {

// Vectors of a thread, wavefronts and lanes of a team of a backward pass; vectors 0: long rows.  One vector a thread up to 8192 channels: the sums and the row
// that is on its way leave no registers for more.  Two, of 16 wavefronts with 128 registers a thread, hold a norm alone and what goes through no norm; the rest spills
// and is left to the passes of long rows (us, in registers | long: 2048 x 16384 bf16 with two norms, gate and dropout 591 | 457; a norm alone 4096 x 16384
// 109 | 225, 4096 x 12001 120 | 282; 2048 x 8001 with two norms, gate and dropout, one vector, 147 | 360)
TeamShape back_shape(const JoinGradients& g) {
  const int vectors = ceil_div(g.C, 8);
  if (vectors <= 64) {
    int lanes = 1;
    while (lanes < vectors) lanes *= 2;
    return {1, 1, lanes};
  }
  for (int waves = 2; waves <= 8; waves *= 2)
    if (vectors <= 64 * waves) return {1, waves, 64};
  if (vectors <= 1024) return {1, 16, 64};
  const bool alone = !g.gate_rows && !g.ds && !g.dx, little = !g.post.kind && (!g.pre.kind || alone);
  if (vectors <= 2048 && little) return {2, 16, 64};
  return {0, 16, 64};
}

void join_plan(JoinGradients* g) {
  const TeamShape t = back_shape(*g);
  const long long teams = t.waves > 1 ? 1 : 256 / t.lanes;
  g->segments = g->gate_rows == kGateSample ? g->rows / g->per : 1;
  const long long length = g->segments > 1 ? g->per : g->rows;
  // Workgroups: what the compute units hold at once (kMinWaves: more would wait for their turn and leave more parts; us, 16384 x 2048 bf16, two norms, gate and
  // dropout, at 8 | 12 | 16 wavefronts a compute unit 135 | 171 | 138, without post and gate 82 | 79 | 74), with two rows a team where there are so many
  const int held = g->post.kind || g->gate_rows == kGateRow ? 8 : g->pre.kind && (g->gate_rows || !g->s) ? 12 : 16;
  // (long rows: parts of at most 256 MB a sum)
  const long long most = t.vectors == 0 ? std::max(1ll, std::min<long long>(kCus, (64ll << 20) / g->C)) : kCus * std::max(1, held / (t.waves == 1 ? 4 : t.waves));
  // (more than four a compute unit only with eight rows each: a second row of parts costs more than it spreads; us, layer norm of 4096 x 1024 bf16, 2048 | 1024
  // workgroups 23.4 | 18.1, 8192 x 1024 24.5 | 21.8, 32768 x 1024 57 with 2048)
  const long long wanted = std::max(1ll, std::min(most, std::max(std::min(4ll * kCus, ceil_div_ll(g->rows, 2 * teams)), ceil_div_ll(g->rows, 8 * teams))));
  g->parts = (int)std::max(1ll, std::min(wanted / g->segments, ceil_div_ll(length, teams)));
  g->blocks = (int)std::min<long long>(g->segments * g->parts, most);
}

int join_backward(const JoinGradients& g, int dtype, void* stream) {
  return dispatch_dtype(dtype, [&](auto t) { return join_backward_of<decltype(t)>(g, stream); });
}

namespace {

// 32 channels by 32 parts a workgroup
struct SumsArgs { JoinSum sum[5]; int n, C, wide_blocks; };
template <typename T>
__global__ __launch_bounds__(1024) void join_sums_kernel(SumsArgs a, long long first) {
  __shared__ float t[32][33];
  long long b = (first + blockIdx.x) / a.wide_blocks;
  const int c0 = (int)((first + blockIdx.x) % a.wide_blocks) * 32;
  int k = 0;
  while (k + 1 < a.n && b >= a.sum[k].segments) b -= a.sum[k++].segments;
  const JoinSum s = a.sum[k];
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, c = min(c0 + col, a.C - 1);
  const float* const from = s.part + b * s.parts * a.C + c;
  float u = 0.f;
  int r = lane;
  // (sixteen on their way at a time: there may be a few workgroups alone, and a thousand parts)
  auto some = [&](auto n) {
    constexpr int N = decltype(n)::value;
    for (; r + 32 * (N - 1) < s.parts; r += 32 * N) {
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = from[(long long)(r + 32 * i) * a.C];
#pragma unroll
      for (int i = 0; i < N; ++i) u += v[i];
    }
  };
  some(ic<16>{});
  some(ic<4>{});
  for (; r < s.parts; r += 32) u += from[(long long)r * a.C];
  t[lane][col] = u;
  __syncthreads();
  if (lane || c0 + col >= a.C) return;
  u = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) u += t[i][col];
  if (s.wide) static_cast<float*>(s.dst)[b * a.C + c] = u;
  else static_cast<T*>(s.dst)[b * a.C + c] = static_cast<T>(u);
}

}  // namespace

int join_sums(const JoinSum* sums, int n, int C, int dtype, void* stream) {
  if (n == 0) return WC_OK;
  SumsArgs a = {};
  long long blocks = 0;
  a.n = n;
  a.C = C;
  a.wide_blocks = ceil_div(C, 32);
  for (int k = 0; k < n; ++k) {
    a.sum[k] = sums[k];
    blocks += sums[k].segments * a.wide_blocks;
  }
  return dispatch_dtype(dtype, [&](auto t) {
    return in_launches(blocks, [&](long long first, unsigned count) -> int {
      hipLaunchKernelGGL((join_sums_kernel<decltype(t)>), dim3(count), dim3(1024), 0, as_stream(stream), a, first);
      WC_CHECK_LAUNCH("join_sums_kernel");
      return WC_OK;
    }, kMostBlocks / 2);
  });
}

}  // namespace wc
