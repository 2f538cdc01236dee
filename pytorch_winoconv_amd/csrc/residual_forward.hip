// s = a x + b g drop(post(f)) and y = pre(s) of residual.h, a row a team at a time: one read of f and x, one write of s and y, whatever of it there is.
// Bound by memory: us and TB/s, fp16 layer norm of 200704 x 256 37 (5.6), bf16 RMS norm of 16384 x 4096 48 (5.6), dropout of 8192 x 8192 51 (5.2; inputs from memory 59); two norms,
// gate and dropout of 16384 x 2048 57 (4.7), whose arithmetic takes about as long.
#include "residual.h"

#include <algorithm>

namespace wc {

namespace {

// (v - mean) / deviation, in place; zeros behind `have`
template <int ROW, int NV, int WAVES>
__device__ __forceinline__ void normalise(Team<WAVES>& team, float (&v)[NV][8], const int (&have)[NV], const Norm& n, int C, float* stats, long long row, bool first) {
  float mean = 0.f;
  if (n.kind == WC_NORM_LAYER) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) t += v[i][e];
    mean = team.sum(t) / C;
  }
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[i][e] = kept_element<ROW>(v[i][e] - (have[i] ? mean : 0.f), e, have[i]);
      t = fmaf(v[i][e], v[i][e], t);
    }
  const float inverse = 1.f / sqrtf(team.sum(t) / C + n.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] *= inverse;
  if (stats && first) *reinterpret_cast<float2*>(stats + 2 * row) = float2{mean, inverse};
}

template <typename T>
__device__ __forceinline__ void scale_shift(const Norm& n, int c, int have, float (&v)[8]) {
  float w[8], b[8];
  load_parameter<T>(n.weight, n.wide, c, have, w, 1.f);
  load_parameter<T>(n.bias, n.wide, c, have, b, 0.f);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e], w[e], b[e]);
}

// Rows block, block + blocks, ... a team; one vector a thread: the next row is on its way while one is worked on, and the parameters stay in registers.  Without a
// norm two wavefronts take one of the `pieces` of a row, neighbouring workgroups those of one row
template <typename T, int NV, int WAVES, int ROW, bool AHEAD, bool ALONE>
__global__ __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256) void join_kernel(JoinArgs a, int lanes, int pieces) {
  __shared__ float meet[WAVES > 1 ? 4 * WAVES : 1];
  const int width = WAVES > 1 ? 64 * WAVES : lanes, slot = threadIdx.x & (width - 1), teams = WAVES > 1 ? 1 : 256 / lanes;
  constexpr bool SPLIT = AHEAD && !ALONE && WAVES == 2;
  const unsigned block = SPLIT ? blockIdx.x / (unsigned)pieces : blockIdx.x, piece = SPLIT ? blockIdx.x % (unsigned)pieces : 0u;
  const long long step = (long long)(SPLIT ? gridDim.x / (unsigned)pieces : gridDim.x) * teams;
  Team<WAVES> team = {lanes, meet, 0};
  const Keys keys = !ALONE && a.drop.level ? keys_of(a.drop) : Keys{0, 0};
  int c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) c[i] = (((int)piece * NV + i) * width + slot) * 8;
  Raw8<T> f[NV], x[NV];
  auto load = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) f[i] = load8<T, ROW>(a.f, row, c[i], a.C, row < a.rows);
    if (!ALONE && a.x) {
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i] = load8<T, ROW>(a.x, row, c[i], a.C, row < a.rows);
    }
  };
  constexpr int KEPT = AHEAD ? NV : 1;
  float post_w[KEPT][8], post_b[KEPT][8], pre_w[KEPT][8], pre_b[KEPT][8], gate[KEPT][8];
  auto parameters = [&](const Norm& n, int c, float (&w)[8], float (&b)[8]) {
    parameter8<T, ROW>(n.weight, n.wide, 0, c, a.C, w, 1.f);
    parameter8<T, ROW>(n.bias, n.wide, 0, c, a.C, b, 0.f);
  };
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      if (!ALONE && a.post.kind) parameters(a.post, c[i], post_w[i], post_b[i]);
      if (a.pre.kind) parameters(a.pre, c[i], pre_w[i], pre_b[i]);
      if (!ALONE && a.gate_rows == kGateChannel) parameter8<T, ROW>(a.gate, a.gate_wide, 0, c[i], a.C, gate[i], 0.f);
    }
    load((long long)block * teams + threadIdx.x / width);
  }
  for (long long base = (long long)block * teams; base < a.rows; base += step) {
    const long long row = base + (WAVES > 1 ? 0 : threadIdx.x / lanes);
    const bool there = row < a.rows;           // (lanes of other teams of the wavefront go on, and it takes them for its exchanges)
    if constexpr (!AHEAD) load(row);
    int have[NV];
    float v[NV][8], r[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      have[i] = there ? max(min(a.C - c[i], 8), 0) : 0;
      asm volatile("" : "+v"(have[i]));
      floats_of<T>(settled8<T, ROW>(f[i], c[i], a.C, there), v[i]);
      if (!ALONE && a.x) floats_of<T>(settled8<T, ROW>(x[i], c[i], a.C, there), r[i]);
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[i][e] = 0.f;
      }
    }
    if constexpr (AHEAD) {
      if (base + step < a.rows) load(row + step);
    }
    if (!ALONE && a.post.kind) {
      normalise<ROW, NV, WAVES>(team, v, have, a.post, a.C, a.post_stats, row, slot == 0 && there);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = AHEAD ? i : 0;
        if constexpr (!AHEAD) parameters(a.post, c[i], post_w[k], post_b[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = fmaf(v[i][e], post_w[k][e], post_b[k][e]);
      }
    }
    if (!ALONE && a.drop.level) {
      const unsigned all = a.drop.per_sample ? kept_sample(a.drop, keys, (unsigned)row / (unsigned)a.per) : 0u;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned kept = a.drop.per_sample ? all : kept8(a.drop, keys, (unsigned)c[i] / 8, (unsigned)row);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = kept >> e & 1 ? v[i][e] * a.drop.scale : 0.f;
      }
    }
    const long long g0 = !ALONE && a.gate_rows && there ? gate_row(a.gate_rows, row, a.per) : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!ALONE && a.gate_rows) {
        const int k = AHEAD ? i : 0;
        if (!AHEAD || a.gate_rows != kGateChannel) parameter8<T, ROW>(a.gate, a.gate_wide, g0, c[i], a.C, gate[k], 0.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= gate[k][e];
      }
      if (!ALONE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= a.b;
      }
      if (!ALONE && a.x) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = fmaf(a.a, r[i][e], v[i][e]);
      }
      if (!ALONE && a.s) store_floats<T>(a.s, row * a.C + c[i], have[i], v[i]);
    }
    if (!ALONE && !a.pre.kind) continue;
    // (of s before its rounding)
    normalise<ROW, NV, WAVES>(team, v, have, a.pre, a.C, a.pre_stats, row, slot == 0 && there);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = AHEAD ? i : 0;
      if constexpr (!AHEAD) parameters(a.pre, c[i], pre_w[k], pre_b[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = fmaf(v[i][e], pre_w[k][e], pre_b[k][e]);
      store_floats<T>(a.y, row * a.C + c[i], have[i], v[i]);
    }
  }
}

// Rows of more channels than a workgroup's registers hold: passes over f and x, a workgroup a row
constexpr int kLong = 1024;
template <typename T>
__global__ __launch_bounds__(kLong) void join_long_kernel(JoinArgs a, long long first_block) {
  __shared__ float meet[4 * kLong / 64];
  const long long row = first_block + blockIdx.x;
  Team<kLong / 64> team = {64, meet, 0};
  const Keys k = a.drop.level ? keys_of(a.drop) : Keys{0, 0};
  const unsigned all = a.drop.level && a.drop.per_sample ? kept_sample(a.drop, k, (unsigned)row / (unsigned)a.per) : 0u;
  const long long g0 = a.gate_rows ? gate_row(a.gate_rows, row, a.per) * a.C : 0;
  float post_mean = 0.f, post_inverse = 1.f, pre_mean = 0.f, pre_inverse = 1.f;
  auto f_at = [&](int c, int have, float (&v)[8]) {
    load_floats<T>(a.f, row * a.C + c, have, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < have ? (v[e] - post_mean) * post_inverse : 0.f;
  };
  auto s_at = [&](int c, int have, float (&v)[8]) {
    f_at(c, have, v);
    if (a.post.kind) scale_shift<T>(a.post, c, have, v);
    if (a.drop.level) {
      const unsigned kept = a.drop.per_sample ? all : kept8(a.drop, k, (unsigned)c / 8, (unsigned)row);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = kept >> e & 1 ? v[e] * a.drop.scale : 0.f;
    }
    float g[8], x[8];
    if (a.gate_rows) {
      load_parameter<T>(a.gate, a.gate_wide, g0 + c, have, g, 0.f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= a.b;
    if (a.x) {
      load_floats<T>(a.x, row * a.C + c, have, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(a.a, x[e], v[e]);
    }
  };
  auto over = [&](auto&& at) {
    for (int c = threadIdx.x * 8; c < a.C; c += kLong * 8) at(c, min(a.C - c, 8));
  };
  auto statistics = [&](const Norm& n, auto&& values, float& mean, float& inverse, float* stats) {
    float m = 0.f, v[8];
    if (n.kind == WC_NORM_LAYER) {
      float t = 0.f;
      over([&](int c, int have) {
        values(c, have, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) t += e < have ? v[e] : 0.f;
      });
      m = team.sum(t) / a.C;
    }
    float t = 0.f;
    over([&](int c, int have) {
      values(c, have, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) t = e < have ? fmaf(v[e] - m, v[e] - m, t) : t;
    });
    t = 1.f / sqrtf(team.sum(t) / a.C + n.eps);
    mean = m;
    inverse = t;
    if (stats && threadIdx.x == 0) *reinterpret_cast<float2*>(stats + 2 * row) = float2{m, t};
  };
  if (a.post.kind) statistics(a.post, f_at, post_mean, post_inverse, a.post_stats);
  if (a.pre.kind) statistics(a.pre, s_at, pre_mean, pre_inverse, a.pre_stats);
  over([&](int c, int have) {
    float v[8];
    s_at(c, have, v);
    if (a.s) store_floats<T>(a.s, row * a.C + c, have, v);
    if (!a.pre.kind) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (v[e] - pre_mean) * pre_inverse;
    scale_shift<T>(a.pre, c, have, v);
    store_floats<T>(a.y, row * a.C + c, have, v);
  });
}

}  // namespace

int join_forward(const JoinArgs& a, int dtype, void* stream) {
  const int vectors = ceil_div(a.C, 8);
  const bool even = a.C % 8 == 0;
  const bool alone = a.pre.kind && !a.post.kind && !a.x && !a.gate_rows && !a.drop.level && !a.s && a.b == 1.f;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    // as many workgroups as the compute units hold at once, or as there are rows; of two wavefronts, which end soon, four times as many (us, inputs from memory,
    // one | four times: dropout of 8192 x 8192 bf16 64 | 59, with a stream 86 | 78; 60000 x 1000 fp16 with two norms, gate and dropout 137 | 129.  Of more wavefronts
    // 8192 x 4096 takes 65 | 72, of less 200704 x 256 101 | 103)
    auto go = [&](auto nv, auto waves, auto ahead, int lanes, int pieces = 1) -> int {
      constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value, THREADS = WAVES > 1 ? 64 * WAVES : 256;
      constexpr bool AHEAD = decltype(ahead)::value;
      const long long wanted = WAVES > 1 ? a.rows : ceil_div_ll(a.rows, 256 / lanes), most = AHEAD ? std::max(1, kCus * (2048 / THREADS) * (WAVES == 2 ? 4 : 1) / pieces) : kMostBlocks / 2;
      // (what is there of a form: two vectors a thread of even rows alone, and of joins in 16 wavefronts alone)
      auto fn = alone ? &join_kernel<T, NV, WAVES, kEven, AHEAD, true> : &join_kernel<T, NV, WAVES, kEven, AHEAD, NV == 2 && WAVES < 16>;
      if constexpr (NV == 1) {
        if (!even) fn = alone ? &join_kernel<T, NV, WAVES, kOdd, AHEAD, true> : &join_kernel<T, NV, WAVES, kOdd, AHEAD, false>;
      }
      if constexpr (NV == 1 && WAVES == 1) {
        if (a.C < 8) fn = alone ? &join_kernel<T, NV, WAVES, kTiny, AHEAD, true> : &join_kernel<T, NV, WAVES, kTiny, AHEAD, false>;
      }
      hipLaunchKernelGGL(fn, dim3((unsigned)((wanted < most ? wanted : most) * pieces)), dim3(THREADS), 0, as_stream(stream), a, lanes, pieces);
      WC_CHECK_LAUNCH("join_kernel");
      return WC_OK;
    };
    const std::true_type ahead;
    const std::false_type whole;
    if (vectors <= 64) {
      int lanes = 1;
      while (lanes < vectors) lanes *= 2;
      return go(ic<1>{}, ic<1>{}, ahead, lanes);
    }
    // Without a norm nothing is wanted of a whole row: pieces of 1024 channels (us, dropout of 8192 x 8192 bf16 59, in whole rows 66)
    if (!a.post.kind && !a.pre.kind) return go(ic<1>{}, ic<2>{}, ahead, 64, ceil_div(vectors, 128));
    // A norm alone of even rows takes two vectors a thread and every row a workgroup of its own: there is little to keep in registers, and fewer wait at a barrier
    // (us, bf16 rms, two | one ahead: 65536 x 1024 46.9 | 47.3, 16384 x 4096 46.0 | 49.3, 8192 x 8192 45.2 | 57.8).  Joins the other way about (8192 x 4096 76 | 63)
    if (alone && even) {
      if (vectors <= 128) return go(ic<2>{}, ic<1>{}, whole, 64);
      if (vectors <= 256) return go(ic<2>{}, ic<2>{}, whole, 64);
      if (vectors <= 512) return go(ic<2>{}, ic<4>{}, whole, 64);
      if (vectors <= 1024) return go(ic<2>{}, ic<8>{}, whole, 64);
    } else {
      if (vectors <= 128) return go(ic<1>{}, ic<2>{}, ahead, 64);
      if (vectors <= 256) return go(ic<1>{}, ic<4>{}, ahead, 64);
      if (vectors <= 512) return go(ic<1>{}, ic<8>{}, ahead, 64);
      if (vectors <= 1024) return go(ic<1>{}, ic<16>{}, ahead, 64);
    }
    // (two vectors of odd rows spill in 16 wavefronts; us, 2048 x 12001 bf16 with two norms, gate and dropout, in registers | long: 602 | 171)
    if (vectors <= 2048 && even) return go(ic<2>{}, ic<16>{}, whole, 64);
    return in_launches(a.rows, [&](long long first, unsigned blocks) -> int {
      hipLaunchKernelGGL((join_long_kernel<T>), dim3(blocks), dim3(kLong), 0, as_stream(stream), a, first);
      WC_CHECK_LAUNCH("join_long_kernel");
      return WC_OK;
    }, kMostBlocks / 2);
  });
}

}  // namespace wc
