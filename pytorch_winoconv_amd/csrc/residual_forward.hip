// s = a x + b g drop(post(f)) and y = pre(s) of residual.h, a row a team at a time: one read of f and x, one write of s and y, whatever of it there is.
#include "residual.h"

namespace wc {

namespace {

// (v - mean) / deviation, in place; zeros behind `have`
template <int NV, int WAVES>
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
      v[i][e] = e < have[i] ? v[i][e] - mean : 0.f;
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

template <typename T, int NV, int WAVES>
__global__ __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256) void join_kernel(JoinArgs a, int lanes, long long first_block) {
  __shared__ float meet[WAVES > 1 ? 4 * WAVES : 1];
  const int width = WAVES > 1 ? 64 * WAVES : lanes, slot = threadIdx.x & (width - 1);
  const long long row = (first_block + blockIdx.x) * (WAVES > 1 ? 1 : 256 / lanes) + (WAVES > 1 ? 0 : threadIdx.x / lanes);
  const bool there = row < a.rows;             // (lanes of other teams of the wavefront go on, and it takes them for its exchanges)
  Team<WAVES> team = {lanes, meet, 0};
  int c[NV], have[NV];
  float v[NV][8], r[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    c[i] = (i * width + slot) * 8;
    have[i] = there ? max(min(a.C - c[i], 8), 0) : 0;
    load_floats<T>(a.f, row * a.C + c[i], have[i], v[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.x) {
      load_floats<T>(a.x, row * a.C + c[i], have[i], r[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[i][e] = 0.f;
    }
  }
  if (a.post.kind) {
    normalise<NV, WAVES>(team, v, have, a.post, a.C, a.post_stats, row, slot == 0 && there);
#pragma unroll
    for (int i = 0; i < NV; ++i) scale_shift<T>(a.post, c[i], have[i], v[i]);
  }
  if (a.drop.level) {
    const Keys k = keys_of(a.drop);
    const unsigned all = a.drop.per_sample ? kept_sample(a.drop, k, (unsigned)row / (unsigned)a.per) : 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const unsigned kept = a.drop.per_sample ? all : kept8(a.drop, k, (unsigned)c[i] / 8, (unsigned)row);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = kept >> e & 1 ? v[i][e] * a.drop.scale : 0.f;
    }
  }
  const long long g0 = a.gate_rows ? gate_row(a.gate_rows, row, a.per) * a.C : 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.gate_rows) {
      float g[8];
      load_parameter<T>(a.gate, a.gate_wide, g0 + c[i], have[i], g, 0.f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] *= a.b;
    if (a.x) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = fmaf(a.a, r[i][e], v[i][e]);
    }
    if (a.s) store_floats<T>(a.s, row * a.C + c[i], have[i], v[i]);
  }
  if (!a.pre.kind) return;
  // (of s before its rounding)
  normalise<NV, WAVES>(team, v, have, a.pre, a.C, a.pre_stats, row, slot == 0 && there);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    scale_shift<T>(a.pre, c[i], have[i], v[i]);
    store_floats<T>(a.y, row * a.C + c[i], have[i], v[i]);
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
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto go = [&](auto nv, auto waves, int lanes) {
      constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value;
      return in_launches(WAVES > 1 ? a.rows : ceil_div_ll(a.rows, 256 / lanes), [&](long long first, unsigned blocks) -> int {
        hipLaunchKernelGGL((join_kernel<T, NV, WAVES>), dim3(blocks), dim3(WAVES > 1 ? 64 * WAVES : 256), 0, as_stream(stream), a, lanes, first);
        WC_CHECK_LAUNCH("join_kernel");
        return WC_OK;
      }, kMostBlocks / 2);
    };
    // a wavefront a row waits for nobody; few rows are over sooner with more threads each
    const bool many = a.rows >= 4 * kCus;
    if (vectors <= 64) {
      int lanes = 1;
      while (lanes < vectors) lanes *= 2;
      return go(ic<1>{}, ic<1>{}, lanes);
    }
    if (vectors <= 128 && many) return go(ic<2>{}, ic<1>{}, 64);
    if (vectors <= 256 && many) return go(ic<4>{}, ic<1>{}, 64);
    if (vectors <= 256) return go(ic<1>{}, ic<4>{}, 64);
    if (vectors <= 512) return go(ic<2>{}, ic<4>{}, 64);
    if (vectors <= 1024) return go(ic<4>{}, ic<4>{}, 64);
    if (vectors <= 4096) return go(ic<4>{}, ic<16>{}, 64);
    return in_launches(a.rows, [&](long long first, unsigned blocks) -> int {
      hipLaunchKernelGGL((join_long_kernel<T>), dim3(blocks), dim3(kLong), 0, as_stream(stream), a, first);
      WC_CHECK_LAUNCH("join_long_kernel");
      return WC_OK;
    }, kMostBlocks / 2);
  });
}

}  // namespace wc
