// The gradients of residual.h in one pass over the rows: ds, dy, s and f are read once, df and dx written once, a row in a team's registers as in the
// forward pass; the mask is drawn again.
//
//   dr = ds + (dh - mean(dh) - s^ mean(dh s^)) / dev_s,   dh = dy w_pre,  s^ = (s - mean) / dev_s   (RMS: without the first mean)
//   dx = a dr,   dd = b dr,   dg += dd d,   dv = g drop'(dd),   df = the same of dv through post
//
// The sums over rows (dw += dy s^, db += dy, of either norm, and dg) stay in the registers of the threads that hold those channels, from row to
// row of a workgroup's share; then the teams of a workgroup add up in LDS, and a second launch adds the workgroups', in a fixed order.
#include "residual.h"

#include <algorithm>

namespace wc {

namespace {

constexpr int kSums = 5;

template <int NV> using Row = float[NV][8];

// (dh - mean(dh) - v mean(dh v)) times inverse, in place of dh; v normalised
template <int NV, int WAVES>
__device__ __forceinline__ void through_norm(Team<WAVES>& team, Row<NV>& dh, const Row<NV>& v, int kind, int C, float inverse) {
  float t = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t += dh[i][e];
      u = fmaf(dh[i][e], v[i][e], u);
    }
  if (kind == WC_NORM_LAYER) team.sum(t, u);
  else {
    t = 0.f;
    u = team.sum(u);
  }
  t /= C;
  u /= C;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dh[i][e] = (dh[i][e] - t - v[i][e] * u) * inverse;
}

template <typename T, int NV, int WAVES, bool PRE, bool POST>
__global__ __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256) void join_back_kernel(JoinGradients g, int lanes) {
  constexpr int THREADS = WAVES > 1 ? 64 * WAVES : 256;
  __shared__ float meet[WAVES > 1 ? 4 * WAVES : 1];
  __shared__ float rows_of_sums[WAVES > 1 ? 1 : THREADS * 8 * NV];
  const int width = WAVES > 1 ? THREADS : lanes, teams = THREADS / width, slot = threadIdx.x & (width - 1), mine = threadIdx.x / width;
  Team<WAVES> team = {lanes, meet, 0};
  const Keys keys = g.drop.level ? keys_of(g.drop) : Keys{0, 0};
  const bool gate_sums = g.part[kGateSum] != nullptr, need_f = POST || gate_sums || g.dgate_rows;
  int c[NV], have_c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    c[i] = (i * width + slot) * 8;
    have_c[i] = max(min(g.C - c[i], 8), 0);
  }
  float acc[kSums][NV][8];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[k][i][e] = 0.f;

  // the workgroup's sums of one kind, to row `at` of its parts
  auto give = [&](auto kk, long long at) {
    constexpr int K = decltype(kk)::value;
    float* const part = g.part[K];
    if (!part) return;
    if constexpr (WAVES > 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) store_run<float, 8>(part, at * g.C + c[i], have_c[i], acc[K][i]);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) rows_of_sums[(mine * NV + i) * width * 8 + slot * 8 + e] = acc[K][i][e];
      __syncthreads();
      const int row = NV * width * 8;
      for (int j = threadIdx.x; j < row && j < g.C; j += THREADS) {
        float t = 0.f;
        for (int m = 0; m < teams; ++m) t += rows_of_sums[m * row + j];
        part[at * g.C + j] = t;
      }
    }
  };

  const long long length = g.segments > 1 ? g.per : g.rows;
  for (long long w = blockIdx.x; w < g.segments * g.parts; w += g.blocks) {
    const long long segment = w / g.parts, part = w - segment * g.parts;
    const long long begin = segment * length + part * length / g.parts, end = segment * length + (part + 1) * length / g.parts;
    for (long long base = begin; base < end; base += teams) {
      const long long row = base + mine;
      const bool there = row < end;
      const long long at = row * g.C;
      int have[NV];
      float dr[NV][8], v[NV][8];
      T f[NV][8];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        have[i] = there ? have_c[i] : 0;
        if (g.ds) load_floats<T>(g.ds, at + c[i], have[i], dr[i]);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) dr[i][e] = 0.f;
        }
      }
      if (need_f) {
#pragma unroll
        for (int i = 0; i < NV; ++i) load_run<T, 8>(g.f, at + c[i], have[i], f[i]);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[i][e] = static_cast<T>(0.f);
      }
      if constexpr (PRE) {
        float dh[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          load_floats<T>(g.dy, at + c[i], have[i], dh[i]);
          load_floats<T>(g.s, at + c[i], have[i], v[i]);
        }
        const float2 st = there ? *reinterpret_cast<const float2*>(g.pre_stats + 2 * row) : float2{0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float wt[8];
          load_parameter<T>(g.pre.weight, g.pre.wide, c[i], have[i], wt, 1.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[i][e] = e < have[i] ? (v[i][e] - st.x) * st.y : 0.f;
            acc[kPreWeight][i][e] = fmaf(dh[i][e], v[i][e], acc[kPreWeight][i][e]);
            acc[kPreBias][i][e] += dh[i][e];
            dh[i][e] *= wt[e];
          }
        }
        through_norm<NV, WAVES>(team, dh, v, g.pre.kind, g.C, st.y);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) dr[i][e] = e < have[i] ? dr[i][e] + dh[i][e] : 0.f;
      }
      if (g.dx) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = g.a * dr[i][e];
          store_floats<T>(g.dx, at + c[i], have[i], o);
        }
      }
      if (!g.df && !need_f) continue;
      const float2 st = POST && there ? *reinterpret_cast<const float2*>(g.post_stats + 2 * row) : float2{0.f, 0.f};
      const long long g0 = g.gate_rows ? gate_row(g.gate_rows, row, g.per) * g.C : 0;
      const unsigned all = g.drop.level && g.drop.per_sample ? kept_sample(g.drop, keys, (unsigned)row / (unsigned)g.per) : 255u;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        unsigned kept = all;
        if (g.drop.level && !g.drop.per_sample) kept = kept8(g.drop, keys, (unsigned)c[i] / 8, (unsigned)row);
        float wt[8];
        if constexpr (POST) load_parameter<T>(g.post.weight, g.post.wide, c[i], have[i], wt, 1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[i][e] = static_cast<float>(f[i][e]);
          if constexpr (POST) v[i][e] = e < have[i] ? (v[i][e] - st.x) * st.y : 0.f;
          dr[i][e] *= g.b;
        }
        if (g.gate_rows) {
          float gt[8], dg[8];
          if (need_f) {
            float b[8];
            if constexpr (POST) load_parameter<T>(g.post.bias, g.post.wide, c[i], have[i], b, 0.f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float n = POST ? fmaf(v[i][e], wt[e], b[e]) : v[i][e];
              dg[e] = kept >> e & 1 ? dr[i][e] * (n * g.drop.scale) : 0.f;
            }
            if (g.dgate_rows) {
              if (g.gate_wide) store_run<float, 8>(g.dgate_rows, at + c[i], have[i], dg);
              else store_floats<T>(g.dgate_rows, at + c[i], have[i], dg);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) acc[kGateSum][i][e] += dg[e];
            }
          }
          load_parameter<T>(g.gate, g.gate_wide, g0 + c[i], have[i], gt, 0.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) dr[i][e] *= gt[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) dr[i][e] = kept >> e & 1 ? dr[i][e] * g.drop.scale : 0.f;
        if constexpr (POST) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            acc[kPostWeight][i][e] = fmaf(dr[i][e], v[i][e], acc[kPostWeight][i][e]);
            acc[kPostBias][i][e] += dr[i][e];
            dr[i][e] *= wt[e];
          }
        }
      }
      if constexpr (POST) through_norm<NV, WAVES>(team, dr, v, g.post.kind, g.C, st.y);
      if (g.df) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store_floats<T>(g.df, at + c[i], have[i], dr[i]);
      }
    }
    if (gate_sums) {
      give(ic<kGateSum>{}, w);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[kGateSum][i][e] = 0.f;
    }
  }
  if constexpr (PRE) {
    give(ic<kPreWeight>{}, blockIdx.x);
    give(ic<kPreBias>{}, blockIdx.x);
  }
  if constexpr (POST) {
    give(ic<kPostWeight>{}, blockIdx.x);
    give(ic<kPostBias>{}, blockIdx.x);
  }
}

// Rows of more channels than that: three passes over a row, which come from the L2, a workgroup's sums in its row of the parts
constexpr int kLong = 1024;
template <typename T>
__global__ __launch_bounds__(kLong) void join_back_long_kernel(JoinGradients g) {
  __shared__ float meet[4 * kLong / 64];
  Team<kLong / 64> team = {64, meet, 0};
  const Keys keys = g.drop.level ? keys_of(g.drop) : Keys{0, 0};
  const bool gate_sums = g.part[kGateSum] != nullptr;
  const long long length = g.segments > 1 ? g.per : g.rows;
  auto over = [&](auto&& at) {
    for (int c = threadIdx.x * 8; c < g.C; c += kLong * 8) at(c, min(g.C - c, 8));
  };
  // sums of channels that this thread alone holds
  auto add = [&](int k, long long row, bool first, int c, int have, const float (&v)[8]) {
    if (!g.part[k]) return;
    float t[8];
    if (first) {
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = v[e];
    } else {
      load_run<float, 8>(g.part[k], row * g.C + c, have, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] += v[e];
    }
    store_run<float, 8>(g.part[k], row * g.C + c, have, t);
  };
  bool first = true;
  for (long long w = blockIdx.x; w < g.segments * g.parts; w += g.blocks) {
    const long long segment = w / g.parts, part = w - segment * g.parts;
    const long long begin = segment * length + part * length / g.parts, end = segment * length + (part + 1) * length / g.parts;
    for (long long row = begin; row < end; ++row, first = false) {
      const long long at = row * g.C;
      const float2 pre = g.pre.kind ? *reinterpret_cast<const float2*>(g.pre_stats + 2 * row) : float2{0.f, 1.f};
      const float2 post = g.post.kind ? *reinterpret_cast<const float2*>(g.post_stats + 2 * row) : float2{0.f, 1.f};
      const long long g0 = g.gate_rows ? gate_row(g.gate_rows, row, g.per) * g.C : 0;
      const unsigned all = g.drop.level && g.drop.per_sample ? kept_sample(g.drop, keys, (unsigned)row / (unsigned)g.per) : 255u;
      float pre_t = 0.f, pre_u = 0.f;
      auto hat = [&](const void* p, const float2& st, int c, int have, float (&v)[8]) {
        load_floats<T>(p, at + c, have, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < have ? (v[e] - st.x) * st.y : 0.f;
      };
      if (g.pre.kind) {
        over([&](int c, int have) {
          float dh[8], v[8], wt[8], dw[8];
          load_floats<T>(g.dy, at + c, have, dh);
          hat(g.s, pre, c, have, v);
          load_parameter<T>(g.pre.weight, g.pre.wide, c, have, wt, 1.f);
          add(kPreBias, blockIdx.x, first, c, have, dh);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dw[e] = dh[e] * v[e];
            pre_t += dh[e] * wt[e];
            pre_u = fmaf(dh[e] * wt[e], v[e], pre_u);
          }
          add(kPreWeight, blockIdx.x, first, c, have, dw);
        });
        team.sum(pre_t, pre_u);
        pre_t = g.pre.kind == WC_NORM_LAYER ? pre_t / g.C : 0.f;
        pre_u /= g.C;
      }
      auto dr_at = [&](int c, int have, float (&dr)[8]) {
        load_parameter<T>(g.ds, 0, at + c, have, dr, 0.f);
        if (!g.pre.kind) return;
        float dh[8], v[8], wt[8];
        load_floats<T>(g.dy, at + c, have, dh);
        hat(g.s, pre, c, have, v);
        load_parameter<T>(g.pre.weight, g.pre.wide, c, have, wt, 1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) dr[e] += (dh[e] * wt[e] - pre_t - v[e] * pre_u) * pre.y;
      };
      // the gradient of what post gave, and, `sums`, the gate's
      auto dv_at = [&](int c, int have, bool sums, const float (&v)[8], float (&dv)[8]) {
        dr_at(c, have, dv);
        unsigned kept = all;
        if (g.drop.level && !g.drop.per_sample) kept = kept8(g.drop, keys, (unsigned)c / 8, (unsigned)row);
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] = e < have ? dv[e] * g.b : 0.f;
        if (g.gate_rows) {
          float gt[8];
          load_parameter<T>(g.gate, g.gate_wide, g0 + c, have, gt, 0.f);
          if (sums && (gate_sums || g.dgate_rows)) {
            float wt[8], b[8], dg[8];
            load_parameter<T>(g.post.weight, g.post.wide, c, have, wt, 1.f);
            load_parameter<T>(g.post.bias, g.post.wide, c, have, b, 0.f);
#pragma unroll
            for (int e = 0; e < 8; ++e) dg[e] = kept >> e & 1 ? dv[e] * (fmaf(v[e], wt[e], b[e]) * g.drop.scale) : 0.f;
            if (gate_sums) add(kGateSum, w, row == begin, c, have, dg);
            else if (g.gate_wide) store_run<float, 8>(g.dgate_rows, at + c, have, dg);
            else store_floats<T>(g.dgate_rows, at + c, have, dg);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) dv[e] *= gt[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] = kept >> e & 1 ? dv[e] * g.drop.scale : 0.f;
      };
      const bool need_f = g.post.kind || gate_sums || g.dgate_rows;
      float post_t = 0.f, post_u = 0.f;
      over([&](int c, int have) {
        if (g.dx) {
          float o[8];
          dr_at(c, have, o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] *= g.a;
          store_floats<T>(g.dx, at + c, have, o);
        }
        if (!g.df && !need_f) return;
        float v[8], dv[8];
        if (need_f) hat(g.f, post, c, have, v);
        dv_at(c, have, true, v, dv);
        if (!g.post.kind) {
          if (g.df) store_floats<T>(g.df, at + c, have, dv);
          return;
        }
        float wt[8], dw[8];
        load_parameter<T>(g.post.weight, g.post.wide, c, have, wt, 1.f);
        add(kPostBias, blockIdx.x, first, c, have, dv);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dw[e] = dv[e] * v[e];
          post_t += dv[e] * wt[e];
          post_u = fmaf(dv[e] * wt[e], v[e], post_u);
        }
        add(kPostWeight, blockIdx.x, first, c, have, dw);
      });
      if (!g.post.kind) continue;
      team.sum(post_t, post_u);
      if (!g.df) continue;
      post_t = g.post.kind == WC_NORM_LAYER ? post_t / g.C : 0.f;
      post_u /= g.C;
      over([&](int c, int have) {
        float v[8], dv[8], wt[8];
        hat(g.f, post, c, have, v);
        dv_at(c, have, false, v, dv);
        load_parameter<T>(g.post.weight, g.post.wide, c, have, wt, 1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] = (dv[e] * wt[e] - post_t - v[e] * post_u) * post.y;
        store_floats<T>(g.df, at + c, have, dv);
      });
    }
  }
}

// 32 channels by 32 parts a workgroup
struct SumsArgs { JoinSum sum[kSums]; int n, C, wide_blocks; };
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
  for (; r + 96 < s.parts; r += 128) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = from[(long long)(r + 32 * i) * a.C];
#pragma unroll
    for (int i = 0; i < 4; ++i) u += v[i];
  }
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

// Vectors of a thread, wavefronts and lanes of a team of a backward pass; vectors 0: long rows
TeamShape back_shape(int C) {
  const int vectors = ceil_div(C, 8);
  if (vectors <= 64) {
    int lanes = 1;
    while (lanes < vectors) lanes *= 2;
    return {1, 1, lanes};
  }
  if (vectors <= 128) return {2, 1, 64};
  if (vectors <= 512) return {2, 4, 64};
  if (vectors <= 1024) return {2, 8, 64};
  return {0, 16, 64};
}

}  // namespace

void join_plan(JoinGradients* g, bool gate_sums) {
  const TeamShape t = back_shape(g->C);
  const long long teams = t.waves > 1 ? 1 : 256 / t.lanes;
  g->segments = g->gate_rows == kGateSample && gate_sums ? g->rows / g->per : 1;
  const long long length = g->segments > 1 ? g->per : g->rows;
  // workgroups: what the compute units hold at once, with four rows a team where there are so many
  const long long most = t.vectors == 0 ? kCus : t.waves > 4 ? kCus : 2 * kCus;
  const long long wanted = std::max(1ll, std::min(most, ceil_div_ll(g->rows, 4 * teams)));
  g->parts = (int)std::max(1ll, std::min(wanted / g->segments, ceil_div_ll(length, teams)));
  g->blocks = (int)std::min<long long>(g->segments * g->parts, most);
}

int join_backward(const JoinGradients& g, int dtype, void* stream) {
  const TeamShape shape = back_shape(g.C);
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (shape.vectors == 0) {
      hipLaunchKernelGGL((join_back_long_kernel<T>), dim3((unsigned)g.blocks), dim3(kLong), 0, as_stream(stream), g);
      WC_CHECK_LAUNCH("join_back_long_kernel");
      return WC_OK;
    }
    auto norms = [&](auto nv, auto waves, auto pre, auto post) -> int {
      constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value;
      hipLaunchKernelGGL((join_back_kernel<T, NV, WAVES, decltype(pre)::value, decltype(post)::value>), dim3((unsigned)g.blocks), dim3(WAVES > 1 ? 64 * WAVES : 256), 0,
                         as_stream(stream), g, shape.lanes);
      WC_CHECK_LAUNCH("join_back_kernel");
      return WC_OK;
    };
    auto go = [&](auto nv, auto waves) {
      if (g.pre.kind) return g.post.kind ? norms(nv, waves, std::true_type{}, std::true_type{}) : norms(nv, waves, std::true_type{}, std::false_type{});
      return g.post.kind ? norms(nv, waves, std::false_type{}, std::true_type{}) : norms(nv, waves, std::false_type{}, std::false_type{});
    };
    if (shape.waves == 8) return go(ic<2>{}, ic<8>{});
    if (shape.waves == 4) return go(ic<2>{}, ic<4>{});
    return shape.vectors == 2 ? go(ic<2>{}, ic<1>{}) : go(ic<1>{}, ic<1>{});
  });
}

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
