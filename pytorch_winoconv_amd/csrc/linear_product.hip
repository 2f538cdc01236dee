// Which kernel a product of linear.h takes, and the one for every size, alignment and layout: small products of rows that are no multiple
// of 16 bytes, which are not worth a copy to ones that are.
//
// 64 x 64 results per workgroup, a 32 x 32 block of the matrix cores per wavefront.  A stage of 64 bytes of the reduction goes through registers, three
// stages ahead, to one of two LDS buffers with the reduction innermost, whichever way it lies; one barrier a stage.
#include "linear_rows.h"

#include <algorithm>

namespace wc {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct GeneralArgs {
  LinearProduct p;
  float* parts;               // (S, M, N); null: one part, the epilogue here
  long long R_part;
  int tiles_m, tiles_n, n_blocks, per_xcd;
};

template <typename T>
__device__ __forceinline__ void finish(const LinearEpilogue& e, long long m, long long n, long long N, float v) {
  const long long i = m * N + n;
  if (e.bias) v += static_cast<float>(static_cast<const T*>(e.bias)[n]);
  const float r = e.res ? static_cast<float>(static_cast<const T*>(e.res)[i]) : 0.f;
  if (!e.res_after) v += r;
  if (e.z) static_cast<T*>(e.z)[i] = static_cast<T>(v);
  v = activate(v, e.act);
  if (e.res_after) v += r;
  if (e.y_f32) static_cast<float*>(e.y)[i] = v;
  else static_cast<T*>(e.y)[i] = static_cast<T>(v);
}

template <typename T, bool AO, bool BO>
__global__ __launch_bounds__(256) void product_general_kernel(GeneralArgs g) {
  constexpr int EPC = 16 / sizeof(T), BK = 4 * EPC, PITCH = BK + EPC, AHEAD = 4;
  __shared__ __attribute__((aligned(16))) T tile[2][2][64 * PITCH];
  const int blk = xcd_remap(blockIdx.x, g.per_xcd);
  if (blk >= g.n_blocks) return;
  const int tn = blk % g.tiles_n, tm = blk / g.tiles_n % g.tiles_m, s = blk / (g.tiles_n * g.tiles_m);
  const LinearProduct& p = g.p;
  const long long m0 = (long long)tm * 64, n0 = (long long)tn * 64;
  const long long begin = s * g.R_part, end = min(p.R, begin + g.R_part);
  const int nk = end > begin ? (int)((end - begin + BK - 1) / BK) : 0;
  const int tid = threadIdx.x;

  // EPC elements a thread: of one row along the reduction, or of one reduction element along the rows
  auto load = [&](auto outer, const void* src, long long ld, long long row0, long long rows, int ks, T (&v)[EPC]) {
    const long long r = row0 + (outer() ? tid % (64 / EPC) * EPC : tid / 4), k = begin + (long long)ks * BK + (outer() ? tid / (64 / EPC) : tid % 4 * EPC);
    const long long have = outer() ? (k < end ? rows - r : 0) : (r < rows ? end - k : 0);
    load_run<T, EPC>(src, outer() ? k * ld + r : r * ld + k, (int)min(max(have, 0ll), (long long)EPC), v);
  };
  auto store = [&](auto outer, T* to, const T (&v)[EPC]) {
    if constexpr (outer()) {
#pragma unroll
      for (int e = 0; e < EPC; ++e) to[(tid % (64 / EPC) * EPC + e) * PITCH + tid / (64 / EPC)] = v[e];
    } else {
      Pack<T, EPC> w;
#pragma unroll
      for (int e = 0; e < EPC; ++e) w.v[e] = v[e];
      *reinterpret_cast<Pack<T, EPC>*>(to + tid / 4 * PITCH + tid % 4 * EPC) = w;
    }
  };
  using OA = std::integral_constant<bool, AO>;
  using OB = std::integral_constant<bool, BO>;

  const int lane = tid & 63, wave = tid >> 6, l32 = lane & 31, lhi = lane >> 5;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x16 acc = {};
  T va[AHEAD][EPC], vb[AHEAD][EPC];
#pragma unroll
  for (int u = 0; u < AHEAD - 1; ++u) {
    if (u >= nk) break;
    load(OA{}, p.a, p.lda, m0, p.M, u, va[u]);
    load(OB{}, p.b, p.ldb, n0, p.N, u, vb[u]);
  }
#pragma unroll 1
  for (int k0 = 0; k0 < nk; k0 += AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int ks = k0 + u;
      if (ks >= nk) break;
      if (ks + AHEAD - 1 < nk) {
        load(OA{}, p.a, p.lda, m0, p.M, ks + AHEAD - 1, va[(u + AHEAD - 1) % AHEAD]);
        load(OB{}, p.b, p.ldb, n0, p.N, ks + AHEAD - 1, vb[(u + AHEAD - 1) % AHEAD]);
      }
      T(&lds)[2][64 * PITCH] = tile[u & 1];
      store(OA{}, lds[0], va[u]);
      store(OB{}, lds[1], vb[u]);
      __syncthreads();                             // and nobody multiplies from the other buffer any more
      const T* const ra = lds[0] + (wm + l32) * PITCH;
      const T* const rb = lds[1] + (wn + l32) * PITCH;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < BK; k += 2) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(rb[k + lhi], ra[k + lhi], acc, 0, 0, 0);
      } else {
#pragma unroll
        for (int k = 0; k < BK; k += 16) {
          if constexpr (std::is_same<T, half_t>::value)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8*>(rb + k + lhi * 8), *reinterpret_cast<const f16x8*>(ra + k + lhi * 8), acc, 0, 0, 0);
          else
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(rb + k + lhi * 8), *reinterpret_cast<const bf16x8*>(ra + k + lhi * 8), acc, 0, 0, 0);
        }
      }
    }
  }
  // register 4 q + e of a lane: row l32, column 8 q + 4 lhi + e of the block
  const long long m = m0 + wm + l32;
  if (m >= p.M) return;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long long n = n0 + wn + 8 * q + 4 * lhi + e;
      if (n >= p.N) continue;
      if (g.parts) g.parts[(s * p.M + m) * p.N + n] = acc[4 * q + e];
      else finish<T>(p.e, m, n, p.N, acc[4 * q + e]);
    }
}

long long tiles_of(const LinearProduct& p, ProductTile t) { return ceil_div_ll(p.M, t.m) * ceil_div_ll(p.N, t.n); }

// beside: steps of 64 elements of another product's tiles that run beside this one's
ProductPlan plan_of(const LinearProduct& p, bool dma, int dtype, long long beside) {
  ProductPlan l = {dma, {64, 64}, 1, 0};
  const int forced = test_gemm_config();
  const bool heavy = p.e.act != WC_ACT_NONE || p.e.z || p.e.res;
  if (forced >= 32 && forced <= 34 && dma) {
    const ProductTile tiles[] = {{64, 64}, {128, 128}, {256, 256}};
    l.tile = tiles[std::min(forced - 32, dtype == WC_F32 || heavy ? 1 : 2)];
  } else if (dma) {
    if (dtype != WC_F32 && !heavy && tiles_of(p, {256, 256}) >= kCus && p.R >= 2048) l.tile = {256, 256};
    else if (tiles_of(p, {128, 128}) * std::max(1ll, p.R / 512) >= 3 * kCus / 2) l.tile = {128, 128};
  }
  // Parts: the number with the least estimate.  Two tiles of 128 x 128 or four of 64 x 64 are on a compute unit at a time, whose workgroups take some 0.5
  // or 0.35 us for 64 elements then (product_general_kernel's 2); a part's sums cost their way to memory and back, and the launch that adds them
  const long long tiles = tiles_of(p, l.tile), steps = std::max(1ll, ceil_div_ll(p.R, 64)), slots = (l.tile.m == 128 ? 2 : 4) * kCus;
  const double step_us = (l.tile.m == 128 ? 0.5 : dma ? 0.35 : 2) * (dtype == WC_F32 ? 4 : 1);
  double least = 0;
  long long best = 1;
  const long long most = l.tile.m == 256 ? 1 : std::min(steps, std::max(1ll, (256ll << 20) / std::max(4 * p.M * p.N, 1ll)));
  for (long long s = 1; s <= most && s <= 4 * kCus; s += 1 + s / 8) {
    const long long each = ceil_div_ll(steps, s), rounds = ceil_div_ll(tiles * ceil_div_ll(steps, each), slots);
    const double us = std::max((double)(rounds * each), (double)(tiles * steps + beside) / slots) * step_us + (s > 1 ? 4 + 8e-6 * s * p.M * p.N / 4 : 0);
    if (s == 1 || us < least) { least = us; best = s; }
  }
  l.R_part = ceil_div_ll(steps, best) * 64;
  l.s = (int)std::max(1ll, ceil_div_ll(p.R, l.R_part));
  return l;
}

}  // namespace

ProductPlan product_plan(const LinearProduct& p, int dtype, const LinearProduct* beside) {
  const bool dma = test_gemm_config() != 31 && product_dma_fits(p, dtype);
  if (!beside) return plan_of(p, dma, dtype, 0);
  const ProductPlan other = plan_of(*beside, dma, dtype, 0);
  const long long per = other.tile.m == 128 ? 1 : 4;           // (a step of a 64 x 64 tile is a quarter of one of 128 x 128)
  const ProductPlan own = plan_of(p, dma, dtype, 0);
  return plan_of(p, dma, dtype, tiles_of(*beside, other.tile) * ceil_div_ll(beside->R, 64) * (own.tile.m == 128 ? 1 : 4) / per);
}

size_t product_parts_bytes(const LinearProduct& p, int dtype) {
  // (what runs beside makes parts fewer)
  const int s = std::max(plan_of(p, true, dtype, 0).s, plan_of(p, false, dtype, 0).s);
  return s > 1 ? (size_t)s * p.M * p.N * 4 : 0;
}

int product_run(const LinearProduct& p, const ProductPlan& plan, float* parts, int dtype, void* stream) {
  const long long tiles = tiles_of(p, plan.tile);
  if (tiles * plan.s >= (1ll << 31) - 8) return fail(WC_ERR_UNSUPPORTED, "a product of %lld x %lld has too many tiles", p.M, p.N);
  if (plan.dma) return product_dma(p, plan, parts, dtype, stream);
  GeneralArgs g;
  g.p = p;
  g.parts = plan.s > 1 ? parts : nullptr;
  g.R_part = plan.R_part;
  g.tiles_m = (int)ceil_div_ll(p.M, 64); g.tiles_n = (int)ceil_div_ll(p.N, 64);
  g.n_blocks = (int)(tiles * plan.s);
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto fn = p.a_outer ? &product_general_kernel<T, true, true> : p.b_outer ? &product_general_kernel<T, false, true> : &product_general_kernel<T, false, false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(256), 0, as_stream(stream), g);
    WC_CHECK_LAUNCH("product_general_kernel");
    return WC_OK;
  });
}

int product_run_pair(const LinearProduct& p, const ProductPlan& plan, float* parts, const LinearProduct& p2, const ProductPlan& plan2, float* parts2, int dtype, void* stream) {
  const bool few = tiles_of(p, plan.tile) * plan.s + tiles_of(p2, plan2.tile) * plan2.s < (1ll << 31) - 16;
  if (few && product_dma_pairs(plan, plan2)) return product_dma_pair(p, plan, parts, p2, plan2, parts2, dtype, stream);
  if (int rc = product_run(p, plan, parts, dtype, stream)) return rc;
  return product_run(p2, plan2, parts2, dtype, stream);
}

}  // namespace wc
