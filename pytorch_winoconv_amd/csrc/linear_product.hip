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

template <typename T> constexpr int kGeneralPitch = 80 / sizeof(T);      // of a row of 64 bytes in LDS
template <typename T> struct GeneralLds { T tile[2][2][64 * kGeneralPitch<T>]; };

template <typename T, bool AO, bool BO>
__device__ __forceinline__ void general_block(const GeneralArgs& g, int hw_block, GeneralLds<T>& shared) {
  constexpr int EPC = 16 / sizeof(T), BK = 4 * EPC, PITCH = kGeneralPitch<T>, AHEAD = 4;
  static_assert(PITCH == BK + EPC, "rows of 64 bytes, 16 apart");
  const int blk = xcd_remap(hw_block, g.per_xcd);
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
      T(&lds)[2][64 * PITCH] = shared.tile[u & 1];
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
      else finish_one<T>(p.e, m, n, p.N, acc[4 * q + e]);
    }
}

template <typename T, bool AO, bool BO>
__global__ __launch_bounds__(256) void product_general_kernel(GeneralArgs g) {
  __shared__ __attribute__((aligned(16))) GeneralLds<T> shared;
  general_block<T, AO, BO>(g, blockIdx.x, shared);
}

// Both gradients of a layer in one launch
template <typename T>
__global__ __launch_bounds__(256) void product_general_pair_kernel(GeneralArgs g, GeneralArgs g2) {
  __shared__ __attribute__((aligned(16))) GeneralLds<T> shared;
  const int n = g.per_xcd * kXcds;
  if ((int)blockIdx.x < n) general_block<T, false, true>(g, blockIdx.x, shared);
  else general_block<T, true, true>(g2, blockIdx.x - n, shared);
}

// Few rows (at most 16 of M, 16-bit types, both operands with the reduction innermost): one pass over B, which bounds it.  A workgroup of 16 wavefronts takes NR
// rows of B (4, 8 or 16, no less than there are of A: few, so that every compute unit has some), whose reduction the wavefronts share, 64 elements
// at a time - both halves of a line of the L2, one after the other, straight into the operands of two 16 x 16 x 32 instructions.  The 16 rows of
// an instruction are NR rows at 16 / NR places of the reduction, of A as of B; of its results those of two equal places count.  The sums meet in LDS, so there
// are no parts and no second launch.
constexpr int kFewWaves = 16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <typename T, int NR>
__global__ __launch_bounds__(64 * kFewWaves) void product_few_kernel(LinearProduct p) {
  constexpr int PLACES = 16 / NR, AT_ONCE = 4;
  __shared__ float sums[kFewWaves * PLACES][NR][NR + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane % NR, place = (lane & 15) / NR, c = lane >> 4;
  const long long n0 = (long long)blockIdx.x * NR;
  const T* const w = static_cast<const T*>(p.b) + min(n0 + r, p.N - 1) * p.ldb;
  const T* const x = static_cast<const T*>(p.a) + min((long long)r, p.M - 1) * p.lda;
  const bool row = r < p.M;
  const int chunks = (int)((p.R + 64 * PLACES - 1) / (64 * PLACES));
  using V = Pack<T, 8>;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  V zero;
#pragma unroll
  for (int e = 0; e < 8; ++e) zero.v[e] = static_cast<T>(0.f);
  auto multiply = [&](const V& a, const V& b) {
    if constexpr (std::is_same<T, half_t>::value) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    else acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  };
  for (int k0 = wave; k0 < chunks; k0 += AT_ONCE * kFewWaves) {
    V wv[AT_ONCE][2], xv[AT_ONCE][2];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long k = ((long long)(k0 + u * kFewWaves) * PLACES + place) * 64 + h * 32 + c * 8;
        const bool in = k < p.R;                    // (R is a multiple of eight, or rows have zeros up to one)
        wv[u][h] = in ? *reinterpret_cast<const V*>(w + k) : zero;
        xv[u][h] = in && row ? *reinterpret_cast<const V*>(x + k) : zero;
      }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) multiply(wv[u][h], xv[u][h]);
  }
  // register e of a lane: row 4 c + e of B's sixteen, row lane % 16 of A's
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if ((4 * c + e) / NR == place) sums[wave * PLACES + place][r][(4 * c + e) % NR] = acc[e];
  __syncthreads();
  const int m = threadIdx.x / NR, n = threadIdx.x % NR;
  if (m >= NR || m >= p.M || n0 + n >= p.N) return;
  float v = 0.f;
#pragma unroll 16
  for (int s = 0; s < kFewWaves * PLACES; ++s) v += sums[s][m][n];
  finish_one<T>(p.e, m, n0 + n, p.N, v);
}
// ... for a B of up to 4 MB, which is over before a second launch would begin; more loads are in flight in parts of tiles.  us, fp16, tiles and parts | this:
// 1 x 1024 -> 1024 10.2 | 6.3, 8 x 2048 -> 2048 10.3 | 10.5, 8 x 4096 -> 4096 12.4 | 20.4
bool few_rows_pay(const LinearProduct& p, int dtype) {
  return dtype != WC_F32 && !p.a_outer && !p.b_outer && p.M <= 16 && p.N * p.R <= 2 << 20;
}

long long tiles_of(const LinearProduct& p, ProductTile t) { return ceil_div_ll(p.M, t.m) * ceil_div_ll(p.N, t.n); }

// What 64 elements of the reduction take a workgroup, alone on its compute unit and with as many as it holds, and what the epilogue takes, plain and
// heavy, in us; measured on 16-bit products of 4096 and 8192 squared (fp32 instructions: 128 x 128 seven times, 64 x 64 five times that, alone three times)
struct TileCost { ProductTile tile; int slots; double alone, full, plain, heavy; };
constexpr TileCost kTileCosts[] = {{{64, 64}, 4, 0.55, 1.1, 1, 3}, {{128, 128}, 2, 0.6, 1.17, 2, 6}, {{256, 256}, 1, 1.85, 1.85, 5, 18}};
constexpr TileCost kGeneralCost = {{64, 64}, 4, 2, 2, 2, 4};

// The least estimate over tiles and numbers of parts; parts' sums cost their way to memory and back, and the launch that adds them.  beside: us that another
// product keeps the chip busy in the same launch, which leaves the tile as it is and makes parts fewer
ProductPlan plan_of(const LinearProduct& p, bool dma, bool heavy, int dtype, double beside, double* busy = nullptr, bool few = true) {
  ProductPlan l = {dma, false, {64, 64}, 1, 0};
  const int forced = test_gemm_config();
  if (few && forced < 0 && dma && few_rows_pay(p, dtype)) {
    l.few = true;
    l.R_part = std::max(p.R, 1ll);
    return l;
  }
  const long long steps = std::max(1ll, ceil_div_ll(p.R, 64)), room = std::max(1ll, (256ll << 20) / std::max(4 * p.M * p.N, 1ll));      // 256 MB of sums
  double least = -1;
  long long best = 1;
  auto consider = [&](const TileCost& c, double beside) {
    const double f = dtype == WC_F32 ? (c.tile.m == 64 ? 5 : 7) : 1, f_alone = dtype == WC_F32 ? 3 : 1;
    const long long tiles = tiles_of(p, c.tile), slots = (long long)c.slots * kCus, most = c.tile.m == 256 || tiles >= slots ? 1 : std::min({steps, room, 4ll * kCus});
    for (long long s = 1; s <= most; s += 1 + s / 4) {
      const long long each = ceil_div_ll(steps, s), n = tiles * ceil_div_ll(steps, each);
      const double end = heavy && s == 1 ? c.heavy : c.plain;
      const double rounds = n <= slots ? (double)n / slots : (double)ceil_div_ll(n, slots);
      const double us = std::max({each * c.alone * f_alone + end, rounds * (each * c.full * f + end), rounds * (each * c.full * f + end) * 0.9 + beside}) + (s > 1 ? 8 + 1e-6 * s * p.M * p.N : 0);
      if (least >= 0 && us >= least) continue;
      least = us;
      best = s;
      l.tile = c.tile;
      if (busy) *busy = c.tile.m == 256 ? 0 : rounds * (each * c.full * f + end);      // (the largest tiles share no launch)
    }
  };
  if (!dma) consider(kGeneralCost, 0);
  else if (forced >= 32 && forced <= 34) consider(kTileCosts[std::min(forced - 32, dtype == WC_F32 ? 1 : 2)], 0);
  else
    for (const TileCost& c : kTileCosts)
      if (c.tile.m < 256 || dtype != WC_F32) consider(c, 0);
  if (beside > 0 && l.tile.m < 256) {
    const TileCost c = dma ? kTileCosts[l.tile.m / 128] : kGeneralCost;
    least = -1;
    consider(c, beside);
  }
  l.R_part = ceil_div_ll(steps, best) * 64;
  l.s = (int)std::max(1ll, ceil_div_ll(p.R, l.R_part));
  return l;
}

}  // namespace

// (codes of 4 bits lie in rows of a quarter as many 16-bit elements, which take the matrix instructions as long)
ProductPlan product_plan4(const LinearProduct& p, bool heavy) { return plan_of(p, true, heavy, WC_F16, 0, nullptr, false); }

ProductPlan product_plan(const LinearProduct& p, int dtype, const LinearProduct* beside) {
  const bool dma = test_gemm_config() != 31 && product_dma_fits(p, dtype);
  double busy = 0;
  if (beside) plan_of(*beside, dma, false, dtype, 0, &busy);
  return plan_of(p, dma, linear_heavy(p.e), dtype, busy);
}

size_t product_parts_bytes(const LinearProduct& p, int dtype, const LinearProduct* beside) {
  double busy = 0;
  long long s = 1;
  for (const bool dma : {true, false}) {
    if (beside) plan_of(*beside, dma, false, dtype, 0, &busy);
    for (const bool heavy : {true, false}) s = std::max<long long>(s, plan_of(p, dma, heavy, dtype, busy).s);
  }
  return s > 1 ? (size_t)s * p.M * p.N * 4 : 0;
}

static GeneralArgs general_args(const LinearProduct& p, const ProductPlan& plan, float* parts) {
  GeneralArgs g;
  g.p = p;
  g.parts = plan.s > 1 ? parts : nullptr;
  g.R_part = plan.R_part;
  g.tiles_m = (int)ceil_div_ll(p.M, 64); g.tiles_n = (int)ceil_div_ll(p.N, 64);
  g.n_blocks = (int)(tiles_of(p, plan.tile) * plan.s);
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  return g;
}

// Rows m0 .. m0 + M - 1 of a product's results
static LinearProduct rows_of(const LinearProduct& p, long long m0, long long M, int dtype) {
  const long long es = dtype == WC_F32 ? 4 : 2;
  LinearProduct q = p;
  q.M = M;
  q.a = static_cast<const char*>(p.a) + (p.a_outer ? m0 : m0 * p.lda) * es;
  if (p.e.res) q.e.res = static_cast<const char*>(p.e.res) + m0 * p.N * es;
  if (p.e.z) q.e.z = static_cast<char*>(p.e.z) + m0 * p.N * es;
  q.e.y = static_cast<char*>(p.e.y) + m0 * p.N * (p.e.y_f32 ? 4 : es);
  return q;
}

int product_run(const LinearProduct& p, const ProductPlan& plan, float* parts, int dtype, void* stream) {
  // (few results are left to parts: those have few tiles)
  const long long most = kMostBlocks / ceil_div_ll(p.N, plan.tile.n) * plan.tile.m;
  if (p.M > most && plan.s == 1) {
    for (long long m0 = 0; m0 < p.M; m0 += most)
      if (int rc = product_run(rows_of(p, m0, std::min(most, p.M - m0), dtype), plan, nullptr, dtype, stream)) return rc;
    return WC_OK;
  }
  if (plan.few) {
    return dispatch_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      if constexpr (sizeof(T) == 2) {
        const int nr = p.M <= 4 ? 4 : p.M <= 8 ? 8 : 16;
        auto fn = nr == 4 ? &product_few_kernel<T, 4> : nr == 8 ? &product_few_kernel<T, 8> : &product_few_kernel<T, 16>;
        hipLaunchKernelGGL(fn, dim3((unsigned)ceil_div_ll(p.N, nr)), dim3(64 * kFewWaves), 0, as_stream(stream), p);
        WC_CHECK_LAUNCH("product_few_kernel");
        return WC_OK;
      } else {
        return fail(WC_ERR_UNSUPPORTED, "product_few_kernel: 16-bit types");
      }
    });
  }
  if (plan.dma) return product_dma(p, plan, parts, dtype, stream);
  const GeneralArgs g = general_args(p, plan, parts);
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto fn = p.a_outer ? &product_general_kernel<T, true, true> : p.b_outer ? &product_general_kernel<T, false, true> : &product_general_kernel<T, false, false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(256), 0, as_stream(stream), g);
    WC_CHECK_LAUNCH("product_general_kernel");
    return WC_OK;
  });
}

int product_run_pair(const LinearProduct& p, const ProductPlan& plan, float* parts, const LinearProduct& p2, const ProductPlan& plan2, float* parts2, int dtype, void* stream) {
  const bool few = tiles_of(p, plan.tile) * plan.s + tiles_of(p2, plan2.tile) * plan2.s <= kMostBlocks - kXcds;
  if (few && product_dma_pairs(plan, plan2)) return product_dma_pair(p, plan, parts, p2, plan2, parts2, dtype, stream);
  if (few && !plan.dma && !plan2.dma) {
    const GeneralArgs g = general_args(p, plan, parts), g2 = general_args(p2, plan2, parts2);
    return dispatch_dtype(dtype, [&](auto t) -> int {
      hipLaunchKernelGGL(product_general_pair_kernel<decltype(t)>, dim3((unsigned)((g.per_xcd + g2.per_xcd) * kXcds)), dim3(256), 0, as_stream(stream), g, g2);
      WC_CHECK_LAUNCH("product_general_pair_kernel");
      return WC_OK;
    });
  }
  if (int rc = product_run(p, plan, parts, dtype, stream)) return rc;
  return product_run(p2, plan2, parts2, dtype, stream);
}

}  // namespace wc
