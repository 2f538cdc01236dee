// Linear layers whose weight is in 4 bits (packed4.h) over more rows of 16-bit x than a pass over w takes, on tiles: w's codes come to LDS as they are and become
// values in the registers, so that neither widened weights nor their way to memory and back stand before a layer of some rows.
//
// Stages of 128 channels, a ring of them brought by LDS-DMA: 256 bytes of a row of x, 64 of w and a word of scales.  A wavefront's
// 32 x 32 x 16 instructions take the channels in the order in which the codes lie: a lane's 16 bytes are 32 channels of its row, of which instruction
// t of four takes eight (a word), and of x the same.  us, fp16 8192 -> 8192: 64 rows 23 (the weight at 1.5 TB/s, parts written and joined), 256 50, 1024 128
// (1.07 PFLOP/s; the weight in 16 bits 146).  x lies in rows of 256 bytes whose 16-byte chunks are exchanged by the row, so that the 16 lanes of a read are in different banks.
#include "linear_dma.h"
#include "packed4.h"

#include <algorithm>

namespace wc {

namespace {

struct WideArgs {
  LinearProduct p;            // R: channels
  Operand4 w;
  long long stages, stages_part;
  float* parts;               // (S, M, N); null: one part, the epilogue here
  int tiles_m, tiles_n, n_blocks, per_xcd;
  int vec;
};

// WM x WN blocks of 32 x 32 a wavefront, NWM x NWN wavefronts, stages of the ring
template <int WM_, int WN_, int NWM_, int NWN_, int RING_> struct ShapeWide {
  static constexpr int WM = WM_, WN = WN_, NWM = NWM_, NWN = NWN_, RING = RING_, NW = NWM * NWN, BM = 32 * WM * NWM, BN = 32 * WN * NWN;
  static constexpr int X = BM * 256, W = BN * 64, STAGE = X + W + BN * 4;
  static constexpr int X_LOADS = BM / (4 * NW), LANES = BN / 4 / NW;      // of a wavefront: 1 KB loads of x a stage, lanes that bring scales
  static constexpr size_t EPILOGUE = NW * 32 * (WN * 32 + 4) * 4, LDS = RING * STAGE > EPILOGUE ? RING * STAGE : EPILOGUE;
};

template <typename T, typename SH>
__global__ __launch_bounds__(64 * SH::NW, SH::NW / 4) void linear4_wide_kernel(WideArgs g) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  constexpr int WM = SH::WM, WN = SH::WN, NWN = SH::NWN, BM = SH::BM, BN = SH::BN, NW = SH::NW, RING = SH::RING;
  using B = DmaOperand<half_t, BN, NW, false>;               // codes, in elements of 16 bits
  constexpr int L = SH::X_LOADS + B::LOADS + 1;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int blk = xcd_remap(blockIdx.x, g.per_xcd);
  if (blk >= g.n_blocks) return;
  // tiles along M are neighbours: they read the same weights
  const int tiles = g.tiles_m * g.tiles_n, s = blk / tiles, t0 = blk % tiles;
  const long long m0 = (long long)(t0 % g.tiles_m) * BM, n0 = (long long)(t0 / g.tiles_m) * BN;
  const LinearProduct& p = g.p;
  const long long begin = s * g.stages_part, end = min(g.stages, begin + g.stages_part);
  const int nk = (int)(end - begin);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN, l32 = lane & 31, lhi = lane >> 5;
  // x: lane l of load i brings 16 bytes of row 4 i + l / 16
  const unsigned char* x_base = static_cast<const unsigned char*>(p.a) + (m0 * p.lda + begin * kStage4) * 2;
  long long x_left = (p.M * p.lda - m0 * p.lda - begin * kStage4) * 2;
  unsigned x_off[SH::X_LOADS];
  int x_channel[SH::X_LOADS];                                // of a stage's 128
#pragma unroll
  for (int i = 0; i < SH::X_LOADS; ++i) {
    const int row = (wave + NW * i) * 4 + lane / 16, chunk = lane % 16 ^ (row & 15);
    x_channel[i] = chunk * 8;
    x_off[i] = m0 + row < p.M ? (unsigned)(row * p.lda * 2 + chunk * 16) : kOutside;
  }
  long long x_have = p.R - begin * kStage4;                  // channels from the next stage on
  B b;
  const long long unit = kStage4 / 4, ld = g.stages * unit;
  b.start(g.w.codes, ld, n0, p.N, begin * unit, end * unit, wave, lane);
  const long long row_bytes = g.stages * (kRows4 * 4), row_blocks = (p.N + kRows4 - 1) / kRows4, first = n0 / kRows4 * row_bytes + begin * (kRows4 * 4);
  const unsigned char* scale_base = g.w.scales + first;
  long long scale_left = row_blocks * row_bytes - first;
  const int piece = wave * SH::LANES + lane;
  const unsigned scale_off = n0 / kRows4 + piece / 8 < row_blocks ? (unsigned)(piece / 8 * row_bytes + piece % 8 * 16) : kOutside;

  long long left = (end - begin) * unit;
  auto queue = [&](int slot) {                               // the next stage
    const unsigned at = lds0 + slot * SH::STAGE;
    const DmaDesc d = dma_descriptor(x_base, x_left);
#pragma unroll
    for (int i = 0; i < SH::X_LOADS; ++i) dma16(d, x_channel[i] < x_have ? x_off[i] : kOutside, at + (wave + NW * i) * 1024);
    b.template aim<false>(left);
#pragma unroll
    for (int q = 0; q < B::LOADS; ++q) b.template queue<false>(at + SH::X, 0, wave, q);
    const DmaDesc ds = dma_descriptor(scale_base, scale_left);
    if (lane < SH::LANES) dma16(ds, scale_off, at + SH::X + SH::W + wave * SH::LANES * 16);
    x_base += kStage4 * 2;
    x_left -= kStage4 * 2;
    x_have -= kStage4;
    left -= unit;
    scale_base += kRows4 * 4;
    scale_left -= kRows4 * 4;
  };
  static_assert(SH::X_LOADS >= 1 && SH::LANES >= 1 && SH::LANES * NW * 4 == BN, "the wavefronts' shares");

  f32x16 acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  auto step = [&](const unsigned char* st) {
    unsigned sw[WN];
#pragma unroll
    for (int j = 0; j < WN; ++j) sw[j] = *reinterpret_cast<const unsigned*>(st + SH::X + SH::W + (wn * WN * 32 + j * 32 + l32) * 4) >> (8 * lhi);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      s16x8 x[WM][4], c[WN];
#pragma unroll
      for (int j = 0; j < WN; ++j) c[j] = B::read(st + SH::X + B::offset(wn * WN + j, kk, lane));
#pragma unroll
      for (int i = 0; i < WM; ++i) {
        const int row = (wm * WM + i) * 32 + l32;
#pragma unroll
        for (int t = 0; t < 4; ++t) x[i][t] = *reinterpret_cast<const s16x8*>(st + row * 256 + ((8 * kk + 4 * lhi + t) ^ (row & 15)) * 16);
      }
#pragma unroll
      for (int j = 0; j < WN; ++j) {
        const float scale = scale4(sw[j] >> (16 * kk) & 255u);
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 words = __builtin_bit_cast(u32x4, c[j]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          Pack<T, 8> w;
          values4<T>(words[t], scale, w.v);
#pragma unroll
          for (int i = 0; i < WM; ++i) acc[i][j] = product(__builtin_bit_cast(s16x8, w), x[i][t], acc[i][j], T{});
        }
      }
    }
  };

  // RING - 1 stages on their way beside the one that is multiplied
  for (int k = 0; k < RING - 1 && k < nk; ++k) queue(k);
#pragma unroll 1
  for (int k = 0; k < nk; ++k) {
    // stage k has landed, those after it may be on their way; nobody reads stage k - 1 any more, which that of k + RING - 1 overwrites
    const int after = min(nk - 1 - k, RING - 2);
    if (after == RING - 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((RING - 2) * L) : "memory");
    else if (RING > 3 && after == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(L) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (k + RING - 1 < nk) queue((k + RING - 1) % RING);
    step(lds + k % RING * SH::STAGE);
  }
  static_assert(RING == 3 || RING == 4, "what may be on its way is counted for these");

  const long long wm0 = m0 + wm * WM * 32, wn0 = n0 + wn * WN * 32;
  if (g.parts) {
    store_parts<WM, WN>(g.parts + s * p.M * p.N, acc, wm0, p.M, wn0, p.N, g.vec, lane);
    return;
  }
  __syncthreads();                                           // the ring is done with
  float* const stage = reinterpret_cast<float*>(lds) + wave * 32 * (WN * 32 + 4);
  with_activation(p.e.act, [&](auto act) {
    if (m0 + BM <= p.M && n0 + BN <= p.N) finish_blocks<T, act(), true, true, WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
    else finish_blocks<T, act(), false, true, WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
  });
}

using Wide64 = ShapeWide<2, 1, 1, 4, 4>;          // 64 x 128, 97 KB
using Wide128 = ShapeWide<2, 2, 2, 4, 3>;         // 128 x 256, 150 KB

template <typename T, typename SH>
int launch(const WideArgs& g, void* stream) {
  auto fn = &linear4_wide_kernel<T, SH>;
  if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(fn), SH::LDS)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(64 * SH::NW), SH::LDS, as_stream(stream), g);
  WC_CHECK_LAUNCH("linear4_wide_kernel");
  return WC_OK;
}

}  // namespace

bool linear4_wide_fits(const void* x, long long C, int dtype) { return dtype != WC_F32 && C % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0; }

// a workgroup a compute unit, in parts where there are fewer tiles, of four stages at the least
ProductPlan linear4_wide_plan(const LinearProduct& p) {
  ProductPlan l = {true, false, p.M <= 64 ? ProductTile{64, 128} : ProductTile{128, 256}, 1, 0};
  const long long stages = stages4(p.R), tiles = ceil_div_ll(p.M, l.tile.m) * ceil_div_ll(p.N, l.tile.n);
  const long long s = std::max(1ll, std::min(kCus / tiles, stages / 4));
  l.R_part = ceil_div_ll(stages, s);                         // in stages
  l.s = (int)ceil_div_ll(stages, l.R_part);
  return l;
}

int linear4_wide(const LinearProduct& p, const Operand4& w, const ProductPlan& plan, float* parts, int dtype, void* stream) {
  WideArgs g;
  g.p = p;
  g.w = w;
  g.stages = stages4(p.R);
  g.stages_part = plan.R_part;
  g.parts = plan.s > 1 ? parts : nullptr;
  g.tiles_m = (int)ceil_div_ll(p.M, plan.tile.m);
  g.tiles_n = (int)ceil_div_ll(p.N, plan.tile.n);
  g.n_blocks = g.tiles_m * g.tiles_n * plan.s;
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  g.vec = p.N % 4 == 0;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) return plan.tile.m == 64 ? launch<T, Wide64>(g, stream) : launch<T, Wide128>(g, stream);
    else return fail(WC_ERR_UNSUPPORTED, "linear4_wide_kernel: 16-bit types");
  });
}

}  // namespace wc
