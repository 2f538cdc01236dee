// Products of two operands in 4 bits (packed4.h) on the matrix cores' scaled instructions, fed by LDS-DMA.
//
// A 32 x 32 x 64 instruction takes 16 bytes of codes a lane and operand and lasts as long as a 16-bit one of 16 reduction elements, so a
// product of codes is, byte for byte, the 16-bit product of a quarter as many elements (linear_dma.hip): the same stages of 64 bytes, the same way
// through LDS, 64 reduction channels for 16.  Beside them come the scales, a word a row and stage: a lane's group is one byte of it, shifted into place
// once a stage.  The stages' 64-byte halves of L2 lines come in pairs, two pairs of buffers: while one is multiplied the other lands.
//
// us and PFLOP/s without an epilogue: 4096^3 41 (3.4), 8192^3 287 (3.8), 8192 x 25088 -> 4096 399 (4.2), matrix cores busy 39 % of the cycles: the wavefronts' reads of LDS, 96 of
// its 128 bytes a cycle, and the stages' way there take as long as the instructions (8192^3 with that way left out 222, without the reads 253, the instructions alone 194).  Four wavefronts of 128 x 128, which read a third less, have nobody to wait beside
// them (8192^3 300); single stages in a ring of four come at half lines of the L2 (306).
//
// The wavefronts each bring a share of a stage's scales, some of their lanes 16 bytes each, so that all count the same loads.
#include "linear_dma.h"
#include "packed4.h"

namespace wc {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int HALF>
__device__ __forceinline__ f32x16 product4(s16x8 a, s16x8 b, f32x16 c, int scale_a, int scale_b) {
  const i32x4 p = __builtin_bit_cast(i32x4, a), q = __builtin_bit_cast(i32x4, b);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(i32x8{p[0], p[1], p[2], p[3], 0, 0, 0, 0}, i32x8{q[0], q[1], q[2], q[3], 0, 0, 0, 0}, c, 4, 4,
                                                         2 * HALF, scale_a, 2 * HALF, scale_b);
}

struct Dma4Args {
  LinearProduct p;            // extents of the operands' rows in elements of 16 bits
  const unsigned char* scale_a; const unsigned char* scale_b;
  long long stages;
  float* parts;               // (S, M, N); null: one part, the epilogue here
  long long R_part;
  int tiles_m, tiles_n, n_blocks, per_xcd;
  int vec;
};

// WM x WN blocks of 32 x 32 a wavefront, NWM x NWN wavefronts
template <int WM_, int WN_, int NWM_, int NWN_> struct Shape4 {
  static constexpr int WM = WM_, WN = WN_, NWM = NWM_, NWN = NWN_, NW = NWM * NWN, BM = 32 * WM * NWM, BN = 32 * WN * NWN;
  static constexpr int CODES = 64 * (BM + BN), STAGE = CODES + 4 * (BM + BN);
  static constexpr int LANES = (BM + BN) / 4 / NW;        // of a wavefront that bring scales
  static constexpr size_t EPILOGUE = NW * 32 * (WN * 32 + 4) * 4, LDS = 4 * STAGE > EPILOGUE ? 4 * STAGE : EPILOGUE;
};
constexpr int kBand4 = 8;

template <typename T, typename SH>
__global__ __launch_bounds__(64 * SH::NW, 2) void product4_dma_kernel(Dma4Args g) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  constexpr int WM = SH::WM, WN = SH::WN, NWM = SH::NWM, NWN = SH::NWN, BM = SH::BM, BN = SH::BN, NW = SH::NW;
  using E = half_t;           // what an element of 16 bits is called
  using A = DmaOperand<E, BM, NW, false>;
  using B = DmaOperand<E, BN, NW, false>;
  constexpr int L = A::LOADS + B::LOADS;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int blk = xcd_remap(blockIdx.x, g.per_xcd);
  if (blk >= g.n_blocks) return;
  const int tiles = g.tiles_m * g.tiles_n, s = blk / tiles, t = blk % tiles;
  const int band = t / (kBand4 * g.tiles_n), in_band = t % (kBand4 * g.tiles_n), high = min(kBand4, g.tiles_m - band * kBand4);
  const long long m0 = (long long)(band * kBand4 + in_band % high) * BM, n0 = (long long)(in_band / high) * BN;
  const LinearProduct& p = g.p;
  const long long begin = s * g.R_part, end = min(p.R, begin + g.R_part);
  const int nk = end > begin ? (int)((end - begin) / kDeep<E>) : 0;           // (whole stages)

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN, l32 = lane & 31, lhi = lane >> 5;
  A a;
  B b;
  a.start(p.a, p.lda, m0, p.M, begin, end, wave, lane);
  b.start(p.b, p.ldb, n0, p.N, begin, end, wave, lane);
  // scales: the wavefronts' first half brings A's, a row of blocks of 32 rows, 128 bytes a stage each
  const bool of_b = wave >= NW / 2;
  const int piece = (wave % (NW / 2)) * SH::LANES + lane;
  const long long row0 = of_b ? n0 : m0, rows = of_b ? p.N : p.M, row_bytes = g.stages * (kRows4 * 4);
  const long long blocks = (rows + kRows4 - 1) / kRows4, first = row0 / kRows4 * row_bytes + begin / kDeep<E> * (kRows4 * 4);
  const unsigned char* scale_base = (of_b ? g.scale_b : g.scale_a) + first;
  long long scale_left = blocks * row_bytes - first;
  const unsigned scale_off = row0 / kRows4 + piece / 8 < blocks ? (unsigned)((piece / 8) * row_bytes + piece % 8 * 16) : kOutside;
  const unsigned scale_to = SH::CODES + (of_b ? BM * 4 : 0) + (wave % (NW / 2)) * SH::LANES * 16;

  long long left = end - begin;
  auto queue_pair = [&](int half) {               // the next two stages, into slots 2 half and 2 half + 1
    const unsigned at = lds0 + half * 2 * SH::STAGE, at2 = at + SH::STAGE;
    a.template aim<true>(left);
    b.template aim<true>(left);
    left -= 2 * kDeep<E>;
#pragma unroll
    for (int q = 0; q < A::LOADS; ++q) a.template queue<true>(at, at2, wave, q);
#pragma unroll
    for (int q = 0; q < B::LOADS; ++q) b.template queue<true>(at + A::BYTES, at2 + A::BYTES, wave, q);
    const DmaDesc d = dma_descriptor(scale_base, scale_left), d2 = dma_descriptor(scale_base + kRows4 * 4, scale_left - kRows4 * 4);
    if (lane < SH::LANES) {
      dma16(d, scale_off, at + scale_to);
      dma16(d2, scale_off, at2 + scale_to);
    }
    scale_base += 2 * kRows4 * 4;
    scale_left -= 2 * kRows4 * 4;
  };
  static_assert(L > 0 && SH::LANES <= 64 && SH::LANES * NW * 4 == BM + BN, "the wavefronts' shares");

  f32x16 acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  int fa[2][WM], fb[2][WN];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
    for (int i = 0; i < WM; ++i) fa[kk][i] = A::offset(wm * WM + i, kk, lane);
#pragma unroll
    for (int j = 0; j < WN; ++j) fb[kk][j] = A::BYTES + B::offset(wn * WN + j, kk, lane);
  }
  const int ga = SH::CODES + (wm * WM * 32 + l32) * 4, gb = SH::CODES + BM * 4 + (wn * WN * 32 + l32) * 4;
  // The halves of a pair's stages, 64 channels each: while one is multiplied the next is read, and with it, stage by stage, the scales
  s16x8 va[2][WM], vb[2][WN];
  unsigned sa[2][WM], sb[2][WN];
  auto read = [&](const unsigned char* st, int kk) {
    if (kk == 0) {
#pragma unroll
      for (int i = 0; i < WM; ++i) sa[0][i] = *reinterpret_cast<const unsigned*>(st + ga + i * 128) >> (8 * lhi);
#pragma unroll
      for (int j = 0; j < WN; ++j) sb[0][j] = *reinterpret_cast<const unsigned*>(st + gb + j * 128) >> (8 * lhi);
    }
#pragma unroll
    for (int i = 0; i < WM; ++i) va[kk][i] = A::read(st + fa[kk][i]);
#pragma unroll
    for (int j = 0; j < WN; ++j) vb[kk][j] = B::read(st + fb[kk][j]);
  };
  auto keep_scales = [&] {
#pragma unroll
    for (int i = 0; i < WM; ++i) sa[1][i] = sa[0][i];
#pragma unroll
    for (int j = 0; j < WN; ++j) sb[1][j] = sb[0][j];
  };
  auto multiply = [&](auto half) {
    constexpr int H = decltype(half)::value;
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
      for (int j = 0; j < WN; ++j) acc[i][j] = product4<H>(vb[H][j], va[H][i], acc[i][j], sb[H][j], sa[H][i]);
  };

  const int pairs = (nk + 1) / 2;
  if (pairs > 0) queue_pair(0);
#pragma unroll 1
  for (int j = 0; j < pairs; ++j) {
    // pair j has landed, and nobody reads pair j - 1 any more, which pair j + 1 overwrites
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const unsigned char* const st = lds + (j & 1) * 2 * SH::STAGE;
    read(st, 0);
    keep_scales();
    read(st, 1);
    if (j + 1 < pairs) queue_pair((j + 1) & 1);
    multiply(ic<0>{});
    if (2 * j + 1 < nk) {
      read(st + SH::STAGE, 0);
      multiply(ic<1>{});
      keep_scales();
      read(st + SH::STAGE, 1);
      multiply(ic<0>{});
    }
    multiply(ic<1>{});
  }

  const long long wm0 = m0 + wm * WM * 32, wn0 = n0 + wn * WN * 32;
  if (g.parts) {
    store_parts<WM, WN>(g.parts + s * p.M * p.N, acc, wm0, p.M, wn0, p.N, g.vec, lane);
    return;
  }
  __syncthreads();                                          // the buffers are done with
  float* const stage = reinterpret_cast<float*>(lds) + wave * 32 * (WN * 32 + 4);
  with_activation(p.e.act, [&](auto act) {
    if (m0 + BM <= p.M && n0 + BN <= p.N) finish_blocks<T, act(), true, true, WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
    else finish_blocks<T, act(), false, true, WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
  });
}

using Tile256 = Shape4<4, 2, 2, 4>;
using Tile128 = Shape4<2, 2, 2, 2>;
using Tile64 = Shape4<1, 1, 2, 2>;

template <typename T, typename SH>
int launch(const Dma4Args& g, void* stream) {
  auto fn = &product4_dma_kernel<T, SH>;
  if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(fn), SH::LDS)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(64 * SH::NW), SH::LDS, as_stream(stream), g);
  WC_CHECK_LAUNCH("product4_dma_kernel");
  return WC_OK;
}

// the product in elements of 16 bits
LinearProduct in_halves(const LinearProduct& p) {
  LinearProduct q = p;
  q.R = p.R / 4;
  q.lda = q.ldb = q.R;
  return q;
}

}  // namespace

ProductPlan product4_plan(const LinearProduct& p) { return product_plan4(in_halves(p), linear_heavy(p.e)); }

int product4_dma(const LinearProduct& p4, const Operand4& x, const Operand4& w, const ProductPlan& plan, float* parts, int dtype, void* stream) {
  Dma4Args g;
  g.p = in_halves(p4);
  g.p.a = x.codes;
  g.p.b = w.codes;
  g.scale_a = x.scales;
  g.scale_b = w.scales;
  g.stages = p4.R / kStage4;
  g.parts = plan.s > 1 ? parts : nullptr;
  g.R_part = plan.R_part;
  g.tiles_m = (int)ceil_div_ll(p4.M, plan.tile.m);
  g.tiles_n = (int)ceil_div_ll(p4.N, plan.tile.n);
  const long long blocks = (long long)g.tiles_m * g.tiles_n * plan.s;
  if (blocks > kMostBlocks) return fail(WC_ERR_UNSUPPORTED, "linear layer in 4 bits: %lld x %lld results", p4.M, p4.N);
  g.n_blocks = (int)blocks;
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  g.vec = p4.N % 4 == 0;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (plan.tile.m == 256) return launch<T, Tile256>(g, stream);
    return plan.tile.m == 128 ? launch<T, Tile128>(g, stream) : launch<T, Tile64>(g, stream);
  });
}

}  // namespace wc
