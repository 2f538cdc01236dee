// The products of linear.h on the matrix cores, both operands brought to LDS by LDS-DMA: rows that are multiples of 16 bytes.
//
// A workgroup's four wavefronts (2 x 2) take WM x WN blocks of 32 x 32 each.  A ring of stages of 64 bytes of the reduction (32 elements of
// 16-bit types, 16 of fp32).  An operand whose reduction axis is innermost lies in LDS in rows of 64 bytes, its 16-byte chunks exchanged by the row, and
// is read 16 bytes a lane; one whose reduction axis is outermost lies as it does in memory, pieces of its rows exchanged by the row, and is read by
// ds_read_b64_tr_b16, which hands each lane four elements of a column (fp32: four reads of an element): nothing is transposed in memory
// for either gradient.  Both swizzles keep the lanes of a read in different banks.  What lies outside an operand - rows, columns, the end
// of the reduction - are offsets outside its descriptor, which bring zeros.
//
// Results go through LDS in fp32, 32 rows of a wavefront at a time, so that bias, residual, y and z are read and written 16 bytes a lane in
// whole row segments; few tiles: parts of the reduction, whose sums join_kernel (linear_gradient.hip) adds.
#include "linear_dma.h"

#include <algorithm>

namespace wc {

namespace {

struct DmaArgs {
  LinearProduct p;
  float* parts;               // (S, M, N); null: one part, the epilogue here
  long long R_part;
  int tiles_m, tiles_n, n_blocks, per_xcd;
  int vec;                    // rows of the parts' sums are multiples of 16 bytes
};

// Template of a product: blocks of a wavefront, wavefronts, stages of the ring, whether the first half of a stage is read while the last one of the
// stage before is multiplied (a wavefront alone on its SIMD waits for every read that is not ahead)
template <int WM_, int WN_, int NWM_, int NWN_, int RING_, bool AHEAD_> struct Shape {
  static constexpr int WM = WM_, WN = WN_, NWM = NWM_, NWN = NWN_, RING = RING_, NW = NWM * NWN, BM = 32 * WM * NWM, BN = 32 * WN * NWN;
  static constexpr bool AHEAD = AHEAD_;
  static constexpr size_t STAGE = 64 * (BM + BN), EPILOGUE = NW * 32 * (WN * 32 + 4) * 4;
};

template <typename T, typename SH, bool AO, bool BO>
__device__ __forceinline__ void product_block(const DmaArgs& g, int hw_block, unsigned char* lds) {
  constexpr int WM = SH::WM, WN = SH::WN, kRing = SH::RING;
  constexpr bool AHEAD = SH::AHEAD;
  constexpr int NWM = SH::NWM, NWN = SH::NWN, BM = SH::BM, BN = SH::BN;
  using A = DmaOperand<T, BM, NWM * NWN, AO>;
  using B = DmaOperand<T, BN, NWM * NWN, BO>;
  constexpr int STAGE = A::BYTES + B::BYTES, L = A::LOADS + B::LOADS;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int blk = xcd_remap(hw_block, g.per_xcd);
  if (blk >= g.n_blocks) return;
  // a band of tiles along M, then along N: the workgroups of an XCD that run together share the rows of few tiles of either operand
  const int tiles = g.tiles_m * g.tiles_n, s = blk / tiles, t = blk % tiles;
  const int band = t / (kBand * g.tiles_n), in_band = t % (kBand * g.tiles_n), high = min(kBand, g.tiles_m - band * kBand);
  const long long m0 = (long long)(band * kBand + in_band % high) * BM, n0 = (long long)(in_band / high) * BN;
  const LinearProduct& p = g.p;
  const long long begin = s * g.R_part, end = min(p.R, begin + g.R_part);
  const int nk = end > begin ? (int)((end - begin + kDeep<T> - 1) / kDeep<T>) : 0;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  A a;
  B b;
  a.start(p.a, p.lda, m0, p.M, begin, end, wave, lane);
  b.start(p.b, p.ldb, n0, p.N, begin, end, wave, lane);
  constexpr bool PAIR = !AHEAD;
  long long left = end - begin;
  int to = 0;                                       // slot of the ring of the next stage to be queued ...
  auto after = [](int slot) { return slot + 1 == kRing ? 0 : slot + 1; };
  auto queue = [&](int q) {                         // load q of the L of a stage, or of two
    const unsigned at = lds0 + to * STAGE, at2 = lds0 + after(to) * STAGE;
    if (q < A::LOADS) a.template queue<PAIR>(at, at2, wave, q);
    else b.template queue<PAIR>(at + A::BYTES, at2 + A::BYTES, wave, q - A::LOADS);
  };
  auto aim = [&] {
    a.template aim<PAIR>(left);
    b.template aim<PAIR>(left);
    left -= (PAIR ? 2 : 1) * kDeep<T>;
  };
  auto queue_next = [&] { to = PAIR ? after(after(to)) : after(to); aim(); };
  aim();

  const long long wm0 = m0 + wm * WM * 32, wn0 = n0 + wn * WN * 32;
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
  s16x8 va[2][WM], vb[2][WN];

  int now = 0;                                      // ... and of the stage that is multiplied
  if constexpr (AHEAD) {
    // One wavefront to a SIMD.  Three stages in flight; the first half of a stage is read while the last one of the stage before is multiplied
    static_assert(kRing == 4, "three stages in flight beside the one that is multiplied");
    if (nk > 0) {
#pragma unroll
      for (int k = 0; k < kRing - 1; ++k) {
        if (k >= nk) break;
#pragma unroll
        for (int q = 0; q < L; ++q) queue(q);
        queue_next();
      }
      if (nk >= 3) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(2 * L) : "memory");
      else if (nk == 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int i = 0; i < WM; ++i) va[0][i] = A::read(lds + fa[0][i]);
#pragma unroll
      for (int j = 0; j < WN; ++j) vb[0][j] = B::read(lds + fb[0][j]);
    }
#pragma unroll 1
    for (int ks = 0; ks < nk; ++ks) {
      // stage ks + 1 has landed, in flight may be that of ks + 2; nobody reads stage ks - 1 any more, which that of ks + 3 overwrites
      if (ks + 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const bool more = ks + kRing - 1 < nk;
      const int then = ks + 1 < nk ? after(now) : now;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const unsigned char* const st = lds + (kk ? then : now) * STAGE;      // of the half after this one
#pragma unroll
        for (int i = 0; i < WM; ++i) {
          va[kk ^ 1][i] = A::read(st + fa[kk ^ 1][i]);
          if (i < WN) vb[kk ^ 1][i] = B::read(st + fb[kk ^ 1][i]);
#pragma unroll
          for (int j = 0; j < WN; ++j) acc[i][j] = product(vb[kk][j], va[kk][i], acc[i][j], T{});
#pragma unroll
          for (int j = 0; j < WN; ++j) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (more) {
#pragma unroll
            for (int q = 0; q < L; ++q)
              if (q * 2 * WM / L == kk * WM + i) queue(q);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      now = after(now);
      if (more) queue_next();
    }
  } else {
    // Several wavefronts to a SIMD.  Stages are queued in pairs, load by load: the 64 bytes of a row and stage are half a line of the L2, whose other half
    // the load of the next stage finds in the L1 where it follows at once: an operand with the reduction innermost then comes at 120
    // bytes a ns and compute unit from the L2, at 64 otherwise (measured on loads alone).
    static_assert(kRing == 5, "a pair in flight and one that lands beside the stage that is multiplied");
    const int pairs = (nk + 1) / 2;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k >= pairs) break;
#pragma unroll
      for (int q = 0; q < L; ++q) queue(q);
      queue_next();
    }
    auto wait = [&](bool one_in_flight) {           // for all but the last pair, and for all wavefronts
      if (one_in_flight) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(2 * L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto step = [&](bool more) {
      const unsigned char* const st = lds + now * STAGE;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int i = 0; i < WM; ++i) va[kk][i] = A::read(st + fa[kk][i]);
#pragma unroll
        for (int j = 0; j < WN; ++j) vb[kk][j] = B::read(st + fb[kk][j]);
      }
      if (more) {
#pragma unroll
        for (int q = 0; q < L; ++q) queue(q);
        queue_next();
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
          for (int j = 0; j < WN; ++j) acc[i][j] = product(vb[kk][j], va[kk][i], acc[i][j], T{});
      now = after(now);
    };
#pragma unroll 1
    for (int j = 0; j < nk / 2; ++j) {
      // stages 2 j and 2 j + 1 have landed, in flight may be the pair after them
      wait(j + 1 < pairs);
      step(false);
      // nobody reads stages 2 j - 1 and 2 j any more: there goes the pair after the next
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      step(j + 2 < pairs);
    }
    if (nk & 1) {
      wait(false);
      step(false);
    }
  }

  if (g.parts) {
    store_parts<WM, WN>(g.parts + s * p.M * p.N, acc, wm0, p.M, wn0, p.N, g.vec, lane);
    return;
  }
  __syncthreads();                                          // the ring is done with
  float* const stage = reinterpret_cast<float*>(lds) + wave * 32 * (WN * 32 + 4);
  auto finish = [&](auto act, auto more) {
    if (m0 + BM <= p.M && n0 + BN <= p.N) finish_blocks<T, act(), true, more(), WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
    else finish_blocks<T, act(), false, more(), WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
  };
  // (a gradient has no epilogue, and the largest tiles, whose epilogue nothing runs beside, are left to products without a heavy one)
  if constexpr (BO || AHEAD) finish(ic<WC_ACT_NONE>{}, std::false_type{});
  else with_activation(p.e.act, [&](auto act) { finish(act, std::true_type{}); });
}

template <typename SH> constexpr int kMinWaves = SH::AHEAD ? 1 : 2;

template <typename T, typename SH, bool AO, bool BO>
__global__ __launch_bounds__(64 * SH::NW, kMinWaves<SH>) void product_dma_kernel(DmaArgs g) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  product_block<T, SH, AO, BO>(g, blockIdx.x, lds);
}

// Both gradients of a layer, which wait for nothing of each other: one launch less, and the last workgroups of one run beside the other's first
template <typename T, typename SH, typename SH2>
__global__ __launch_bounds__(256, 2) void product_pair_kernel(DmaArgs g, DmaArgs g2) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int n = g.per_xcd * kXcds;
  if ((int)blockIdx.x < n) product_block<T, SH, false, true>(g, blockIdx.x, lds);
  else product_block<T, SH2, true, true>(g2, blockIdx.x - n, lds);
}

DmaArgs dma_args(const LinearProduct& p, const ProductPlan& plan, float* parts) {
  DmaArgs g;
  g.p = p;
  g.parts = plan.s > 1 ? parts : nullptr;
  g.R_part = plan.R_part;
  g.tiles_m = (int)ceil_div_ll(p.M, plan.tile.m);
  g.tiles_n = (int)ceil_div_ll(p.N, plan.tile.n);
  g.n_blocks = g.tiles_m * g.tiles_n * plan.s;
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  g.vec = p.N % 4 == 0;
  return g;
}

// LDS of a product: the stages that its reduction has, and no less than the epilogue takes
template <typename T, typename SH>
size_t lds_of(const DmaArgs& g) {
  const long long pairs = std::max(1ll, ceil_div_ll(std::min(g.R_part, g.p.R), 2 * kDeep<T>)), stages = std::min<long long>(SH::RING, 2 * pairs);
  return std::max<size_t>((size_t)stages * SH::STAGE, SH::EPILOGUE);
}
template <typename SH> constexpr size_t kMostLds = SH::RING * SH::STAGE > SH::EPILOGUE ? SH::RING * SH::STAGE : SH::EPILOGUE;

// 256 x 256 with a heavy epilogue takes two wavefronts to a SIMD, one of which finishes results while the other waits for its own.  us, bf16
// 8192 x 2048 -> 8192, gelu with z: four wavefronts 343, eight 309 (128 x 128 349); 4096 x 4096 -> 4096, bias alone 122, 128 (153)
using Tile256 = Shape<4, 4, 2, 2, 4, true>;
using Tile256Heavy = Shape<4, 2, 2, 4, 5, false>;
using Tile128 = Shape<2, 2, 2, 2, 5, false>;
using Tile64 = Shape<1, 1, 2, 2, 5, false>;

template <typename T, typename SH>
int launch(const DmaArgs& g, void* stream) {
  const LinearProduct& p = g.p;
  auto fn = &product_dma_kernel<T, SH, false, false>;
  if constexpr (!std::is_same<SH, Tile256Heavy>::value) {      // (gradients have no epilogue)
    if (p.b_outer) fn = p.a_outer ? &product_dma_kernel<T, SH, true, true> : &product_dma_kernel<T, SH, false, true>;
  }
  if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(fn), kMostLds<SH>)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(64 * SH::NW), (lds_of<T, SH>(g)), as_stream(stream), g);
  WC_CHECK_LAUNCH("product_dma_kernel");
  return WC_OK;
}

template <typename T, typename SH, typename SH2>
int launch_pair(const DmaArgs& g, const DmaArgs& g2, void* stream) {
  auto fn = &product_pair_kernel<T, SH, SH2>;
  if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(fn), std::max(kMostLds<SH>, kMostLds<SH2>))) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)((g.per_xcd + g2.per_xcd) * kXcds)), dim3(256), (std::max(lds_of<T, SH>(g), lds_of<T, SH2>(g2))), as_stream(stream), g, g2);
  WC_CHECK_LAUNCH("product_pair_kernel");
  return WC_OK;
}

}  // namespace

// (rows longer than the reduction have zeros behind it up to a multiple of 16 bytes)
bool product_dma_fits(const LinearProduct& p, int dtype) {
  const int epc = dtype == WC_F32 ? 4 : 8;
  auto fits = [&](const void* q, long long ld, bool outer) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % epc == 0 && (outer || ceil_div_ll(p.R, epc) * epc <= ld) && ld < (1 << 21);
  };
  return fits(p.a, p.lda, p.a_outer) && fits(p.b, p.ldb, p.b_outer) && (!p.a_outer || p.b_outer);
}

int product_dma(const LinearProduct& p, const ProductPlan& plan, float* parts, int dtype, void* stream) {
  const DmaArgs g = dma_args(p, plan, parts);
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (plan.tile.m == 256) return linear_heavy(p.e) ? launch<T, Tile256Heavy>(g, stream) : launch<T, Tile256>(g, stream);
    }
    return plan.tile.m == 128 ? launch<T, Tile128>(g, stream) : launch<T, Tile64>(g, stream);
  });
}

bool product_dma_pairs(const ProductPlan& plan, const ProductPlan& plan2) { return plan.dma && plan2.dma && plan.tile.m <= 128 && plan2.tile.m <= 128; }

// p: the input gradient's (its second operand alone outer), p2: the weight gradient's
int product_dma_pair(const LinearProduct& p, const ProductPlan& plan, float* parts, const LinearProduct& p2, const ProductPlan& plan2, float* parts2, int dtype, void* stream) {
  const DmaArgs g = dma_args(p, plan, parts), g2 = dma_args(p2, plan2, parts2);
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (plan.tile.m == 128) return plan2.tile.m == 128 ? launch_pair<T, Tile128, Tile128>(g, g2, stream) : launch_pair<T, Tile128, Tile64>(g, g2, stream);
    return plan2.tile.m == 128 ? launch_pair<T, Tile64, Tile128>(g, g2, stream) : launch_pair<T, Tile64, Tile64>(g, g2, stream);
  });
}

}  // namespace wc
