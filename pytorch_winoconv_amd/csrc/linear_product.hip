// The products of a linear layer and of its gradients, D (M, N) = sum over R of A (x) B with an epilogue, operands with the reduction
// axis innermost (x and w of the forward pass, dz of the input gradient) or outermost (w of the input gradient, dz and x of the weight
// gradient), in any size and at any alignment.
//
// 64 x 64 results per workgroup, a 32 x 32 block of the matrix cores per wavefront; a stage of the reduction is brought to LDS with the
// reduction innermost, whichever way it lies.  Where there are few tiles the reduction is cut into parts, whose fp32 sums a second kernel
// adds in a fixed order before the epilogue.
#include "linear.h"

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
  bool vec_a, vec_b;          // 16-byte loads
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

template <typename T>
__global__ __launch_bounds__(256) void product_general_kernel(GeneralArgs g) {
  constexpr int EPC = 16 / sizeof(T), BK = 4 * EPC, PITCH = BK + EPC;       // 64 bytes of a row and stage
  __shared__ __attribute__((aligned(16))) T tile[2][64 * PITCH];
  const int blk = xcd_remap(blockIdx.x, g.per_xcd);
  if (blk >= g.n_blocks) return;
  const int tn = blk % g.tiles_n, tm = blk / g.tiles_n % g.tiles_m, s = blk / (g.tiles_n * g.tiles_m);
  const LinearProduct& p = g.p;
  const long long m0 = (long long)tm * 64, n0 = (long long)tn * 64;
  const long long begin = s * g.R_part, end = min(p.R, begin + g.R_part);
  const int tid = threadIdx.x;

  // EPC elements a thread: of one row along the reduction, or of one reduction element along the rows
  auto load = [&](const void* src, long long ld, bool outer, bool vec, long long row0, long long rows, long long k0, T (&v)[EPC]) {
    const long long r = row0 + (outer ? tid % (64 / EPC) * EPC : tid / 4), k = k0 + (outer ? tid / (64 / EPC) : tid % 4 * EPC);
    const T* q = static_cast<const T*>(src) + (outer ? k * ld + r : r * ld + k);
    const long long have = outer ? (k < end ? rows - r : 0) : (r < rows ? end - k : 0);
    if (vec && have >= EPC) {
      const Pack<T, EPC> w = *reinterpret_cast<const Pack<T, EPC>*>(q);
#pragma unroll
      for (int e = 0; e < EPC; ++e) v[e] = w.v[e];
    } else {
#pragma unroll
      for (int e = 0; e < EPC; ++e) v[e] = e < have ? q[e] : static_cast<T>(0.f);
    }
  };
  auto store = [&](T* to, bool outer, const T (&v)[EPC]) {
    if (outer) {
#pragma unroll
      for (int e = 0; e < EPC; ++e) to[(tid % (64 / EPC) * EPC + e) * PITCH + tid / (64 / EPC)] = v[e];
    } else {
      Pack<T, EPC> w;
#pragma unroll
      for (int e = 0; e < EPC; ++e) w.v[e] = v[e];
      *reinterpret_cast<Pack<T, EPC>*>(to + tid / 4 * PITCH + tid % 4 * EPC) = w;
    }
  };

  const int lane = tid & 63, wave = tid >> 6, l32 = lane & 31, lhi = lane >> 5;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x16 acc = {};
  T va[EPC], vb[EPC];
  if (begin < end) {
    load(p.a, p.lda, p.a_outer, g.vec_a, m0, p.M, begin, va);
    load(p.b, p.ldb, p.b_outer, g.vec_b, n0, p.N, begin, vb);
  }
  for (long long k0 = begin; k0 < end; k0 += BK) {
    __syncthreads();
    store(tile[0], p.a_outer, va);
    store(tile[1], p.b_outer, vb);
    __syncthreads();
    if (k0 + BK < end) {
      load(p.a, p.lda, p.a_outer, g.vec_a, m0, p.M, k0 + BK, va);
      load(p.b, p.ldb, p.b_outer, g.vec_b, n0, p.N, k0 + BK, vb);
    }
    const T* const ra = tile[0] + (wm + l32) * PITCH;
    const T* const rb = tile[1] + (wn + l32) * PITCH;
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

// the parts' sums added in their order, and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(LinearEpilogue e, const float* __restrict__ parts, int S, long long M, long long N) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * N) return;
  float v = 0.f;
#pragma unroll 4
  for (int s = 0; s < S; ++s) v += parts[s * M * N + i];
  finish<T>(e, i / N, i % N, N, v);
}

// Tiles of 64 w x 64 w (w = 1: product_general_kernel, too), s parts of the reduction
struct ProductPlan { bool dma; int w, s; long long R_part; };

ProductPlan plan_of(const LinearProduct& p, bool dma) {
  ProductPlan l = {dma, 1, 1, 0};
  auto tiles = [&](int w) { return ceil_div_ll(p.M, 64 * w) * ceil_div_ll(p.N, 64 * w); };
  if (l.dma) l.w = tiles(4) >= kCus ? 4 : tiles(2) >= kCus / 4 ? 2 : 1;
  // as many as bring two (w = 2) or four tiles to a compute unit, of 256 elements and more, within 256 MB of sums
  long long s = l.w == 4 ? 1 : std::min((l.w == 2 ? 2 : 4) * kCus / std::max(tiles(l.w), 1ll), std::max(p.R / 256, 1ll));
  s = std::max(1ll, std::min(s, (256ll << 20) / std::max(4 * p.M * p.N, 1ll)));
  l.R_part = std::max(64ll, ceil_div_ll(ceil_div_ll(p.R, s), 64) * 64);
  l.s = (int)std::max(1ll, ceil_div_ll(p.R, l.R_part));
  return l;
}

bool vectors(const void* p, long long ld, int es) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0; }

}  // namespace

// (where the operands start is not known yet)
size_t linear_product_bytes(const LinearProduct& p, int) {
  const int s = std::max(plan_of(p, true).s, plan_of(p, false).s);
  return s > 1 ? (size_t)s * p.M * p.N * 4 : 0;
}

int linear_product(const LinearProduct& p, int dtype, void* workspace, void* stream) {
  const int es = dtype == WC_F32 ? 4 : 2;
  const ProductPlan l = plan_of(p, product_dma_fits(p, dtype));
  const long long tiles = ceil_div_ll(p.M, 64 * l.w) * ceil_div_ll(p.N, 64 * l.w);
  if (tiles * l.s >= (1ll << 31) - 8 || ceil_div_ll(p.M * p.N, 256) >= (1ll << 31)) return fail(WC_ERR_UNSUPPORTED, "a product of %lld x %lld has too many tiles", p.M, p.N);
  float* const parts = l.s > 1 ? static_cast<float*>(workspace) : nullptr;
  if (l.dma) {
    if (int rc = product_dma(p, l.w, l.s, l.R_part, parts, dtype, stream)) return rc;
  }
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (!l.dma) {
      GeneralArgs g;
      g.p = p;
      g.parts = parts;
      g.R_part = l.R_part;
      g.tiles_m = (int)ceil_div_ll(p.M, 64); g.tiles_n = (int)ceil_div_ll(p.N, 64);
      g.n_blocks = (int)(tiles * l.s);
      g.per_xcd = ceil_div(g.n_blocks, kXcds);
      g.vec_a = vectors(p.a, p.lda, es);
      g.vec_b = vectors(p.b, p.ldb, es);
      hipLaunchKernelGGL(product_general_kernel<T>, dim3((unsigned)(g.per_xcd * kXcds)), dim3(256), 0, as_stream(stream), g);
      WC_CHECK_LAUNCH("product_general_kernel");
    }
    if (parts) {
      hipLaunchKernelGGL(product_join_kernel<T>, dim3((unsigned)ceil_div_ll(p.M * p.N, 256)), dim3(256), 0, as_stream(stream), p.e, parts, l.s, p.M, p.N);
      WC_CHECK_LAUNCH("product_join_kernel");
    }
    return WC_OK;
  });
}

}  // namespace wc
