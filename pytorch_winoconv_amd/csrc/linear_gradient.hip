// What the activation's derivative makes of dy: dz = dy act'(z) in the storage type - the operand of both products of a layer's
// gradient, and the gradient of its residual -, and the column sums of dz before that rounding (the bias gradient), in one read of dy and z.
//
// Bound by that read.  A workgroup takes a run of rows, a thread VEC neighbouring columns with fp32 sums in registers; the threads of a column
// meet in LDS, the workgroups in a second kernel, all in a fixed order.
#include "linear.h"

#include <algorithm>

namespace wc {

namespace {

constexpr int kSlopeThreads = 256;

struct SlopeArgs {
  LinearSlope s;
  float* part;               // (blocks, K); null: no sums
  long long rows_per_block;
  int cols, groups;          // threads side by side, rows in flight
};

template <typename T, int VEC>
__global__ __launch_bounds__(kSlopeThreads) void slope_kernel(SlopeArgs a) {
  __shared__ float sums[kSlopeThreads * (VEC + (VEC > 1))];
  constexpr int PITCH = VEC + (VEC > 1);
  const LinearSlope& l = a.s;
  const int group = threadIdx.x / a.cols, col = threadIdx.x - group * a.cols;
  const int k = (blockIdx.y * a.cols + col) * VEC;
  const long long begin = blockIdx.x * a.rows_per_block, end = min(l.rows, begin + a.rows_per_block);
  const long long n_groups = pack_groups(l.K);
  float s[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = 0.f;
  if (group < a.groups && k < l.K) {
#pragma unroll 2
    for (long long r = begin + group; r < end; r += a.groups) {
      const long long i = r * l.K + k;
      const Pack<T, VEC> dy = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(l.dy) + i);
      Pack<T, VEC> dz;
      float z[VEC];
      if (l.act == WC_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = 0.f;
      } else if (l.z_exp) {
        const Pack<signed char, VEC> q = *reinterpret_cast<const Pack<signed char, VEC>*>(static_cast<const signed char*>(l.z) + i);
        const float step = pack_step(l.z_exp[r * n_groups + k / kPackGroup]);      // (VEC divides the group)
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = (float)q.v[e] * step;
      } else {
        const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(l.z) + i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = static_cast<float>(v.v[e]);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = through(static_cast<float>(dy.v[e]), z[e], l.act);
        s[e] += v;
        dz.v[e] = static_cast<T>(v);
      }
      if (l.dz) *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(l.dz) + i) = dz;
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sums[threadIdx.x * PITCH + e] = s[e];
  __syncthreads();
  for (int i = threadIdx.x; i < a.cols * VEC; i += kSlopeThreads) {
    const int c = i / VEC, e = i - c * VEC;
    const int kk = (blockIdx.y * a.cols + c) * VEC + e;
    if (kk >= l.K) continue;
    float t = 0.f;
    for (int g = 0; g < a.groups; ++g) t += sums[(g * a.cols + c) * PITCH + e];
    a.part[(long long)blockIdx.x * l.K + kk] = t;
  }
}

// db[k] = sum over the workgroups' rows; 16 channels a workgroup, 64 threads to a channel's sums
template <typename T>
__global__ __launch_bounds__(1024) void slope_sums_kernel(const float* __restrict__ part, void* __restrict__ db, int blocks, int K, bool f32) {
  __shared__ float sums[64][16];
  const int c = threadIdx.x & 15, group = threadIdx.x >> 4, k = blockIdx.x * 16 + c;
  float s = 0.f;
  if (k < K) {
#pragma unroll 4
    for (int b = group; b < blocks; b += 64) s += part[(long long)b * K + k];
  }
  sums[group][c] = s;
  __syncthreads();
  for (int half = 32; half > 0; half >>= 1) {
    if (group < half) sums[group][c] += sums[group + half][c];
    __syncthreads();
  }
  if (group || k >= K) return;
  if (f32) static_cast<float*>(db)[k] = sums[0][c];
  else static_cast<T*>(db)[k] = static_cast<T>(sums[0][c]);
}

struct SlopePlan { int vec, cols, col_tiles, groups, blocks; long long rows_per_block; };
SlopePlan slope_plan(long long rows, int K, int es, bool aligned) {
  SlopePlan p;
  p.vec = aligned && K * es % 16 == 0 ? 16 / es : 1;
  const int n = K / p.vec;
  p.cols = std::min(n, kSlopeThreads);
  p.col_tiles = ceil_div(n, p.cols);
  p.groups = kSlopeThreads / p.cols;
  // 32 KB of dy a workgroup, at most two rounds of the eight that a CU holds
  const long long blocks = std::max(1ll, std::min(std::max(1ll, 4096ll / p.col_tiles), rows * K * es / p.col_tiles / 32768));
  p.rows_per_block = ceil_div_ll(rows, blocks);
  p.blocks = (int)ceil_div_ll(rows, p.rows_per_block);
  return p;
}

}  // namespace

size_t linear_slope_bytes(const LinearSlope& s, int dtype) {
  if (!s.db) return 0;
  const int es = dtype == WC_F32 ? 4 : 2;
  return (size_t)std::max(slope_plan(s.rows, s.K, es, true).blocks, slope_plan(s.rows, s.K, es, false).blocks) * s.K * 4;
}

int linear_slope(const LinearSlope& s, int dtype, void* part, void* stream) {
  const int es = dtype == WC_F32 ? 4 : 2;
  const bool aligned = (reinterpret_cast<uintptr_t>(s.dy) | reinterpret_cast<uintptr_t>(s.z) | reinterpret_cast<uintptr_t>(s.dz)) % 16 == 0;
  const SlopePlan p = slope_plan(s.rows, s.K, es, aligned);
  const SlopeArgs a = {s, s.db ? static_cast<float*>(part) : nullptr, p.rows_per_block, p.cols, p.groups};
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    constexpr int FULL = 16 / sizeof(T);
    hipLaunchKernelGGL((p.vec == FULL ? &slope_kernel<T, FULL> : &slope_kernel<T, 1>), dim3((unsigned)p.blocks, (unsigned)p.col_tiles), dim3(kSlopeThreads), 0, as_stream(stream), a);
    WC_CHECK_LAUNCH("slope_kernel");
    if (s.db) {
      hipLaunchKernelGGL(slope_sums_kernel<T>, dim3((unsigned)ceil_div(s.K, 16)), dim3(1024), 0, as_stream(stream), a.part, s.db, p.blocks, s.K, s.db_f32 != 0);
      WC_CHECK_LAUNCH("slope_sums_kernel");
    }
    return WC_OK;
  });
}

}  // namespace wc
