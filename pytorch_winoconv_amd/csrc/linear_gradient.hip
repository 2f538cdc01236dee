// What stands before and behind the products of a layer's gradient, one launch each: small kernels of their own cost a few us apiece.
//
// Before them, dz = dy act'(z) in the storage type - the operand of both products, and the gradient of the layer's residual - and the column sums
// of dz before that rounding (the bias gradient), in one read of dy and z, which bounds it: a workgroup takes a run of rows and some
// columns, a thread eight neighbouring ones (16 bytes of 16-bit types, wherever they start) with fp32 sums in registers; the threads of a column
// meet in LDS.  The rounding of dz is what the matrix cores take; two products with an unrounded one would be fp32's, at a ninth of the rate.  It makes the
// error of the 16-bit gradients of gelu and silu 1.4 times as large (2-norm, bf16 0.0017 -> 0.0023); relu's and a plain layer's dz are not rounded by it.
// Beside it the copies of operands whose rows are no multiple of 16 bytes, and activations that were kept in 8 bits.
// Behind them, the sums of the parts of a product's reduction and of the workgroups' columns, all in a fixed order.
#include "linear_rows.h"

#include <algorithm>

namespace wc {

namespace {

constexpr int kThreads = 256;

constexpr int VEC = 8;

struct SlopeArgs {
  LinearSlope s;
  float* part;               // (blocks, K); null: no sums, or one block, whose sums are db
  long long rows_per_block;
  int cols, groups;          // threads side by side, rows in flight
};

template <typename T>
__device__ __forceinline__ void store_sum(const LinearSlope& l, int k, float v) {
  if (l.db_f32) static_cast<float*>(l.db)[k] = v;
  else static_cast<T*>(l.db)[k] = static_cast<T>(v);
}

template <typename T, int ACT, bool PACKED>
__device__ __forceinline__ void slope_rows(const SlopeArgs& a, int k, long long begin, long long end, float (&s)[VEC]) {
  const LinearSlope& l = a.s;
  const long long n_groups = pack_groups(l.K);
  const int have = max(min(l.K - k, VEC), 0);
  constexpr int AHEAD = 4;                        // rows asked for before the first is used
  auto rows = [&](auto full, long long r0, int n) {
    const int h = full() ? VEC : have;
    T dy[AHEAD][VEC], v[AHEAD][VEC];
    signed char q[AHEAD][VEC];
    int e8[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (j >= n) break;
      const long long r = r0 + j * a.groups, i = r * l.K + k;
      load_run<T, VEC>(l.dy, i, h, dy[j]);
      if constexpr (ACT != WC_ACT_NONE && PACKED) {
        load_run<signed char, VEC>(l.z, i, h, q[j]);
        e8[j] = h > 0 ? l.z_exp[r * n_groups + k / kPackGroup] : 0;
      } else if constexpr (ACT != WC_ACT_NONE) {
        load_run<T, VEC>(l.z, i, h, v[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (j >= n) break;
      const long long r = r0 + j * a.groups;
      T dz[VEC];
      float step = 0.f;
      if constexpr (ACT != WC_ACT_NONE && PACKED) step = ACT == WC_ACT_RELU ? gate_step(e8[j]) : pack_step(e8[j]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float z = 0.f;
        if constexpr (ACT != WC_ACT_NONE && PACKED) z = (float)q[j][e] * step;
        else if constexpr (ACT != WC_ACT_NONE) z = static_cast<float>(v[j][e]);
        const float g = full() || e < have ? through(static_cast<float>(dy[j][e]), z, ACT) : 0.f;
        s[e] += g;
        dz[e] = static_cast<T>(g);
      }
      if (l.dz) store_run<T, VEC>(l.dz, r * l.K + k, h, dz);
      if (l.dz_wide) store_run<T, VEC>(l.dz_wide, r * l.ld_wide + k, full() ? VEC : (int)min(l.ld_wide - k, (long long)VEC), dz);
    }
  };
  auto all = [&](auto full) {
    long long r = begin;
    for (; r + (AHEAD - 1) * a.groups < end; r += AHEAD * a.groups) rows(full, r, AHEAD);
    for (; r < end; r += a.groups) rows(full, r, 1);
  };
  if (have == VEC) all(std::true_type{});
  else all(std::false_type{});
}

template <typename T>
__device__ __forceinline__ void slope_block(const SlopeArgs& a, int block, int tile, float* sums) {
  constexpr int PITCH = VEC + 1;
  const LinearSlope& l = a.s;
  const int group = threadIdx.x / a.cols, col = threadIdx.x - group * a.cols;
  const int k = (tile * a.cols + col) * VEC;
  const long long begin = block * a.rows_per_block, end = min(l.rows, begin + a.rows_per_block);
  float s[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = 0.f;
  if (k < l.K) {
    auto run = [&](auto act) {
      if (act() != WC_ACT_NONE && l.z_exp) slope_rows<T, act(), true>(a, k, begin + group, end, s);
      else slope_rows<T, act(), false>(a, k, begin + group, end, s);
    };
    switch (l.act) {
      case WC_ACT_RELU: run(ic<WC_ACT_RELU>{}); break;
      case WC_ACT_GELU: run(ic<WC_ACT_GELU>{}); break;
      case WC_ACT_GELU_TANH: run(ic<WC_ACT_GELU_TANH>{}); break;
      case WC_ACT_SILU: run(ic<WC_ACT_SILU>{}); break;
      default: run(ic<WC_ACT_NONE>{});
    }
  }
  if (!l.db) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sums[threadIdx.x * PITCH + e] = s[e];
  __syncthreads();
  for (int i = threadIdx.x; i < a.cols * VEC; i += kThreads) {
    const int c = i / VEC, e = i % VEC, kk = (tile * a.cols + c) * VEC + e;
    if (kk >= l.K) continue;
    float t = 0.f;
    for (int g = 0; g < a.groups; ++g) t += sums[(g * a.cols + c) * PITCH + e];
    if (a.part) a.part[(long long)block * l.K + kk] = t;
    else store_sum<T>(l, kk, t);
  }
}

struct PrepareArgs {
  long long first;                     // workgroup of this launch
  SlopeArgs slope;
  int slope_blocks, slope_tiles;       // none: 0
  WideCopy copies[2];
  long long copy_blocks[2];
  UnpackArgs unpack;
  int line;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void prepare_kernel(PrepareArgs a) {
  __shared__ float sums[kThreads * (VEC + 1)];
  long long b = a.first + blockIdx.x;
  const long long n = (long long)a.slope_blocks * a.slope_tiles;
  if (b < n) return slope_block<T>(a.slope, (int)(b / a.slope_tiles), (int)(b % a.slope_tiles), sums);
  b -= n;
  if (b < a.copy_blocks[0]) return widen_block<T>(a.copies[0], b);
  b -= a.copy_blocks[0];
  if (b < a.copy_blocks[1]) return widen_block<T>(a.copies[1], b);
  b -= a.copy_blocks[1];
  if (a.line) unpack_line_block<T>(a.unpack, b);
  else unpack_block<T>(a.unpack, b);
}

struct JoinArgs {
  LinearJoin join[2];
  long long blocks[2];
  LinearSlope slope;
  const float* sums;
  int sum_rows;
};

// four neighbouring results a thread: the parts' sums in their order, and the epilogue
template <typename T>
__device__ __forceinline__ void join_block(const LinearJoin& j, long long block) {
  const long long total = j.M * j.N, i = (block * kThreads + threadIdx.x) * 4;
  if (i >= total) return;
  const int have = (int)min(total - i, 4ll);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (have == 4 && total % 4 == 0) {
#pragma unroll 8
    for (int s = 0; s < j.s; ++s) {
      const float4 p = *reinterpret_cast<const float4*>(j.parts + s * total + i);
      v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
    }
  } else {
    for (int s = 0; s < j.s; ++s) {
      float p[4];
      load_run<float, 4>(j.parts, s * total + i, have, p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
  }
  const LinearEpilogue& e = j.e;
  T r[4], z[4], y[4];
  if (e.res) load_run<T, 4>(e.res, i, have, r);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float res = e.res ? static_cast<float>(r[k]) : 0.f;
    if (e.bias) v[k] += static_cast<float>(static_cast<const T*>(e.bias)[min(i + k, total - 1) % j.N]);
    if (!e.res_after) v[k] += res;
    z[k] = static_cast<T>(v[k]);
    v[k] = activate(v[k], e.act);
    if (e.res_after) v[k] += res;
    y[k] = static_cast<T>(v[k]);
  }
  if (e.z) store_run<T, 4>(e.z, i, have, z);
  if (e.y_f32) store_run<float, 4>(e.y, i, have, v);
  else store_run<T, 4>(e.y, i, have, y);
}

// db[k] = the sum of the workgroups' sums; 16 channels a workgroup, 16 threads to a channel's
template <typename T>
__device__ __forceinline__ void sums_block(const LinearSlope& l, const float* part, int rows, int block, float* lds) {
  const int c = threadIdx.x & 15, group = threadIdx.x >> 4, k = block * 16 + c;
  float s = 0.f;
  if (k < l.K) {
#pragma unroll 8
    for (int b = group; b < rows; b += 16) s += part[(long long)b * l.K + k];
  }
  lds[threadIdx.x] = s;
  __syncthreads();
  for (int half = 8; half > 0; half >>= 1) {
    if (group < half) lds[threadIdx.x] += lds[threadIdx.x + half * 16];
    __syncthreads();
  }
  if (group == 0 && k < l.K) store_sum<T>(l, k, lds[c]);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(JoinArgs a) {
  __shared__ float lds[kThreads];
  long long b = blockIdx.x;
  if (b < a.blocks[0]) return join_block<T>(a.join[0], b);
  b -= a.blocks[0];
  if (b < a.blocks[1]) return join_block<T>(a.join[1], b);
  sums_block<T>(a.slope, a.sums, a.sum_rows, (int)(b - a.blocks[1]), lds);
}

struct SlopePlan { int cols, col_tiles, groups, blocks; long long rows_per_block; };
// As many columns side by side as leave four workgroups to a compute unit; two of them run at a time, since the bodies of all activations in one kernel
// take 231 registers
SlopePlan slope_plan(long long rows, int K) {
  SlopePlan p;
  for (p.cols = kThreads;; p.cols /= 2) {
    p.groups = kThreads / p.cols;
    p.col_tiles = ceil_div(ceil_div(K, VEC), p.cols);
    const long long most = std::max(1ll, rows / p.groups), blocks = std::min<long long>(most, ceil_div(4 * kCus, p.col_tiles));
    p.rows_per_block = ceil_div_ll(rows, blocks);
    p.blocks = (int)ceil_div_ll(rows, p.rows_per_block);
    if (p.cols == 16 || (ceil_div(K, VEC) > p.cols / 2 && (long long)p.col_tiles * blocks >= 4 * kCus)) return p;
  }
}

}  // namespace

size_t linear_sums_bytes(const LinearSlope& s) {
  const int blocks = slope_plan(s.rows, s.K).blocks;
  return s.db && blocks > 1 ? (size_t)blocks * s.K * 4 : 0;
}

int linear_prepare(const LinearPrepare& p, int dtype, float* sums, void* stream) {
  PrepareArgs a = {};
  if (p.run_slope) {
    const SlopePlan l = slope_plan(p.slope.rows, p.slope.K);
    a.slope = {p.slope, p.slope.db && l.blocks > 1 ? sums : nullptr, l.rows_per_block, l.cols, l.groups};
    a.slope_blocks = l.blocks;
    a.slope_tiles = l.col_tiles;
  }
  for (int i = 0; i < p.n_copies; ++i) {
    a.copies[i] = p.copies[i];
    a.copy_blocks[i] = widen_blocks(p.copies[i]);
  }
  long long n = (long long)a.slope_blocks * a.slope_tiles + a.copy_blocks[0] + a.copy_blocks[1];
  if (p.codes) {
    const int rg = (int)pack_groups(p.x_C);
    a.unpack = {0, p.codes, p.exps, p.x, p.x_rows * rg, p.x_ld, p.x_C, rg};
    a.line = p.x_ld == p.x_C && on_a_line(p.x_C, p.x, p.codes);
    n += unpack_blocks(a.unpack, a.line != 0);
  }
  return dispatch_dtype(dtype, [&](auto t) {
    return in_launches(n, [&](long long first, unsigned blocks) -> int {
      a.first = first;
      hipLaunchKernelGGL(prepare_kernel<decltype(t)>, dim3(blocks), dim3(kThreads), 0, as_stream(stream), a);
      WC_CHECK_LAUNCH("prepare_kernel");
      return WC_OK;
    });
  });
}

int linear_join(const LinearJoin* joins, int n, const LinearSlope* slope, const float* sums, int dtype, void* stream) {
  JoinArgs a = {};
  long long blocks = 0;
  for (int i = 0; i < n; ++i) {
    a.join[i] = joins[i];
    a.blocks[i] = joins[i].s > 1 ? ceil_div_ll(joins[i].M * joins[i].N, 4 * kThreads) : 0;
    blocks += a.blocks[i];
  }
  if (slope && linear_sums_bytes(*slope)) {
    a.slope = *slope;
    a.sums = sums;
    a.sum_rows = slope_plan(slope->rows, slope->K).blocks;
    blocks += ceil_div(slope->K, 16);
  }
  if (blocks == 0) return WC_OK;      // (parts are of few results, and the columns no more than 2^24: one launch holds them)
  return dispatch_dtype(dtype, [&](auto t) -> int {
    hipLaunchKernelGGL(join_kernel<decltype(t)>, dim3((unsigned)blocks), dim3(kThreads), 0, as_stream(stream), a);
    WC_CHECK_LAUNCH("join_kernel");
    return WC_OK;
  });
}

}  // namespace wc
