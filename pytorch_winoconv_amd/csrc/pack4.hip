// Tensors in 4 bits (packed4.h): e = floor(log2(largest magnitude)) - 2 but at least -127, the OCP formats' rule - the largest value's
// exponent becomes that of 4, the largest of e2m1 -, and a value is the nearest code, ties to the even one, at most 6: values above 6 of the scale
// (a largest of 1.5 to 2 times its power of two) are off by up to a quarter, the others by at most half a step, 2^-2 of themselves at the least.
// A group with an infinity or a NaN has the scale 255 and reads as NaN.  Scales are powers of two, so v 2^-e is exact and the code does not
// hang on how a division rounds.
//
// Bound by memory: 8192 x 8192 bf16 33 us (5.2 TB/s) there, 37 back.  A workgroup takes 32 rows by two stages (256 channels), a thread eight channels four times, 16 bytes a load; four lanes
// share a group.
#include "packed4.h"

namespace wc {

namespace {

constexpr int kSpan = 2;                   // stages of a workgroup

struct Pack4Args {
  long long first;                         // workgroup of the launch
  const void* x;
  unsigned char* codes; unsigned char* scales;
  long long rows;
  int C, stages, spans;
};

// the exponent bits of a group's scale, from eight of its values in each of four neighbouring lanes
__device__ __forceinline__ unsigned group_scale4(const float (&v)[8]) {
  unsigned top = 0;                        // bits: a maximum of floats would drop a NaN
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = max(top, (unsigned)__shfl_xor((int)top, 1));
  top = max(top, (unsigned)__shfl_xor((int)top, 2));
  const unsigned bits = top >> 23;         // floor(log2) + 127, 0 below 2^-126
  return bits == 255 ? 255u : bits > 2 ? bits - 2 : 0u;
}

__device__ __forceinline__ unsigned word4(const float (&v)[8], unsigned e) {
  const float s = scale4(e);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  return e == 255 ? 0u : w;
}

template <typename T>
__global__ __launch_bounds__(256) void pack4_kernel(Pack4Args a) {
  const long long block = a.first + blockIdx.x, rb = block / a.spans;
  const int s0 = (int)(block - rb * a.spans) * kSpan, slot = threadIdx.x & 15;
  T x[2][kSpan][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < kSpan; ++k) {
      const long long row = rb * kRows4 + i * 16 + (threadIdx.x >> 4);
      const int c = (s0 + k) * kStage4 + slot * 8;
      load_run<T, 8>(a.x, row * a.C + c, row < a.rows ? max(min(a.C - c, 8), 0) : 0, x[i][k]);
    }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < kSpan; ++k) {
      const int r = i * 16 + (threadIdx.x >> 4), stage = s0 + k;
      const long long row = rb * kRows4 + r;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(x[i][k][e]);
      const unsigned e = group_scale4(v), w = word4(v, e);
      if (stage >= a.stages) continue;
      if (row < a.rows) *reinterpret_cast<unsigned*>(a.codes + (row * a.stages + stage) * (kStage4 / 2) + slot * 4) = w;
      if ((slot & 3) == 0) a.scales[(rb * a.stages + stage) * (kRows4 * 4) + r * 4 + slot / 4] = (unsigned char)e;      // (rows behind the last: 0)
    }
}

template <typename T>
__global__ __launch_bounds__(256) void unpack4_kernel(Pack4Args a, void* out) {
  const long long block = a.first + blockIdx.x, rb = block / a.spans;
  const int s0 = (int)(block - rb * a.spans) * kSpan, slot = threadIdx.x & 15;
  unsigned w[2][kSpan], e[2][kSpan];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < kSpan; ++k) {
      const int r = i * 16 + (threadIdx.x >> 4), stage = min(s0 + k, a.stages - 1);
      const long long row = min(rb * kRows4 + r, a.rows - 1);
      w[i][k] = *reinterpret_cast<const unsigned*>(a.codes + (row * a.stages + stage) * (kStage4 / 2) + slot * 4);
      e[i][k] = a.scales[scale_at4(row, (long long)stage * 4 + slot / 4, a.stages)];
    }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < kSpan; ++k) {
      const long long row = rb * kRows4 + i * 16 + (threadIdx.x >> 4);
      const int c = (s0 + k) * kStage4 + slot * 8;
      T v[8];
      values4<T>(w[i][k], scale4(e[i][k]), v);
      store_run<T, 8>(out, row * a.C + c, row < a.rows ? max(min(a.C - c, 8), 0) : 0, v);
    }
}

Pack4Args args_of(const void* x, const unsigned char* codes, const unsigned char* scales, long long rows, int C) {
  const int stages = (int)stages4(C);
  return {0, x, const_cast<unsigned char*>(codes), const_cast<unsigned char*>(scales), rows, C, stages, ceil_div(stages, kSpan)};
}

}  // namespace

int pack4(const void* x, unsigned char* codes, unsigned char* scales, long long rows, int C, int dtype, void* stream) {
  Pack4Args a = args_of(x, codes, scales, rows, C);
  return dispatch_dtype(dtype, [&](auto t) {
    return in_launches(ceil_div_ll(rows, kRows4) * a.spans, [&](long long first, unsigned blocks) -> int {
      a.first = first;
      hipLaunchKernelGGL(pack4_kernel<decltype(t)>, dim3(blocks), dim3(256), 0, as_stream(stream), a);
      WC_CHECK_LAUNCH("pack4_kernel");
      return WC_OK;
    });
  });
}

int unpack4(const unsigned char* codes, const unsigned char* scales, void* x, long long rows, int C, int dtype, void* stream) {
  Pack4Args a = args_of(nullptr, codes, scales, rows, C);
  return dispatch_dtype(dtype, [&](auto t) {
    return in_launches(ceil_div_ll(rows, kRows4) * a.spans, [&](long long first, unsigned blocks) -> int {
      a.first = first;
      hipLaunchKernelGGL(unpack4_kernel<decltype(t)>, dim3(blocks), dim3(256), 0, as_stream(stream), a, x);
      WC_CHECK_LAUNCH("unpack4_kernel");
      return WC_OK;
    });
  });
}

}  // namespace wc
