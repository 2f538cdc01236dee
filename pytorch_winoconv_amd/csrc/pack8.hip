// Activations in 8 bits for the backward pass: the groups of 32 neighbouring channels of a row share a step 2^e, e = floor(log2(largest
// magnitude)) - 6 but at least -126, and a value v is the whole number q nearest to v 2^-e (ties to even), at most 127 either way.
//
// The steps are powers of two, so v 2^-e is exact, q does not hang on how a division rounds, and q 2^e is exact in every type a group came
// from: it has seven bits, lies between the type's smallest number and its largest (127 2^(e) is below 2^(e + 7), where the group's largest
// value has its exponent), which steps rounded up to hold 128 2^e would exceed.  A value is off by at most half a step, 2^-7 of the group's
// largest, but for those above 127.5 steps, which are off by less than one, 2^-7 of themselves; half a step is no less than 2^-127, so that groups
// whose largest is below 2^-120 (fp32 and bf16) lose more of it and those of up to 2^-127 read as 0.  Against a floating type of 8 bits with three
// bits of mantissa (off by 2^-4 of the value) the large values of a group, which are most of the sums they enter, are eight times as exact.
// A group with an infinity or a NaN has the exponent 127 and reads as NaN throughout, so that such values still show in the gradients.
// keep_sign: values other than zero keep a code other than zero, one step - for what is read by its sign alone.
// kPackGates, for the gate of a ReLU: the codes of a group with an infinity or a NaN are 1 above zero, -1 for the rest and 0 for a NaN, so that its
// other channels keep their gates.
//
// Bound by memory.  Rows of whole groups are one line of groups: a thread takes eight neighbouring elements four times, 16 bytes a load, and
// four threads a group.  Other rows take eight threads a group, four elements each, wherever they start.
#include "linear_rows.h"

#include <algorithm>

namespace wc {

namespace {

struct PackArgs {
  long long first;           // workgroup of the launch
  const void* x;
  signed char* codes; signed char* exps;
  long long groups;          // of all rows
  int C, row_groups;
  int keep_sign;
};

__device__ __forceinline__ int pack_exponent(float top) {
  const int bits = (int)(__float_as_uint(top) >> 23);          // top >= 0
  return bits == 255 ? kPackNoNumber : max(bits - 127 - 6, kPackLeast);
}
// 2^-e is a normal number for every e there is but NoNumber, whose codes are read as gates alone
__device__ __forceinline__ int pack_code(float v, int e, int keep_sign) {
  if (e == kPackNoNumber) return keep_sign == kPackGates ? (v > 0.f ? 1 : v <= 0.f ? -1 : 0) : 0;
  const float q = fminf(fmaxf(rintf(v * __uint_as_float((unsigned)(127 - e) << 23)), -127.f), 127.f);
  return keep_sign && q == 0.f && v != 0.f ? (v > 0.f ? 1 : -1) : (int)q;
}

// the exponent of a group from N of its elements in each of 32 / N neighbouring lanes
template <typename T, int N>
__device__ __forceinline__ int group_exponent(const T (&x)[N]) {
  unsigned top = 0;                                        // bits: a maximum of floats would drop a NaN
#pragma unroll
  for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(static_cast<float>(x[e])) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < kPackGroup / N; d <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
  return pack_exponent(__uint_as_float(top));
}

template <typename T>
__global__ __launch_bounds__(256) void pack8_line_kernel(PackArgs a) {
  const long long total = a.groups * kPackGroup, first = (a.first + blockIdx.x) * kLine + threadIdx.x * 8;
  T x[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) load_run<T, 8>(a.x, first + j * 2048, first + j * 2048 < total ? 8 : 0, x[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long i = first + j * 2048;
    const int e = group_exponent<T, 8>(x[j]);
    Pack<signed char, 8> q;
#pragma unroll
    for (int k = 0; k < 8; ++k) q.v[k] = (signed char)pack_code(static_cast<float>(x[j][k]), e, a.keep_sign);
    if (i >= total) continue;
    *reinterpret_cast<Pack<signed char, 8>*>(a.codes + i) = q;
    if ((threadIdx.x & 3) == 0) a.exps[i / kPackGroup] = (signed char)e;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void pack8_kernel(PackArgs a) {
  const long long g = ((a.first + blockIdx.x) * 256 + threadIdx.x) >> 3;
  const int part = threadIdx.x & 7;
  const long long row = g / a.row_groups;
  const int c0 = (int)(g - row * a.row_groups) * kPackGroup + part * 4;
  const int n = g < a.groups ? min(a.C - c0, 4) : 0;
  T x[4];
  load_run<T, 4>(a.x, row * a.C + c0, n, x);
  const int e = group_exponent<T, 4>(x);
  signed char q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) q[k] = (signed char)pack_code(static_cast<float>(x[k]), e, a.keep_sign);
  store_run<signed char, 4>(a.codes, row * a.C + c0, n, q);
  if (part == 0 && n > 0) a.exps[g] = (signed char)e;
}

template <typename T, bool LINE>
__global__ __launch_bounds__(256) void unpack8_kernel(UnpackArgs a) {
  if constexpr (LINE) unpack_line_block<T>(a, a.first + blockIdx.x);
  else unpack_block<T>(a, a.first + blockIdx.x);
}

}  // namespace

int pack8(const void* x, signed char* codes, signed char* exps, long long rows, int C, int keep_sign, int dtype, void* stream) {
  const int rg = (int)pack_groups(C);
  PackArgs a = {0, x, codes, exps, rows * rg, C, rg, keep_sign};
  const bool line = on_a_line(C, x, codes);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return in_launches(line ? ceil_div_ll(a.groups * kPackGroup, kLine) : ceil_div_ll(a.groups, 32), [&](long long first, unsigned blocks) -> int {
      a.first = first;
      hipLaunchKernelGGL((line ? &pack8_line_kernel<T> : &pack8_kernel<T>), dim3(blocks), dim3(256), 0, as_stream(stream), a);
      WC_CHECK_LAUNCH("pack8_kernel");
      return WC_OK;
    });
  });
}

int unpack8(const signed char* codes, const signed char* exps, void* x, long long rows, int C, int dtype, void* stream) {
  const int rg = (int)pack_groups(C);
  UnpackArgs a = {0, codes, exps, x, rows * rg, C, C, rg};
  const bool line = on_a_line(C, x, codes);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return in_launches(unpack_blocks(a, line), [&](long long first, unsigned blocks) -> int {
      a.first = first;
      hipLaunchKernelGGL((line ? &unpack8_kernel<T, true> : &unpack8_kernel<T, false>), dim3(blocks), dim3(256), 0, as_stream(stream), a);
      WC_CHECK_LAUNCH("unpack8_kernel");
      return WC_OK;
    });
  });
}

}  // namespace wc
