// Activations in 8 bits for the backward pass: the groups of 32 neighbouring channels of a row share a step 2^e, e = floor(log2(largest
// magnitude)) - 6 but at least -126, and a value v is the whole number q nearest to v 2^-e (ties to even), at most 127 either way.
//
// The steps are powers of two, so v 2^-e is exact, q does not hang on how a division rounds, and q 2^e is exact in every type a group came
// from: it has seven bits, lies between the type's smallest number and its largest (127 2^(e) is below 2^(e + 7), where the group's largest
// value has its exponent), which steps rounded up to hold 128 2^e would exceed.  A value is off by at most half a step, 2^-7 of the group's
// largest, but for those above 127.5 steps, which are off by less than one, 2^-7 of themselves.  Against a floating type of 8 bits with three
// bits of mantissa (off by 2^-4 of the value) the large values of a group, which are most of the sums they enter, are eight times as exact.
// A group with an infinity or a NaN has the exponent 127 and reads as NaN throughout, so that such values still show in the gradients.
// keep_sign: values other than zero keep a code other than zero, one step - for what is read by its sign alone (the gate of a ReLU).
//
// Bound by memory.  A thread takes four neighbouring elements, eight threads a group.
#include "linear.h"

#include <algorithm>

namespace wc {

namespace {

struct PackArgs {
  const void* x; void* out;
  signed char* codes; signed char* exps;
  long long groups;          // of all rows
  int C, row_groups;
  int keep_sign;
};

__device__ __forceinline__ int pack_exponent(float top) {
  const int bits = (int)(__float_as_uint(top) >> 23);          // top >= 0
  return bits == 255 ? kPackNoNumber : max(bits - 127 - 6, kPackLeast);
}
// 2^-e is a normal number for every e there is but NoNumber, whose codes are not read
__device__ __forceinline__ int pack_code(float v, int e, bool keep_sign) {
  if (e == kPackNoNumber) return 0;
  const float q = fminf(fmaxf(rintf(v * __uint_as_float((unsigned)(127 - e) << 23)), -127.f), 127.f);
  return keep_sign && q == 0.f && v != 0.f ? (v > 0.f ? 1 : -1) : (int)q;
}

template <typename T>
__global__ __launch_bounds__(256) void pack8_kernel(PackArgs a) {
  const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) >> 3;
  const int part = threadIdx.x & 7;
  const long long row = g / a.row_groups;
  const int c0 = (int)(g - row * a.row_groups) * kPackGroup + part * 4;
  const int n = g < a.groups ? min(a.C - c0, 4) : 0;
  const T* x = static_cast<const T*>(a.x) + row * a.C + c0;
  float v[4], top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = e < n ? static_cast<float>(x[e]) : 0.f;
    // (bits: a maximum of floats would drop a NaN)
    top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(v[e]) & 0x7fffffffu));
  }
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) top = __uint_as_float(max(__float_as_uint(top), (unsigned)__shfl_xor((int)__float_as_uint(top), d)));
  const int e = pack_exponent(top);
  if (n <= 0) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) a.codes[row * a.C + c0 + i] = (signed char)pack_code(v[i], e, a.keep_sign);
  if (part == 0) a.exps[g] = (signed char)e;
}

template <typename T>
__global__ __launch_bounds__(256) void unpack8_kernel(PackArgs a) {
  const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) >> 3;
  if (g >= a.groups) return;
  const long long row = g / a.row_groups;
  const int c0 = (int)(g - row * a.row_groups) * kPackGroup + (threadIdx.x & 7) * 4;
  const float step = pack_step(a.exps[g]);
  const long long i = row * a.C + c0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c0 + e < a.C) static_cast<T*>(a.out)[i + e] = static_cast<T>((float)a.codes[i + e] * step);
}

}  // namespace

int pack8(const void* x, signed char* codes, signed char* exps, long long rows, int C, bool keep_sign, int dtype, void* stream) {
  const int rg = (int)pack_groups(C);
  const PackArgs a = {x, nullptr, codes, exps, rows * rg, C, rg, keep_sign};
  return dispatch_dtype(dtype, [&](auto t) -> int {
    hipLaunchKernelGGL(pack8_kernel<decltype(t)>, dim3((unsigned)ceil_div_ll(a.groups, 32)), dim3(256), 0, as_stream(stream), a);
    WC_CHECK_LAUNCH("pack8_kernel");
    return WC_OK;
  });
}

int unpack8(const signed char* codes, const signed char* exps, void* x, long long rows, int C, int dtype, void* stream) {
  const int rg = (int)pack_groups(C);
  const PackArgs a = {nullptr, x, const_cast<signed char*>(codes), const_cast<signed char*>(exps), rows * rg, C, rg, 0};
  return dispatch_dtype(dtype, [&](auto t) -> int {
    hipLaunchKernelGGL(unpack8_kernel<decltype(t)>, dim3((unsigned)ceil_div_ll(a.groups, 32)), dim3(256), 0, as_stream(stream), a);
    WC_CHECK_LAUNCH("unpack8_kernel");
    return WC_OK;
  });
}

}  // namespace wc
