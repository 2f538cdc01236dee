// Linear layers of few rows over a weight in 4 bits (packed4.h): a pass over the weight, half a byte and a scale's 32nd a value, which bounds it.
//
// A workgroup of 16 wavefronts takes NR rows of w and as many of x (4, 8 or 16: as many workgroups as there are compute units, where it can be), whose reduction
// the wavefronts share, a stage of 128 channels at a time.  A lane holds a group of 32 channels of its row: 16 bytes of codes and one scale.
// x as it is: the codes become eight values of the type of x at a time, exact, straight into the operands of 16 x 16 x 32 instructions, each
// lane multiplying its own group (the order of the channels within a sum is free); fp32 x is taken as the three bf16 numbers that it is
// the sum of.  x in 4 bits: the codes are the operands of one 16 x 16 x 128 instruction with its scales.  Of its 16 rows an instruction
// spends 16 / NR places of the reduction on the same NR rows, of x as of w; of its results those of two equal places count.  The wavefronts' sums meet
// in LDS, so there are no parts and no second launch.
// us, fp16 x | x in 4 bits: 1 x 4096 -> 4096 4.9 | 4.6, 1 x 25088 -> 4096 19.7 (2.8 TB/s) | 16.4 (3.3), 8 x 25088 -> 4096 24 | 17: every workgroup reads all of x, from the L2.
#include "linear4_rows.h"

namespace wc {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 16;

struct FewArgs {
  LinearProduct p;
  Operand4 x, w;
  long long stages;
  int C;
};

__device__ __forceinline__ i32x8 codes_operand(i32x4 v) { return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// What a lane has of a stage: a group of 32 codes and its scale's exponent, and the same channels of x
struct Group { i32x4 codes; unsigned scale; };
template <typename T> struct Values { T v[4][8]; };

template <typename T, bool X4, int NR>
__global__ __launch_bounds__(64 * kWaves) void linear4_few_kernel(FewArgs g) {
  constexpr int PLACES = 16 / NR, DEPTH = X4 ? 8 : sizeof(T) == 2 ? 4 : 2;
  using W = typename Widened<T>::type;
  using X = typename std::conditional<X4, Group, Values<T>>::type;
  __shared__ float sums[kWaves * PLACES][NR][NR + 1];
  const LinearProduct& p = g.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane % NR, place = (lane & 15) / NR, c = lane >> 4;
  const long long n0 = (long long)blockIdx.x * NR, n = min(n0 + r, p.N - 1), m0 = (long long)blockIdx.y * NR, m = min(m0 + r, p.M - 1);      // (results of rows behind the last go nowhere)
  const unsigned char* const codes = g.w.codes + n * g.stages * (kStage4 / 2) + c * 16;
  const unsigned char* const scales = g.w.scales + scale_at4(n, c, g.stages);
  const unsigned char* const x_codes = X4 ? g.x.codes + m * g.stages * (kStage4 / 2) + c * 16 : nullptr;
  const unsigned char* const x_scales = X4 ? g.x.scales + scale_at4(m, c, g.stages) : nullptr;
  const T* const x_row = X4 ? nullptr : static_cast<const T*>(p.a) + m * p.lda;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};

  // Rounds: two stages of a wavefront, both halves of a line of the L2, then those 32 stages on
  auto stage_of = [&](int k) { return (((long long)(k >> 1) * kWaves + wave) * PLACES + place) * 2 + (k & 1); };
  auto rounds_of = [&](long long pairs) { return pairs > wave ? (int)((pairs - wave + kWaves - 1) / kWaves) * 2 : 0; };
  // all rounds, and those whose every stage is whole
  const int rounds = rounds_of((g.stages + 2 * PLACES - 1) / (2 * PLACES)), whole = rounds_of((X4 ? g.stages : g.C / kStage4) / (2 * PLACES));
  auto group = [&](const unsigned char* codes, const unsigned char* scales, long long at) {
    return Group{*reinterpret_cast<const i32x4*>(codes + at * (kStage4 / 2)), scales[at * (kRows4 * 4)]};
  };
  auto load = [&](int k, Group& w, X& x) {
    const long long at = stage_of(k);
    w = group(codes, scales, at);
    if constexpr (X4) x = group(x_codes, x_scales, at);
    else {
#pragma unroll
      for (int t = 0; t < 4; ++t) load_run<T, 8>(x_row, at * kStage4 + c * 32 + t * 8, 8, x.v[t]);
    }
  };
  auto multiply_in = [&](const Group& w, const X& x) {
    if constexpr (X4) {
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes_operand(w.codes), codes_operand(x.codes), acc, 4, 4, 0, (int)w.scale, 0, (int)x.scale);
    } else {
      const float s = scale4(w.scale);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        Pack<W, 8> v;
        values4<W>((unsigned)w.codes[t], s, v.v);
        acc = multiply_run<T>(x.v[t], v, acc);
      }
    }
  };
  // DEPTH rounds of both operands are on their way.  Loads come back in order, so x, from the L2, comes as far ahead as w; and no load stands
  // behind a branch in the loop, after which all that are on their way would be waited for.
  Group w[DEPTH];
  X x[DEPTH];
  int k = 0;
  if (whole >= 2 * DEPTH) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) load(u, w[u], x[u]);
#pragma unroll 1
    for (; k + 2 * DEPTH <= whole; k += DEPTH) {
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        multiply_in(w[u], x[u]);
        load(k + DEPTH + u, w[u], x[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
      multiply_in(w[u], x[u]);
      if (k + DEPTH + u < whole) load(k + DEPTH + u, w[u], x[u]);
    }
    k += DEPTH;
  } else {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (u < whole) load(u, w[u], x[u]);
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (u < whole) {
        multiply_in(w[u], x[u]);
        if (DEPTH + u < whole) load(DEPTH + u, w[u], x[u]);
      }
    k = DEPTH;
  }
#pragma unroll
  for (int u = 0; u < DEPTH; ++u)
    if (k + u < whole) multiply_in(w[u], x[u]);
  // the rest: stages that end behind the last channel or, of the last round's places, are not there, and count as zeros
#pragma unroll 1
  for (k = whole; k < rounds; ++k) {
    const long long at = stage_of(k);
    Group wk = {i32x4{0, 0, 0, 0}, 0u};
    X xk = {};
    if (at < g.stages) {
      wk = group(codes, scales, at);
      if constexpr (X4) xk = group(x_codes, x_scales, at);
      else {
        const int c0 = (int)at * kStage4 + c * 32;
#pragma unroll
        for (int t = 0; t < 4; ++t) load_run<T, 8>(x_row, c0 + t * 8, max(min(g.C - c0 - t * 8, 8), 0), xk.v[t]);
      }
    }
    multiply_in(wk, xk);
  }
  // register e of a lane: row 4 c + e of w's sixteen, row lane % 16 of x's
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if ((4 * c + e) / NR == place) sums[wave * PLACES + place][r][(4 * c + e) % NR] = acc[e];
  __syncthreads();
  const int mr = threadIdx.x / NR, nr = threadIdx.x % NR;
  if (mr >= NR || m0 + mr >= p.M || n0 + nr >= p.N) return;
  float v = 0.f;
#pragma unroll 16
  for (int s = 0; s < kWaves * PLACES; ++s) v += sums[s][mr][nr];
  finish_one<T>(p.e, m0 + mr, n0 + nr, p.N, v);
}

}  // namespace

int product4_few(const LinearProduct& p, const Operand4* x, const Operand4& w, int dtype, void* stream) {
  const FewArgs g = {p, x ? *x : Operand4{nullptr, nullptr}, w, stages4(p.R), (int)p.R};
  int nr = p.M <= 4 ? 4 : p.M <= 8 ? 8 : 16;
  while (nr < 16 && ceil_div_ll(p.N, nr) > kCus) nr *= 2;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto pick = [&](auto x4) {
      constexpr bool X4 = decltype(x4)::value;
      return nr == 4 ? &linear4_few_kernel<T, X4, 4> : nr == 8 ? &linear4_few_kernel<T, X4, 8> : &linear4_few_kernel<T, X4, 16>;
    };
    auto fn = x ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(fn, dim3((unsigned)ceil_div_ll(p.N, nr), (unsigned)ceil_div_ll(p.M, nr)), dim3(64 * kWaves), 0, as_stream(stream), g);
    WC_CHECK_LAUNCH("linear4_few_kernel");
    return WC_OK;
  });
}

}  // namespace wc
