// Linear layers of few rows over a weight in 4 bits (packed4.h): a pass over the weight, half a byte and a scale's 32nd a value, which bounds it.
//
// A workgroup of 16 wavefronts takes NR rows of w (4, 8 or 16: as many workgroups as there are compute units, where it can be), whose reduction
// the wavefronts share, a stage of 128 channels at a time.  A lane holds a group of 32 channels of its row: 16 bytes of codes and one scale.
// x as it is: the codes become eight values of the type of x at a time, exact, straight into the operands of 16 x 16 x 32 instructions, each
// lane multiplying its own group (the order of the channels within a sum is free); fp32 x is taken as the three bf16 numbers that it is
// the sum of.  x in 4 bits: the codes are the operands of one 16 x 16 x 128 instruction with its scales.  Of its 16 rows an instruction
// spends 16 / NR places of the reduction on the same NR rows, of x as of w; of its results those of two equal places count.  Up to 64
// rows of x are up to four operands to one of w.  The wavefronts' sums meet in LDS, so there are no parts and no second launch.
#include "packed4.h"

namespace wc {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 16;

struct FewArgs {
  LinearProduct p;
  Operand4 x, w;
  long long stages;
  int C;
};

__device__ __forceinline__ f32x4 multiply(const Pack<half_t, 8>& a, const Pack<half_t, 8>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(const Pack<bf16_t, 8>& a, const Pack<bf16_t, 8>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x8 codes_operand(i32x4 v) { return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// what the weight's codes become
template <typename T> struct Widened { using type = T; };
template <> struct Widened<float> { using type = bf16_t; };

// x: eight values of T, times eight of the weight
template <typename T>
__device__ __forceinline__ f32x4 multiply_run(const T (&x)[8], const Pack<typename Widened<T>::type, 8>& w, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
    Pack<bf16_t, 8> part;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned bits = __float_as_uint(x[e]);
      const float high = __uint_as_float(bits & 0xffff0000u);
      part.v[e] = __builtin_bit_cast(bf16_t, (unsigned short)(bits >> 16));
      // (of an infinity nothing is left; a NaN whose upper half says infinity stays one)
      rest[e] = (bits & 0x7fffffffu) == 0x7f800000u ? 0.f : x[e] - high;
    }
    c = multiply(w, part, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      part.v[e] = static_cast<bf16_t>(rest[e]);
      rest[e] -= static_cast<float>(part.v[e]);
    }
    c = multiply(w, part, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) part.v[e] = static_cast<bf16_t>(rest[e]);
    return multiply(w, part, c);
  } else {
    Pack<T, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] = x[e];
    return multiply(w, v, c);
  }
}

template <typename T, bool X4, int NR, int MB>
__global__ __launch_bounds__(64 * kWaves) void linear4_few_kernel(FewArgs g) {
  constexpr int PLACES = 16 / NR, AT_ONCE = X4 ? 4 : MB == 1 && sizeof(T) == 2 ? 2 : 1;
  static_assert(MB == 1 || NR == 16, "more than 16 rows of x leave one place");
  using W = typename Widened<T>::type;
  __shared__ float sums[kWaves * PLACES][NR][NR + 1];
  const LinearProduct& p = g.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane % NR, place = (lane & 15) / NR, c = lane >> 4;
  const long long n0 = (long long)blockIdx.x * NR, n = min(n0 + r, p.N - 1);
  const unsigned char* const codes = g.w.codes + n * g.stages * (kStage4 / 2) + c * 16;
  const unsigned char* const scales = g.w.scales + scale_at4(n, c, g.stages);
  f32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int rounds = (int)((g.stages + PLACES - 1) / PLACES);
  for (int k0 = wave; k0 < rounds; k0 += AT_ONCE * kWaves) {
    i32x4 wv[AT_ONCE];
    unsigned we[AT_ONCE];
    long long at[AT_ONCE];
    bool in[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const long long stage = (long long)(k0 + u * kWaves) * PLACES + place;
      in[u] = stage < g.stages;
      at[u] = min(stage, g.stages - 1);
      wv[u] = *reinterpret_cast<const i32x4*>(codes + at[u] * (kStage4 / 2));
      we[u] = scales[at[u] * (kRows4 * 4)];
    }
    if constexpr (X4) {
      i32x4 xv[AT_ONCE][MB];
      unsigned xe[AT_ONCE][MB];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          const long long m = min((long long)(b * 16 + r), p.M - 1);
          xv[u][b] = *reinterpret_cast<const i32x4*>(g.x.codes + (m * g.stages + at[u]) * (kStage4 / 2) + c * 16);
          xe[u][b] = g.x.scales[scale_at4(m, at[u] * 4 + c, g.stages)];
        }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        if (!in[u]) { wv[u] = i32x4{0, 0, 0, 0}; we[u] = 0; }
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          if (!in[u]) xe[u][b] = 0;          // (no number times a zero is no number)
          acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes_operand(wv[u]), codes_operand(xv[u][b]), acc[b], 4, 4, 0, (int)we[u], 0, (int)xe[u][b]);
        }
      }
    } else {
      T x[AT_ONCE][MB][4][8];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const long long m = b * 16 + r;
            const int k = (int)at[u] * kStage4 + c * 32 + t * 8;
            load_run<T, 8>(p.a, m * p.lda + k, in[u] && m < p.M ? max(min(g.C - k, 8), 0) : 0, x[u][b][t]);
          }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const float s = scale4(in[u] ? we[u] : 0);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          W v[8];
          values4<W>(in[u] ? (unsigned)wv[u][t] : 0u, s, v);
          Pack<W, 8> w;
#pragma unroll
          for (int e = 0; e < 8; ++e) w.v[e] = v[e];
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[b] = multiply_run<T>(x[u][b][t], w, acc[b]);
        }
      }
    }
  }
  // register e of a lane: row 4 c + e of w's sixteen, row lane % 16 of x's
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    if (b) __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((4 * c + e) / NR == place) sums[wave * PLACES + place][r][(4 * c + e) % NR] = acc[b][e];
    __syncthreads();
    const int mr = threadIdx.x / NR, nr = threadIdx.x % NR;
    const long long m = b * 16 + mr;
    if (mr >= NR || m >= p.M || n0 + nr >= p.N) continue;
    float v = 0.f;
#pragma unroll 16
    for (int s = 0; s < kWaves * PLACES; ++s) v += sums[s][mr][nr];
    finish_one<T>(p.e, m, n0 + nr, p.N, v);
  }
}

}  // namespace

int product4_few(const LinearProduct& p, const Operand4* x, const Operand4& w, int dtype, void* stream) {
  const FewArgs g = {p, x ? *x : Operand4{nullptr, nullptr}, w, stages4(p.R), (int)p.R};
  const int mb = (int)ceil_div_ll(p.M, 16);
  int nr = p.M <= 4 ? 4 : p.M <= 8 ? 8 : 16;
  while (nr < 16 && ceil_div_ll(p.N, nr) > 2 * kCus) nr *= 2;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto pick = [&](auto x4) {
      constexpr bool X4 = decltype(x4)::value;
      return mb == 1 ? (nr == 4 ? &linear4_few_kernel<T, X4, 4, 1> : nr == 8 ? &linear4_few_kernel<T, X4, 8, 1> : &linear4_few_kernel<T, X4, 16, 1>)
           : mb == 2 ? &linear4_few_kernel<T, X4, 16, 2> : &linear4_few_kernel<T, X4, 16, 4>;
    };
    auto fn = x ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(fn, dim3((unsigned)ceil_div_ll(p.N, nr)), dim3(64 * kWaves), 0, as_stream(stream), g);
    WC_CHECK_LAUNCH("linear4_few_kernel");
    return WC_OK;
  });
}

}  // namespace wc
