// dx = dz w over a weight in 4 bits (packed4.h): a pass over the codes, which bounds it for few rows, where widening them first writes and reads four times their bytes.
//
// A wavefront takes 32 rows of w by a stage of 128 channels: a lane eight rows by the eight channels of a word.  Its 64 values, widened to the type of dz, turn
// about in the registers into eight operands of 16 x 16 x 32 instructions, each a channel's eight rows, for eight neighbouring elements of a row of dz; fp32 dz is
// taken as the three bf16 numbers that it is the sum of.  The wavefronts of a workgroup share the rows of w, and their sums meet in LDS; where the channels
// give too few workgroups the rows are shared among several, whose parts are joined in a fixed order.  A pass takes 16 MB rows of dz; more are passes of the same launch, side by side.
// us, the weight widened first | this: fp16 1 x 4096 <- 4096 33 | 8.2, 8 x 25088 <- 4096 108 | 16 (3.3 TB/s of codes), 7 x 15435 <- 5920 266 | 19, 32 x 8192 <- 8192
// 67 | 18.5, 512 133 | 97; fp32 16 x 8192 <- 8192 173 | 18, 4096 4219 | 1674.
#include "linear4_rows.h"

#include <algorithm>

namespace wc {

namespace {

constexpr int kWaves = 8, kStep = 32;      // rows of w a wavefront takes at a time

struct GradientArgs {
  const void* dz;
  long long M;
  int K, C;
  Operand4 w;
  long long stages;
  void* dx; float* parts;                  // parts (S, M, C); null: one
  int steps, steps_part, n_blocks, per_xcd;
};

// What a lane has of a step: a word of eight rows each, their scales, and the same eight elements of rows of dz
template <typename T, int MB> struct Step { unsigned codes[8]; i32x4 scales[2]; T dz[MB][8]; };

template <typename T, int MB>
__global__ __launch_bounds__(64 * kWaves) void linear4_gradient_kernel(GradientArgs g) {
  using W = typename Widened<T>::type;
  __shared__ __attribute__((aligned(16))) float sums[kWaves][16][kStage4];
  const int blk = xcd_remap(blockIdx.x, g.per_xcd);
  if (blk >= g.n_blocks) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, kg = lane >> 4;
  const long long s = blk / g.stages, stage = blk % g.stages;
  const int begin = (int)s * g.steps_part, end = min(g.steps, begin + g.steps_part), whole = min(end, g.K / kStep);
  const unsigned char* const codes = g.w.codes + stage * (kStage4 / 2) + r * 4;
  const unsigned char* const scales = g.w.scales + stage * (kRows4 * 4) + kg * 32;
  const long long m0 = (long long)blockIdx.y * (16 * MB);
  long long from[MB];                      // (rows behind the last give results that go nowhere)
#pragma unroll
  for (int i = 0; i < MB; ++i) from[i] = min(m0 + i * 16 + r, g.M - 1) * g.K;
  f32x4 acc[MB][8];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto load = [&](int k, Step<T, MB>& t, bool all) {
    const int row = k * kStep + kg * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      t.codes[i] = *reinterpret_cast<const unsigned*>(codes + (all ? row + i : min(row + i, g.K - 1)) * g.stages * (kStage4 / 2));
    const i32x4* const e = reinterpret_cast<const i32x4*>(scales + k * g.stages * (kRows4 * 4));
    t.scales[0] = e[0];
    t.scales[1] = e[1];
#pragma unroll
    for (int i = 0; i < MB; ++i) load_run<T, 8>(g.dz, from[i] + row, all ? 8 : min(g.K - row, 8), t.dz[i]);
  };
  auto multiply_in = [&](const Step<T, MB>& t) {
    W v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) values4<W>(t.codes[i], scale4((unsigned)t.scales[i / 4][i % 4] >> (r / 4 * 8) & 255u), v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      Pack<W, 8> p;
#pragma unroll
      for (int i = 0; i < 8; ++i) p.v[i] = v[i][j];
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i][j] = multiply_run<T>(t.dz[i], p, acc[i][j]);
    }
  };
  // Steps wave, wave + 8, ... of the part; the next is on its way while one is multiplied (behind the last it is the last again: no branch stands before a load)
  if (begin + wave < whole) {
    Step<T, MB> now, next;
    load(begin + wave, now, true);
#pragma unroll 1
    for (int k = begin + wave; k < whole; k += kWaves) {
      load(k + kWaves < whole ? k + kWaves : k, next, true);
      multiply_in(now);
      now = next;
    }
  }
  if (end > whole && whole >= begin && (whole - begin) % kWaves == wave) {      // the rows that are no whole step; those behind the last meet zeros of dz
    Step<T, MB> last;
    load(whole, last, false);
    multiply_in(last);
  }

  // register e of a lane, operand j: channel 8 (4 kg + e) + j, row r of dz.  Chunks of four channels are exchanged by the row, so that rows are in different banks
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    if (m0 + i * 16 >= g.M) break;
    if (i) __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f32x4*>(&sums[wave][r][((4 * kg + e) * 2 + h ^ r * 2) * 4]) = f32x4{acc[i][4 * h][e], acc[i][4 * h + 1][e], acc[i][4 * h + 2][e], acc[i][4 * h + 3][e]};
    __syncthreads();
    const int row = threadIdx.x / 32, chunk = threadIdx.x % 32;
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += *reinterpret_cast<const f32x4*>(&sums[w][row][(chunk ^ row * 2) * 4]);
    const long long m = m0 + i * 16 + row;
    const int c = (int)stage * kStage4 + chunk * 4, have = m < g.M ? max(min(g.C - c, 4), 0) : 0;
    if (g.parts) {
      const float o[4] = {t[0], t[1], t[2], t[3]};
      store_run<float, 4>(g.parts, (s * g.M + m) * g.C + c, have, o);
    } else {
      const T o[4] = {static_cast<T>(t[0]), static_cast<T>(t[1]), static_cast<T>(t[2]), static_cast<T>(t[3])};
      store_run<T, 4>(g.dx, m * g.C + c, have, o);
    }
  }
}

}  // namespace

// Rows of dz that a workgroup takes: fp32 ones, of three parts, leave no registers for more than 32
static int rows_of_pass(long long M, int dtype) { return M <= 16 ? 16 : M <= 32 || dtype == WC_F32 ? 32 : 64; }

// Parts: two workgroups to a compute unit where the rows of w have a step for every wavefront; one where there is one for half of the units anyway; of more than 2 MB
// no more bytes than the codes (us, fp16 64 x 4096 <- 4096 in 8 and 4 parts 24 | 17, 384 x 2048 <- 1000 in 3 and one 21 | 11)
int linear4_gradient_parts(long long M, long long K, long long C, int dtype) {
  const long long tiles = stages4(C) * ceil_div_ll(M, rows_of_pass(M, dtype)), steps = ceil_div_ll(K, kStep);
  if (tiles >= kCus / 2) return 1;
  return (int)std::max(1ll, std::min({ceil_div_ll(2 * kCus, tiles), steps / kWaves, std::max(K / (16 * M), (1ll << 19) / (M * C))}));
}

int linear4_gradient(const void* dz, const Operand4& w, void* dx, float* parts, long long M, int K, int C, int dtype, void* stream) {
  GradientArgs g = {dz, M, K, C, w, stages4(C), dx, nullptr, ceil_div(K, kStep), 0, 0, 0};
  const int S = linear4_gradient_parts(M, K, C, dtype), rows = rows_of_pass(M, dtype);
  g.steps_part = ceil_div(g.steps, S);
  g.parts = S > 1 ? parts : nullptr;
  const long long blocks = g.stages * S;
  g.n_blocks = (int)blocks;                // (stages are at most 2^15)
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto fn = rows == 16 ? &linear4_gradient_kernel<T, 1> : &linear4_gradient_kernel<T, 2>;
    if constexpr (sizeof(T) == 2) {
      if (rows == 64) fn = &linear4_gradient_kernel<T, 4>;
    }
    hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds), (unsigned)ceil_div_ll(M, rows)), dim3(64 * kWaves), 0, as_stream(stream), g);
    WC_CHECK_LAUNCH("linear4_gradient_kernel");
    if (S == 1) return WC_OK;
    LinearJoin join = {{}, parts, S, M, C};
    join.e.y = dx;
    return linear_join(&join, 1, nullptr, nullptr, dtype, stream);
  });
}

}  // namespace wc
