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
#include "linear.h"
#include "lds_dma.h"
#include "wc_transform.h"

#include <algorithm>

namespace wc {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 product(s16x8 a, s16x8 b, f32x16 c, half_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 product(s16x8 a, s16x8 b, f32x16 c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// (the lanes of either half hold four neighbouring reduction elements, and an fp32 instruction takes one of each half)
__device__ __forceinline__ f32x16 product(s16x8 a, s16x8 b, f32x16 c, float) {
  const f32x4 p = __builtin_bit_cast(f32x4, a), q = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_32x32x2f32(p[k], q[k], c, 0, 0, 0);
  return c;
}

// reduction elements of a stage, and of a 16-byte chunk
template <typename T> constexpr int kDeep = 64 / sizeof(T);
template <typename T> constexpr int kChunk = 16 / sizeof(T);

// One operand of a tile of 64 W rows of the result
template <typename T, int W, bool OUTER> struct DmaOperand {
  static constexpr int BT = 64 * W, BYTES = BT * 64, LOADS = W;           // a stage, 1 KB loads per wavefront
  static constexpr int ES = sizeof(T), EPC = kChunk<T>, CHUNKS = BT / EPC, RPI = 64 / CHUNKS;      // outer: chunks of a row, rows of a load
  static_assert(RPI >= 1, "a load holds whole rows");
  const unsigned char* base;       // of the next stage to be queued
  long long left;                  // bytes from there to the operand's end, outer: to the part's
  long long advance;               // a stage
  unsigned voff[LOADS];
  int chunk;                       // inner: the lane's chunk of a stage's row

  // outer: the exchange of a row's chunks
  static __device__ __forceinline__ int exchange(int row) { return ES == 4 ? (row >> 2 & 1) * 8 : W == 1 ? (row >> 1 & 1) * 4 : (row & 3) * 4; }
  static __device__ __forceinline__ int swizzle(int r) { return (((r >> 1) ^ (r >> 3)) & 1) | ((r >> 2) & 1) << 1; }

  __device__ __forceinline__ void start(const void* p, long long ld, long long row0, long long rows, long long begin, long long end, int wave, int lane) {
    const long long first = OUTER ? begin * ld + row0 : row0 * ld + begin;
    base = static_cast<const unsigned char*>(p) + first * ES;
    left = ((OUTER ? end : rows) * ld - first) * ES;
    advance = OUTER ? kDeep<T> * ld * ES : 64;
    chunk = 0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if constexpr (OUTER) {
        const int row = (wave * LOADS + i) * RPI + lane / CHUNKS;
        const int c = lane % CHUNKS ^ exchange(row);
        voff[i] = row0 + c * EPC < rows ? (unsigned)(row * ld * ES + c * 16) : kOutside;
      } else {
        const int row = (wave + 4 * i) * 16 + lane / 4;
        chunk = lane % 4 ^ swizzle(row);
        voff[i] = row0 + row < rows ? (unsigned)(row * ld * ES + chunk * 16) : kOutside;
      }
    }
  }
  // queues the next stage; `have` reduction elements are left of the part
  __device__ __forceinline__ void queue(unsigned lds, int wave, int i, long long have) const {
    const DmaDesc d = dma_descriptor(base, left);
    const unsigned to = lds + (OUTER ? wave * LOADS + i : wave + 4 * i) * 1024;
    dma16(d, OUTER || chunk * EPC < have ? voff[i] : kOutside, to);
  }
  __device__ __forceinline__ void next() { base += advance; left -= advance; }

  // byte offset of a lane's part of the fragment of half `kk` of a stage, rows 32 b .. of the tile
  static __device__ __forceinline__ int offset(int b, int kk, int lane) {
    if constexpr (OUTER && ES == 4) {
      const int row = kk * 8 + 4 * (lane >> 5);                           // and the three after it, exchanged alike
      return row * (BT * 4) + ((b * 8 + (lane & 31) / 4) ^ exchange(row)) * 16 + (lane & 3) * 4;
    } else if constexpr (OUTER) {
      const int row = kk * 16 + 8 * (lane >> 5) + (lane >> 2 & 3), col = b * 64 + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
      return row * (BT * 2) + (col ^ exchange(row) * 16);
    } else {
      const int r = lane & 31;
      return (b * 32 + r) * 64 + ((kk * 2 + (lane >> 5)) ^ swizzle(r)) * 16;
    }
  }
  static __device__ __forceinline__ s16x8 read(const unsigned char* at) {
    if constexpr (OUTER && ES == 4) {
      f32x4 v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float*>(at + k * BT * 4);
      return __builtin_bit_cast(s16x8, v);
    } else if constexpr (OUTER) {
      typedef s16x4 __attribute__((address_space(3)))* LdsVec;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec)(at + 4 * BT * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *reinterpret_cast<const s16x8*>(at);
    }
  }
};

struct DmaArgs {
  LinearProduct p;
  float* parts;               // (S, M, N); null: one part, the epilogue here
  long long R_part;
  int tiles_m, tiles_n, n_blocks, per_xcd;
  int vec;                    // rows of the results are multiples of 16 bytes
};

// Eight elements at a multiple of 16 bytes, 16 bytes an access
template <typename T> using Sixteen = Pack<T, kChunk<T>>;
template <typename T> __device__ __forceinline__ void store8(T* to, const Pack<T, 8>& v) {
#pragma unroll
  for (int i = 0; i < 8 / kChunk<T>; ++i) reinterpret_cast<Sixteen<T>*>(to)[i] = reinterpret_cast<const Sixteen<T>*>(&v)[i];
}
template <typename T> __device__ __forceinline__ void load8(const T* from, Pack<T, 8>& v) {
#pragma unroll
  for (int i = 0; i < 8 / kChunk<T>; ++i) reinterpret_cast<Sixteen<T>*>(&v)[i] = reinterpret_cast<const Sixteen<T>*>(from)[i];
}

// Eight neighbouring results of a row, of which `have` are there: sums to z and y.  VEC: elements of an access.
template <typename T, int ACT, int VEC>
__device__ __forceinline__ void finish_run(const LinearEpilogue& e, long long i, int have, const float (&sum)[8], const float (&bias)[8], const Pack<T, 8>& res) {
  Pack<T, 8> z, y;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = sum[j] + bias[j];
    const float r = static_cast<float>(res.v[j]);
    if (!e.res_after) v[j] += r;
    z.v[j] = static_cast<T>(v[j]);
    v[j] = activate(v[j], ACT);
    if (e.res_after) v[j] += r;
    y.v[j] = static_cast<T>(v[j]);
  }
  if constexpr (VEC == 8) {
    if (e.z) store8(static_cast<T*>(e.z) + i, z);
    if (e.y_f32 && sizeof(T) == 2) {
      float* const to = static_cast<float*>(e.y) + i;
      *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      store8(static_cast<T*>(e.y) + i, y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= have) break;
      if (e.z) static_cast<T*>(e.z)[i + j] = z.v[j];
      if (e.y_f32) static_cast<float*>(e.y)[i + j] = v[j];
      else static_cast<T*>(e.y)[i + j] = y.v[j];
    }
  }
}

// A wavefront's WM x WN blocks through 32 rows of LDS of its own
template <typename T, int ACT, int VEC, int WM, int WN>
__device__ __forceinline__ void finish_blocks(const LinearEpilogue& e, const f32x16 (&acc)[WM][WN], float* stage, long long m0, long long M, int n0, long long N, int lane) {
  constexpr int PITCH = WN * 32 + 4, LPR = WN * 4, RPI = 64 / LPR;          // floats of a row, lanes to a row, rows of an access
  const int l32 = lane & 31, lhi = lane >> 5, row0 = lane / LPR, n = n0 + lane % LPR * 8;
  const int have = (int)min(8ll, N - n);
  float bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = e.bias && j < have ? static_cast<float>(static_cast<const T*>(e.bias)[n + j]) : 0.f;
#pragma unroll
  for (int i = 0; i < WM; ++i) {
    const long long first = (m0 + i * 32 + row0) * N + n;
    const int rows = (int)min(32ll, M - m0 - i * 32);
    Pack<T, 8> res[32 / RPI];
#pragma unroll
    for (int r = 0; r < 32 / RPI; ++r) {
#pragma unroll
      for (int j = 0; j < 8; ++j) res[r].v[j] = static_cast<T>(0.f);
      if (e.res && have > 0 && row0 + r * RPI < rows) {
        const T* const from = static_cast<const T*>(e.res) + first + (long long)(r * RPI) * N;
        if constexpr (VEC == 8) load8(from, res[r]);
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < have) res[r].v[j] = from[j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(stage + l32 * PITCH + j * 32 + 8 * q + 4 * lhi) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
#pragma unroll
    for (int r = 0; r < 32 / RPI; ++r) {
      float v[8];
      const float* const from = stage + (row0 + r * RPI) * PITCH + lane % LPR * 8;
      *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(from);
      *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(from + 4);
      if (have > 0 && row0 + r * RPI < rows) finish_run<T, ACT, VEC>(e, first + (long long)(r * RPI) * N, have, v, bias, res[r]);
    }
  }
}

// Template of a product: blocks of a wavefront, stages of the ring, whether the first half of a stage is read while the last one of the stage before
// is multiplied (a wavefront alone on its SIMD waits for every read that is not ahead)
template <int WM_, int WN_, int RING_, bool AHEAD_> struct Shape {
  static constexpr int WM = WM_, WN = WN_, RING = RING_;
  static constexpr bool AHEAD = AHEAD_;
  static constexpr size_t STAGE = 64 * 64 * (WM + WN), EPILOGUE = 4 * 32 * (WN * 32 + 4) * 4;
};

template <typename T, typename SH, bool AO, bool BO>
__device__ __forceinline__ void product_block(const DmaArgs& g, int hw_block, unsigned char* lds) {
  constexpr int WM = SH::WM, WN = SH::WN, kRing = SH::RING;
  constexpr bool AHEAD = SH::AHEAD;
  using A = DmaOperand<T, WM, AO>;
  using B = DmaOperand<T, WN, BO>;
  constexpr int STAGE = A::BYTES + B::BYTES, L = WM + WN;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int blk = xcd_remap(hw_block, g.per_xcd);
  if (blk >= g.n_blocks) return;
  // eight tiles along M, then along N: the workgroups of an XCD that run together share the rows of few tiles of either operand
  const int tiles = g.tiles_m * g.tiles_n, s = blk / tiles, t = blk % tiles;
  const int band = t / (8 * g.tiles_n), in_band = t % (8 * g.tiles_n), high = min(8, g.tiles_m - band * 8);
  const long long m0 = (long long)(band * 8 + in_band % high) * (64 * WM), n0 = (long long)(in_band / high) * (64 * WN);
  const LinearProduct& p = g.p;
  const long long begin = s * g.R_part, end = min(p.R, begin + g.R_part);
  const int nk = end > begin ? (int)((end - begin + kDeep<T> - 1) / kDeep<T>) : 0;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  A a;
  B b;
  a.start(p.a, p.lda, m0, p.M, begin, end, wave, lane);
  b.start(p.b, p.ldb, n0, p.N, begin, end, wave, lane);
  int queued = 0;
  auto queue = [&](int q) {                         // load q of the L of stage `queued`
    const unsigned to = lds0 + (queued % kRing) * STAGE;
    const long long have = end - begin - (long long)queued * kDeep<T>;
    if (q < WM) a.queue(to, wave, q, have);
    else b.queue(to + A::BYTES, wave, q - WM, have);
  };
  auto queue_next = [&] { a.next(); b.next(); ++queued; };

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

  if (nk > 0) {
#pragma unroll
    for (int k = 0; k < kRing - 1; ++k) {
      if (k >= nk) break;
#pragma unroll
      for (int q = 0; q < L; ++q) queue(q);
      queue_next();
    }
    if constexpr (AHEAD) {
      static_assert(kRing == 4, "three stages in flight");
      if (nk >= 3) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(2 * L) : "memory");
      else if (nk == 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int i = 0; i < WM; ++i) va[0][i] = A::read(lds + fa[0][i]);
#pragma unroll
      for (int j = 0; j < WN; ++j) vb[0][j] = B::read(lds + fb[0][j]);
    }
  }
#pragma unroll 1
  for (int ks = 0; ks < nk; ++ks) {
    const bool more = ks + kRing - 1 < nk;
    if constexpr (AHEAD) {
      // stage ks + 1 has landed, in flight may be that of ks + 2; nobody reads stage ks - 1 any more, which that of ks + 3 overwrites
      if (ks + 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const unsigned char* const st = lds + (kk ? min(ks + 1, nk - 1) % kRing : ks % kRing) * STAGE;      // of the half after this one
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
      if (more) queue_next();
    } else {
      // stage ks has landed, in flight may be the RING - 2 after it; nobody reads stage ks - 1 any more
      if (ks + kRing - 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((kRing - 2) * L) : "memory");
      else if (kRing > 3 && ks + 1 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(L) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const unsigned char* const st = lds + ks % kRing * STAGE;
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
    }
  }

  // register 4 q + e of a lane: row l32, column 8 q + 4 lhi + e of the block
  const int l32 = lane & 31, lhi = lane >> 5;
  const long long wm0 = m0 + wm * WM * 32, wn0 = n0 + wn * WN * 32;
  if (g.parts) {
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const long long m = wm0 + i * 32 + l32;
      float* const row = g.parts + (s * p.M + m) * p.N;
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const long long n = wn0 + j * 32 + 8 * q + 4 * lhi;
          const f32x4 o = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          if (m >= p.M) continue;
          if (g.vec) {
            if (n < p.N) *reinterpret_cast<f32x4*>(row + n) = o;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < p.N) row[n + e] = o[e];
          }
        }
    }
    return;
  }
  __syncthreads();                                          // the ring is done with
  float* const stage = reinterpret_cast<float*>(lds) + wave * 32 * (WN * 32 + 4);
  auto finish = [&](auto act) {
    if (g.vec) finish_blocks<T, act(), 8, WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
    else finish_blocks<T, act(), 1, WM, WN>(p.e, acc, stage, wm0, p.M, (int)wn0, p.N, lane);
  };
  if constexpr (BO) finish(ic<WC_ACT_NONE>{});              // a gradient has no epilogue
  else {
    switch (p.e.act) {
      case WC_ACT_RELU: finish(ic<WC_ACT_RELU>{}); break;
      case WC_ACT_GELU: finish(ic<WC_ACT_GELU>{}); break;
      case WC_ACT_GELU_TANH: finish(ic<WC_ACT_GELU_TANH>{}); break;
      case WC_ACT_SILU: finish(ic<WC_ACT_SILU>{}); break;
      default: finish(ic<WC_ACT_NONE>{});
    }
  }
}

template <typename SH> constexpr int kMinWaves = SH::WM * SH::WN > 8 ? 1 : 2;

template <typename T, typename SH, bool AO, bool BO>
__global__ __launch_bounds__(256, kMinWaves<SH>) void product_dma_kernel(DmaArgs g) {
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
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.e.y) | reinterpret_cast<uintptr_t>(p.e.z) | reinterpret_cast<uintptr_t>(p.e.res);
  g.vec = p.N % 8 == 0 && at % 16 == 0;
  return g;
}

// LDS of a product: the stages that its reduction has, and no less than the epilogue takes
template <typename T, typename SH>
size_t lds_of(const DmaArgs& g) {
  const long long stages = std::min<long long>(SH::RING, std::max(1ll, ceil_div_ll(std::min(g.R_part, g.p.R), kDeep<T>)));
  return std::max<size_t>((size_t)stages * SH::STAGE, SH::EPILOGUE);
}
template <typename SH> constexpr size_t kMostLds = SH::RING * SH::STAGE > SH::EPILOGUE ? SH::RING * SH::STAGE : SH::EPILOGUE;

template <typename T, typename SH>
int launch(const DmaArgs& g, void* stream) {
  const LinearProduct& p = g.p;
  auto fn = p.a_outer ? &product_dma_kernel<T, SH, true, true> : p.b_outer ? &product_dma_kernel<T, SH, false, true> : &product_dma_kernel<T, SH, false, false>;
  if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(fn), kMostLds<SH>)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(256), (lds_of<T, SH>(g)), as_stream(stream), g);
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

using Tile256 = Shape<4, 4, 4, true>;
using Tile256x128 = Shape<4, 2, 3, false>;
using Tile128 = Shape<2, 2, 4, false>;
using Tile64 = Shape<1, 1, 4, false>;

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
      if (plan.tile.n == 256) return launch<T, Tile256>(g, stream);
      if (plan.tile.m == 256) return launch<T, Tile256x128>(g, stream);
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
