// What the products that are fed by LDS-DMA share (linear_dma.hip, linear4_dma.hip): an operand's way to LDS and from there to the registers of the
// matrix instructions, and the epilogue of a wavefront's results.
#pragma once
#include "linear_rows.h"
#include "lds_dma.h"
#include "wc_transform.h"

namespace wc {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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

// One operand of a tile of BT rows of the result, brought by NW wavefronts
template <typename T, int BT, int NW, bool OUTER> struct DmaOperand {
  static constexpr int BYTES = BT * 64, LOADS = BT / (16 * NW);           // a stage, 1 KB loads per wavefront
  static constexpr int ES = sizeof(T), EPC = kChunk<T>, CHUNKS = BT / EPC, RPI = 64 / CHUNKS;      // outer: chunks of a row, rows of a load
  static_assert(RPI >= 1, "a load holds whole rows");
  const unsigned char* base;       // of the next stage to be queued
  long long left;                  // bytes from there to the operand's end, outer: to the part's
  long long advance;               // a stage
  unsigned voff[LOADS];
  int chunk;                       // inner: the lane's chunk of a stage's row

  // outer: the exchange of a row's chunks
  static __device__ __forceinline__ int exchange(int row) { return ES == 4 ? (row >> 2 & 1) * 8 : BT == 64 ? (row >> 1 & 1) * 4 : (row & 3) * 4; }
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
        const int row = (wave + NW * i) * 16 + lane / 4;
        chunk = lane % 4 ^ swizzle(row);
        voff[i] = row0 + row < rows ? (unsigned)(row * ld * ES + chunk * 16) : kOutside;
      }
    }
  }
  // of the next stage, or of the next two: descriptors, and what puts a lane's chunk outside them where the part ends before it
  DmaDesc d, d2;
  unsigned out, out2;
  template <bool PAIR> __device__ __forceinline__ void aim(long long have) {                   // `have` reduction elements are left of the part
    d = dma_descriptor(base, left);
    out = OUTER || chunk * EPC < have ? 0u : kOutside;
    if constexpr (PAIR) {
      d2 = dma_descriptor(base + advance, left - advance);
      out2 = OUTER || chunk * EPC + kDeep<T> < have ? 0u : kOutside;
    }
    base += (PAIR ? 2 : 1) * advance;
    left -= (PAIR ? 2 : 1) * advance;
  }
  // queues load i of them, into LDS at `lds` and `lds2`
  template <bool PAIR> __device__ __forceinline__ void queue(unsigned lds, unsigned lds2, int wave, int i) const {
    const unsigned to = (OUTER ? wave * LOADS + i : wave + NW * i) * 1024;
    dma16(d, voff[i] | out, lds + to);
    if constexpr (PAIR) dma16(d2, voff[i] | out2, lds2 + to);
  }

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

constexpr int kBand = 8;       // tiles along M that are neighbours

// What the lanes of a wavefront wrote to LDS is there for its other lanes, and what they read may be overwritten
__device__ __forceinline__ void exchange_done() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wavefront's WM x WN blocks through 32 rows of LDS of its own, a lane finishing eight neighbouring results of some rows, which start anywhere.
// ALL: the tile is whole, no lane asks whether its results are there - a branch at every access leaves none to overlap.  MORE: there may be a
// residual or z.
template <typename T, int ACT, bool ALL, bool MORE, int WM, int WN>
__device__ __forceinline__ void finish_blocks(const LinearEpilogue& e, const f32x16 (&acc)[WM][WN], float* stage, long long m0, long long M, int n0, long long N, int lane) {
  constexpr int PITCH = WN * 32 + 4, LPR = WN * 4, RPI = 64 / LPR;      // floats of a row, lanes to a row, rows of an access
  constexpr int RUNS = 32 / RPI, AT_ONCE = RUNS < 4 || !MORE ? RUNS : 4;
  const int l32 = lane & 31, lhi = lane >> 5, row0 = lane / LPR, n = n0 + lane % LPR * 8;
  const int have = ALL ? 8 : (int)max(min(8ll, N - n), 0ll);
  float bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = 0.f;
  if (e.bias) {
    T b[8];
    load_run<T, 8>(e.bias, n, have, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) bias[j] = static_cast<float>(b[j]);
  }
#pragma unroll
  for (int i = 0; i < WM; ++i) {
    const long long first = (m0 + i * 32 + row0) * N + n;
    const int rows = (int)min(32ll, M - m0 - i * 32);
    auto there = [&](int r) { return ALL ? 8 : row0 + r * RPI < rows ? have : 0; };
    auto at = [&](int r) { return first + (long long)(r * RPI) * N; };
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(stage + l32 * PITCH + j * 32 + 8 * q + 4 * lhi) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    exchange_done();
#pragma unroll
    for (int r0 = 0; r0 < RUNS; r0 += AT_ONCE) {
      T res[AT_ONCE][8];
      float v[AT_ONCE][8];
      if (MORE && e.res) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r) load_run<T, 8>(e.res, at(r0 + r), there(r0 + r), res[r]);
      } else {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) res[r][j] = static_cast<T>(0.f);
      }
#pragma unroll
      for (int r = 0; r < AT_ONCE; ++r) {
        const float* const from = stage + (row0 + (r0 + r) * RPI) * PITCH + lane % LPR * 8;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[r][j] = lo[j] + bias[j];
          v[r][j + 4] = hi[j] + bias[j + 4];
        }
      }
      if (MORE && !e.res_after) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[r][j] += static_cast<float>(res[r][j]);
      }
      auto store = [&](void* to) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r) {
          T o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = static_cast<T>(v[r][j]);
          store_run<T, 8>(to, at(r0 + r), there(r0 + r), o);
        }
      };
      if (MORE && e.z) store(e.z);
      if constexpr (ACT != WC_ACT_NONE) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[r][j] = activate(v[r][j], ACT);
      }
      if (MORE && e.res_after) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[r][j] += static_cast<float>(res[r][j]);
      }
      if (e.y_f32 && sizeof(T) == 2) {
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r) store_run<float, 8>(e.y, at(r0 + r), there(r0 + r), v[r]);
      } else {
        store(e.y);
      }
    }
    if (i + 1 < WM) exchange_done();
  }
}

// run(ic<act>), the activation a constant of its instructions
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& run) {
  switch (act) {
    case WC_ACT_RELU: run(ic<WC_ACT_RELU>{}); break;
    case WC_ACT_GELU: run(ic<WC_ACT_GELU>{}); break;
    case WC_ACT_GELU_TANH: run(ic<WC_ACT_GELU_TANH>{}); break;
    case WC_ACT_SILU: run(ic<WC_ACT_SILU>{}); break;
    default: run(ic<WC_ACT_NONE>{});
  }
}

// A wavefront's blocks to a part's sums (M, N).  Register 4 q + e of a lane: row l32, column 8 q + 4 lhi + e of the block.  vec: rows are multiples of 16 bytes; of others
// sixteen bytes start at any float (us, the call of fp16 299 x 9352 -> 1745 over a weight in 4 bits, float by float 44, so 33; over one in 16 bits 46 | 36)
template <int WM, int WN>
__device__ __forceinline__ void store_parts(float* part, const f32x16 (&acc)[WM][WN], long long m0, long long M, long long n0, long long N, int vec, int lane) {
  const int l32 = lane & 31, lhi = lane >> 5;
#pragma unroll
  for (int i = 0; i < WM; ++i) {
    const long long m = m0 + i * 32 + l32;
    float* const row = part + m * N;
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long long n = n0 + j * 32 + 8 * q + 4 * lhi;
        const f32x4 o = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        if (m >= M) continue;
        if (vec) {
          if (n < N) *reinterpret_cast<f32x4*>(row + n) = o;
        } else if (n + 3 < N) {
          *reinterpret_cast<Run<float, 4>*>(row + n) = Run<float, 4>{o[0], o[1], o[2], o[3]};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) row[n + e] = o[e];
        }
      }
  }
}

}  // namespace wc
