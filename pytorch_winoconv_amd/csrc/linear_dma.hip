// The products of linear.h in 16-bit types on the matrix cores, both operands brought to LDS by LDS-DMA: rows that are multiples of 16 bytes.
//
// A workgroup's four wavefronts (2 x 2) take WM x WN blocks of 32 x 32 each.  A ring of four stages of 32 reduction elements, three in
// flight; fragments of a 16-deep half are read while the half before is multiplied, and the loads of the step three on are queued
// between.  An operand whose reduction axis is innermost lies in LDS in rows of 64 bytes, its 16-byte chunks exchanged by the row, and is read
// 16 bytes a lane; one whose reduction axis is outermost lies as it does in memory, 64-byte pieces exchanged by the row, and is read by
// ds_read_b64_tr_b16, which hands each lane four elements of a column: nothing is transposed in memory for either gradient.
// Both swizzles keep the lanes of a read in different banks.  What lies outside an operand - rows, columns, the end of the
// reduction - are offsets outside its descriptor, which bring zeros.
//
// Results go through LDS in fp32, 32 rows of a wavefront at a time, so that bias, residual, y and z are read and written 16 bytes a lane in
// whole row segments; few tiles: parts of the reduction, whose sums join_kernel (linear_product.hip) adds.
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

constexpr int kDeep = 32, kRing = 4;

// One operand of a tile of 64 W rows of the result
template <int W, bool OUTER> struct DmaOperand {
  static constexpr int BT = 64 * W, BYTES = BT * 64, LOADS = W;           // a stage, 1 KB loads per wavefront
  static constexpr int CHUNKS = BT / 8, RPI = 64 / CHUNKS;                // outer: chunks of a row, rows of a load
  const unsigned char* base;       // of the next stage to be queued
  long long left;                  // bytes from there to the operand's end, outer: to the part's
  long long advance;               // a stage
  unsigned voff[LOADS];
  int chunk;                       // inner: the lane's chunk of a stage's row

  static __device__ __forceinline__ int swizzle(int r) { return (((r >> 1) ^ (r >> 3)) & 1) | ((r >> 2) & 1) << 1; }

  __device__ __forceinline__ void start(const void* p, long long ld, long long row0, long long rows, long long begin, long long end, int wave, int lane) {
    const long long first = OUTER ? begin * ld + row0 : row0 * ld + begin;
    base = static_cast<const unsigned char*>(p) + first * 2;
    left = ((OUTER ? end : rows) * ld - first) * 2;
    advance = OUTER ? kDeep * ld * 2 : kDeep * 2;
    chunk = 0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if constexpr (OUTER) {
        const int row = (wave * LOADS + i) * RPI + lane / CHUNKS;
        const int c = lane % CHUNKS ^ (W == 1 ? (row >> 1 & 1) * 4 : (row & 3) * 4);
        voff[i] = row0 + c * 8 < rows ? (unsigned)(row * ld * 2 + c * 16) : kOutside;
      } else {
        const int row = (wave + 4 * i) * 16 + lane / 4;
        chunk = lane % 4 ^ swizzle(row);
        voff[i] = row0 + row < rows ? (unsigned)(row * ld * 2 + chunk * 16) : kOutside;
      }
    }
  }
  // queues the next stage; `have` reduction elements are left of the part
  __device__ __forceinline__ void queue(unsigned lds, int wave, int i, long long have) const {
    const DmaDesc d = dma_descriptor(base, left);
    const unsigned to = lds + (OUTER ? wave * LOADS + i : wave + 4 * i) * 1024;
    dma16(d, OUTER || chunk * 8 < have ? voff[i] : kOutside, to);
  }
  __device__ __forceinline__ void next() { base += advance; left -= advance; }

  // byte offset of a lane's part of the fragment of 16-deep half `kk`, rows 32 b .. of the tile
  static __device__ __forceinline__ int offset(int b, int kk, int lane) {
    if constexpr (OUTER) {
      const int row = kk * 16 + 8 * (lane >> 5) + (lane >> 2 & 3), col = b * 64 + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
      return row * (BT * 2) + (col ^ (W == 1 ? (row >> 1 & 1) * 64 : (row & 3) * 64));
    } else {
      const int r = lane & 31;
      return (b * 32 + r) * 64 + ((kk * 2 + (lane >> 5)) ^ swizzle(r)) * 16;
    }
  }
  static __device__ __forceinline__ s16x8 read(const unsigned char* at) {
    if constexpr (OUTER) {
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

// VEC neighbouring results of a row
template <typename T, int VEC>
__device__ __forceinline__ void finish_run(const LinearEpilogue& e, long long i, int n, int have, const float (&sum)[8]) {
#pragma unroll
  for (int j0 = 0; j0 < 8; j0 += VEC) {
    if (j0 >= have) break;
    Pack<T, VEC> r, z, y;
    float v[VEC];
    if (e.res) r = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(e.res) + i + j0);
    else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) r.v[j] = static_cast<T>(0.f);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[j] = sum[j0 + j];
      if (e.bias) v[j] += static_cast<float>(static_cast<const T*>(e.bias)[n + j0 + j]);
      if (!e.res_after) v[j] += static_cast<float>(r.v[j]);
      z.v[j] = static_cast<T>(v[j]);
    }
    if (e.z) *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(e.z) + i + j0) = z;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[j] = activate(v[j], e.act);
      if (e.res_after) v[j] += static_cast<float>(r.v[j]);
      y.v[j] = static_cast<T>(v[j]);
    }
    if (e.y_f32) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) static_cast<float*>(e.y)[i + j0 + j] = v[j];
    } else {
      *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(e.y) + i + j0) = y;
    }
  }
}

template <typename T, int WM, int WN, bool AO, bool BO>
__global__ __launch_bounds__(256, WM * WN >= 8 ? 1 : 2) void product_dma_kernel(DmaArgs g) {
  using A = DmaOperand<WM, AO>;
  using B = DmaOperand<WN, BO>;
  constexpr int STAGE = A::BYTES + B::BYTES, L = WM + WN;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int blk = xcd_remap(blockIdx.x, g.per_xcd);
  if (blk >= g.n_blocks) return;
  // eight tiles along M, then along N: the workgroups of an XCD that run together share the rows of few tiles of either operand
  const int tiles = g.tiles_m * g.tiles_n, s = blk / tiles, t = blk % tiles;
  const int band = t / (8 * g.tiles_n), in_band = t % (8 * g.tiles_n), high = min(8, g.tiles_m - band * 8);
  const long long m0 = (long long)(band * 8 + in_band % high) * (64 * WM), n0 = (long long)(in_band / high) * (64 * WN);
  const LinearProduct& p = g.p;
  const long long begin = s * g.R_part, end = min(p.R, begin + g.R_part);
  const int nk = end > begin ? (int)((end - begin + kDeep - 1) / kDeep) : 0;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  A a;
  B b;
  a.start(p.a, p.lda, m0, p.M, begin, end, wave, lane);
  b.start(p.b, p.ldb, n0, p.N, begin, end, wave, lane);
  int queued = 0;
  auto queue = [&](int q) {                         // load q of the L of stage `queued`
    const unsigned to = lds0 + (queued % kRing) * STAGE;
    const long long have = end - begin - (long long)queued * kDeep;
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
    if (nk >= 3) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(2 * L) : "memory");
    else if (nk == 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(L) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < WM; ++i) va[0][i] = A::read(lds + fa[0][i]);
#pragma unroll
    for (int j = 0; j < WN; ++j) vb[0][j] = B::read(lds + fb[0][j]);
  }
#pragma unroll 1
  for (int ks = 0; ks < nk; ++ks) {
    // stage ks + 1 has landed, in flight may be that of ks + 2; nobody reads stage ks - 1 any more, which that of ks + 3 overwrites
    if (ks + 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(L) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool more = ks + kRing - 1 < nk;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const unsigned char* const st = lds + (kk ? (ks + 1) % kRing : ks % kRing) * STAGE;      // of the half after this one
#pragma unroll
      for (int i = 0; i < WM; ++i) {
        va[kk ^ 1][i] = A::read(st + fa[kk ^ 1][i]);
        if (i < WN) vb[kk ^ 1][i] = B::read(st + fb[kk ^ 1][i]);
        if (i == WM - 1) {
#pragma unroll
          for (int j = WM; j < WN; ++j) vb[kk ^ 1][j] = B::read(st + fb[kk ^ 1][j]);
        }
#pragma unroll
        for (int j = 0; j < WN; ++j) acc[i][j] = product(vb[kk][j], va[kk][i], acc[i][j], T{});
        if constexpr (WM * WN >= 8) {
#pragma unroll
          for (int j = 0; j < WN; ++j) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (more) {
#pragma unroll
          for (int q = 0; q < L; ++q)
            if (q * 2 * WM / L == kk * WM + i) queue(q);
        }
        if constexpr (WM * WN >= 8) __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more) queue_next();
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
  constexpr int PITCH = WN * 32 + 4, LPR = WN * 4;          // floats of a row, lanes to a row
  __syncthreads();                                          // the ring is done with
  float* const stage = reinterpret_cast<float*>(lds) + wave * 32 * PITCH;
  const int n = (int)wn0 + lane % LPR * 8;
  const int have = (int)min((long long)8, p.N - n);
#pragma unroll
  for (int i = 0; i < WM; ++i) {
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(stage + l32 * PITCH + j * 32 + 8 * q + 4 * lhi) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
#pragma unroll 2
    for (int r = lane / LPR; r < 32; r += 64 / LPR) {
      const long long m = wm0 + i * 32 + r;
      float v[8];
      *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(stage + r * PITCH + lane % LPR * 8);
      *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(stage + r * PITCH + lane % LPR * 8 + 4);
      if (m < p.M && have > 0) {
        if (g.vec) finish_run<T, 8>(p.e, m * p.N + n, n, have, v);
        else finish_run<T, 1>(p.e, m * p.N + n, n, have, v);
      }
    }
  }
}

template <int W> constexpr size_t dma_lds(int wm, int wn) { return std::max<size_t>((size_t)kRing * 64 * 64 * (wm + wn), (size_t)4 * 32 * (wn * 32 + 4) * 4); }

template <typename T, int W>
int launch(const DmaArgs& g, bool ao, bool bo, void* stream) {
  const size_t bytes = dma_lds<W>(W, W);
  auto fn = ao ? &product_dma_kernel<T, W, W, true, true> : bo ? &product_dma_kernel<T, W, W, false, true> : &product_dma_kernel<T, W, W, false, false>;
  if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(fn), bytes)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)(g.per_xcd * kXcds)), dim3(256), bytes, as_stream(stream), g);
  WC_CHECK_LAUNCH("product_dma_kernel");
  return WC_OK;
}

}  // namespace

bool product_dma_fits(const LinearProduct& p, int dtype) {
  auto fits = [](const void* q, long long ld, bool outer, long long R) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0 && (outer || R % 8 == 0) && ld < (1 << 21);
  };
  return dtype != WC_F32 && fits(p.a, p.lda, p.a_outer, p.R) && fits(p.b, p.ldb, p.b_outer, p.R) && (!p.a_outer || p.b_outer);
}

int product_dma(const LinearProduct& p, int w, int s, long long R_part, float* parts, int dtype, void* stream) {
  DmaArgs g;
  g.p = p;
  g.parts = parts;
  g.R_part = R_part;
  const long long tm = ceil_div_ll(p.M, 64 * w), tn = ceil_div_ll(p.N, 64 * w);
  g.tiles_m = (int)tm; g.tiles_n = (int)tn;
  g.n_blocks = (int)(tm * tn * s);
  g.per_xcd = ceil_div(g.n_blocks, kXcds);
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.e.y) | reinterpret_cast<uintptr_t>(p.e.z) | reinterpret_cast<uintptr_t>(p.e.res);
  g.vec = p.N % 8 == 0 && at % 16 == 0;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) return w == 4 ? launch<T, 4>(g, p.a_outer, p.b_outer, stream) : w == 2 ? launch<T, 2>(g, p.a_outer, p.b_outer, stream) : launch<T, 1>(g, p.a_outer, p.b_outer, stream);
    else return fail(WC_ERR_UNSUPPORTED, "product_dma: a 16-bit kernel");
  });
}

}  // namespace wc
