// What joins a block to its stream, over rows of channels:
//   n = post(f),  d = drop(n),  s = a x + b g d,  y = pre(s)
// post and pre are norms (RMS: v w / sqrt(mean(v^2) + eps); layer: (v - mean) w / sqrt(var + eps) + bias) or nothing, g a gate of one row of channels, a row
// a sample, or one a row; x, gate and dropout may be missing.  A norm alone is y = pre(f), dropout alone s = drop(f).
//
// All of it is bound by memory, so a row is read once and stays in registers: a team of threads holds it, eight neighbouring channels a thread, sixteen of the
// longest.  A team is a part of a wavefront of as many lanes as the row has vectors of eight, or a workgroup.  Means and variances are taken one after
// the other from the registers, not from sums of squares, which cancel where the mean is large.
#pragma once
#include "linear_rows.h"

namespace wc {

struct Norm { int kind; float eps; const void* weight; const void* bias; int wide; };      // wide: parameters in fp32

// level / 65536 is the probability; keys by the host, or in device memory (seed, offset), for launches that are captured
struct Dropout {
  unsigned level;
  int per_sample;
  float scale;
  unsigned long long seed, offset;
  const unsigned long long* state;
};

enum GateRows { kNoGate, kGateChannel, kGateSample, kGateRow };

struct JoinArgs {
  long long rows, per;         // per: rows of a sample
  int C;
  const void* f; const void* x; const void* gate;
  int gate_rows, gate_wide;
  float a, b;
  Norm post, pre;
  Dropout drop;
  void* s; void* y;            // null: not written
  float* post_stats; float* pre_stats;      // (rows, 2): mean, inverse deviation; null: not kept
};

struct JoinGradients {
  long long rows, per;
  int C;
  const void* ds; const void* dy;          // null: none
  const void* f; const void* s; const void* x; const void* gate;      // pre's s null: computed again from f and x (null: there is no stream)
  int gate_rows, gate_wide;
  float a, b;
  Norm post, pre;
  Dropout drop;
  const float* post_stats; const float* pre_stats;
  void* df; void* dx;                      // null: not asked for
  void* dgate_rows;                        // gate of a row a row: written at once, of the type of gate_wide
  float* part[5];                          // sums of pre's weight and bias, post's weight and bias, gate: (blocks, C) each; null: not asked for
  long long segments;                      // of rows: samples, or 1
  int parts;                               // workgroups a segment, where there are no more segments than workgroups
  int blocks;
};
enum { kPreWeight, kPreBias, kPostWeight, kPostBias, kGateSum };

// ---- dropout --------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011).  Its four words are eight of 16 bits, one for each of
// the eight channels that a thread holds: probabilities are whole multiples of 2^-16, and what is kept is divided by exactly the share that is.
// 32 bits a channel would double its 20 products of 32 x 32 bits, which at eight channels take about as long as the channels' way from memory.
struct Random8 { unsigned w[4]; };
__device__ __forceinline__ Random8 philox(unsigned c0, unsigned c1, unsigned long long offset, unsigned long long seed) {
  unsigned x0 = c0, x1 = c1, x2 = (unsigned)offset, x3 = (unsigned)(offset >> 32), k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  asm volatile("" : "+s"(k0), "+s"(k1));         // (the rounds' keys, kept over the loop over rows, would be spilled)
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p = 0xD2511F53ull * x0, q = 0xCD9E8D57ull * x2;
    x0 = (unsigned)(q >> 32) ^ x1 ^ k0;
    x1 = (unsigned)q;
    x2 = (unsigned)(p >> 32) ^ x3 ^ k1;
    x3 = (unsigned)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{x0, x1, x2, x3}};
}
struct Keys { unsigned long long seed, offset; };
// (the same for all: in scalar registers)
__device__ __forceinline__ unsigned long long uniform(unsigned long long v) {
  return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ Keys keys_of(const Dropout& d) {
  Keys k = {d.seed, d.offset};
  if (d.state) k = {uniform(d.state[0]), uniform(d.state[1])};
  return k;
}

// what channels 8 j .. of a row are multiplied by is `scale` where the bit of the mask is set, and 0 - whatever the value - where it is not
__device__ __forceinline__ unsigned kept8(const Dropout& d, const Keys& k, unsigned j, unsigned row) {
  const Random8 r = philox(j, row, k.offset, k.seed);
  unsigned mask = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) mask |= ((r.w[e / 2] >> (16 * (e & 1)) & 0xffffu) >= d.level ? 1u : 0u) << e;
  return mask;
}
__device__ __forceinline__ unsigned kept_sample(const Dropout& d, const Keys& k, unsigned sample) {
  return (philox(0, sample, k.offset, k.seed).w[0] & 0xffffu) >= d.level ? 255u : 0u;
}

// ---- rows in registers ------------------------------------------------------------------------
// A team: `lanes` neighbouring lanes of a wavefront (a power of two), or, WAVES above 1, the workgroup
template <int WAVES>
struct Team {
  int lanes;
  float* lds;                  // WAVES above 1: two rows of 2 WAVES
  int turn;
  // (exchanges within 16 lanes are operands of the additions; mirrored, not across, which is the same once the halves agree)
  template <int CONTROL> static __device__ __forceinline__ void add_across(float& u) {
    u += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(u), CONTROL, 0xf, 0xf, true));
  }
  __device__ __forceinline__ void sum(float& u, float& v) {
    const int n = WAVES > 1 ? 64 : lanes;
    constexpr int kPairs = 0xB1, kQuads = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;
    if (n > 1) { add_across<kPairs>(u); add_across<kPairs>(v); }
    if (n > 2) { add_across<kQuads>(u); add_across<kQuads>(v); }
    if (n > 4) { add_across<kHalfMirror>(u); add_across<kHalfMirror>(v); }
    if (n > 8) { add_across<kMirror>(u); add_across<kMirror>(v); }
    if (n > 16) { u += __shfl_xor(u, 16); v += __shfl_xor(v, 16); }
    if (n > 32) { u += __shfl_xor(u, 32); v += __shfl_xor(v, 32); }
    if constexpr (WAVES > 1) {
      // (the two rows take turns, so that one barrier is enough: before a row is written again everyone has passed the other's)
      float* const row = lds + turn * 2 * WAVES;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
        row[threadIdx.x >> 6] = u;
        row[WAVES + (threadIdx.x >> 6)] = v;
      }
      __syncthreads();
      u = v = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        u += row[w];
        v += row[WAVES + w];
      }
    }
  }
  __device__ __forceinline__ float sum(float u) {
    float none = 0.f;
    sum(u, none);
    return u;
  }
};

// Channels c .. c + 7 of a row of C, zeros behind its end: one 16-byte load (fp32: two) wherever it starts.  That of an odd row's last channels starts
// before them, and what is in front is shifted out; lanes behind the row's end, or of no row, load something that is there.  The load stands behind no
// branch and the shift where the values are wanted (settled8), so that all loads of a row are on their way at once.
// `there`: the row is, else zeros.
// Rows of whole vectors (C a multiple of eight), others, and those of fewer than eight channels
enum { kEven, kOdd, kTiny };
template <typename T> struct Raw8 { uint32_t w[2 * sizeof(T)]; };
template <typename T, int ROW>
__device__ __forceinline__ Raw8<T> load8(const void* p, long long row, int c, int C, bool there) {
  Raw8<T> r;
  if constexpr (ROW != kOdd) {
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) r.w[i] = 0u;
    if (!there || c >= C) return r;
    T v[8];
    load_run<T, 8>(p, row * C + c, ROW == kEven ? 8 : C - c, v);
    __builtin_memcpy(&r, v, sizeof(r));
  } else {
    const Run<T, 8> v = *reinterpret_cast<const Run<T, 8>*>(static_cast<const T*>(p) + (there ? row : 0) * C + min(c, C - 8));
    __builtin_memcpy(&r, &v, sizeof(r));
  }
  return r;
}
template <typename T, int ROW>
__device__ __forceinline__ Raw8<T> settled8(Raw8<T> r, int c, int C, bool there) {
  if (ROW != kOdd) return r;
  constexpr int W = 2 * sizeof(T);
  int k = c - (C - 8);                                 // channels in front
  if (!there || c >= C) {
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = 0u;
  } else if (k > 0) {
    asm volatile("" : "+v"(k));                        // (compared anew: its bits as masks, kept over the loop over rows, would be spilled)
    // by whole words, then by half a one
    constexpr int ONE = sizeof(T) == 4 ? 1 : 0;        // words of a shift by one element
#pragma unroll
    for (int bit = 4; bit >= (ONE ? 1 : 2); bit /= 2) {
      const int words = bit * (int)sizeof(T) / 4;
#pragma unroll
      for (int i = 0; i < W; ++i) r.w[i] = k & bit ? (i + words < W ? r.w[i + words] : 0u) : r.w[i];
    }
    if constexpr (!ONE) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint32_t next = i + 1 < W ? r.w[i + 1] : 0u;
        r.w[i] = k & 1 ? r.w[i] >> 16 | next << 16 : r.w[i];
      }
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void floats_of(const Raw8<T>& r, float (&v)[8]) {
  T t[8];
  __builtin_memcpy(t, &r, sizeof(r));
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(t[e]);
}
template <typename T, int ROW>
__device__ __forceinline__ void parameter8(const void* p, int wide, long long row, int c, int C, float (&v)[8], float otherwise) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = otherwise;
  } else if (wide) {
    floats_of<float>(settled8<float, ROW>(load8<float, ROW>(p, row, c, C, true), c, C, true), v);
  } else {
    floats_of<T>(settled8<T, ROW>(load8<T, ROW>(p, row, c, C, true), c, C, true), v);
  }
}
// x where element e of `have` is there, 0 where it is not; of whole vectors eight are there or none, whose x is 0 as it is
template <int ROW> __device__ __forceinline__ float kept_element(float x, int e, int have) { return ROW == kEven || e < have ? x : 0.f; }

template <typename T>
__device__ __forceinline__ void load_floats(const void* p, long long i, int have, float (&v)[8]) {
  T t[8];
  load_run<T, 8>(p, i, have, t);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(t[e]);
}
template <typename T>
__device__ __forceinline__ void load_parameter(const void* p, int wide, long long i, int have, float (&v)[8], float otherwise) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = otherwise;
  } else if (wide) {
    load_floats<float>(p, i, have, v);
  } else {
    load_floats<T>(p, i, have, v);
  }
}
template <typename T>
__device__ __forceinline__ void store_floats(void* p, long long i, int have, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = static_cast<T>(v[e]);
  store_run<T, 8>(p, i, have, t);
}

__device__ __forceinline__ long long gate_row(int gate_rows, long long row, long long per) {
  return gate_rows == kGateChannel ? 0 : gate_rows == kGateRow ? row : (unsigned)row / (unsigned)per;
}

// a team's shape for rows of C channels: vectors of eight a thread, wavefronts, lanes of a wavefront
struct TeamShape { int vectors, waves, lanes; };

int join_forward(const JoinArgs& a, int dtype, void* stream);
int join_backward(const JoinGradients& g, int dtype, void* stream);
template <typename T> int join_backward_of(const JoinGradients& g, void* stream);      // residual_backward.inc
TeamShape back_shape(const JoinGradients& g);
// how many workgroups, and in how many parts a segment, a backward pass takes
void join_plan(JoinGradients* g);
// dst[which] = the sums of part[which] over the workgroups (gate of a sample: over a sample's)
struct JoinSum { const float* part; void* dst; int wide; long long segments; int parts; };
int join_sums(const JoinSum* sums, int n, int C, int dtype, void* stream);

}  // namespace wc
