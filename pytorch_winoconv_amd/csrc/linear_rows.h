// Device code over rows of tensors that start anywhere: runs of elements, 8-bit groups back to their type, copies to rows of whole 16 bytes.
#pragma once
#include "linear.h"

namespace wc {

// N elements that start anywhere, of which `have` are there
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Run { T v[N]; };
template <typename T, int N>
__device__ __forceinline__ void load_run(const void* from, long long i, int have, T (&v)[N]) {
  const T* const p = static_cast<const T*>(from) + i;
  if (have >= N) {
    const Run<T, N> r = *reinterpret_cast<const Run<T, N>*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = r.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = static_cast<T>(0);
    if (have > 0) {
      // (loads that no branch stands before wait for each other less)
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = p[min(e, have - 1)];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = e < have ? v[e] : static_cast<T>(0);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_run(void* to, long long i, int have, const T (&v)[N]) {
  T* const p = static_cast<T*>(to) + i;
  if (have >= N) {
    Run<T, N> r;
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[e] = v[e];
    *reinterpret_cast<Run<T, N>*>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < have) p[e] = v[e];
  }
}

// What becomes of one sum of a product
template <typename T>
__device__ __forceinline__ void finish_one(const LinearEpilogue& e, long long m, long long n, long long N, float v) {
  const long long i = m * N + n;
  if (e.bias) v += static_cast<float>(static_cast<const T*>(e.bias)[n]);
  const float r = e.res ? static_cast<float>(static_cast<const T*>(e.res)[i]) : 0.f;
  if (!e.res_after) v += r;
  if (e.z) static_cast<T*>(e.z)[i] = static_cast<T>(v);
  v = activate(v, e.act);
  if (e.res_after) v += r;
  if (e.y_f32) static_cast<float*>(e.y)[i] = v;
  else static_cast<T*>(e.y)[i] = static_cast<T>(v);
}

// Workgroup `block` of 256 threads: rows of 8 bits back to T in rows of ld, zeros behind C; eight threads a group, four elements each
struct UnpackArgs {
  long long first;           // workgroup of the launch, where it does nothing else
  const signed char* codes; const signed char* exps;
  void* out;
  long long groups, ld;      // groups of all rows
  int C, row_groups;
};
constexpr int kUnpackGroups = 32;          // of a workgroup
template <typename T>
__device__ __forceinline__ void unpack_block(const UnpackArgs& a, long long block) {
  const long long g = block * kUnpackGroups + (threadIdx.x >> 3);
  if (g >= a.groups) return;
  const long long row = a.groups < (1ll << 31) ? (unsigned)g / (unsigned)a.row_groups : g / a.row_groups;
  const int c0 = (int)(g - row * a.row_groups) * kPackGroup + (threadIdx.x & 7) * 4;
  const float step = pack_step(a.exps[g]);
  signed char q[4];
  load_run<signed char, 4>(a.codes, row * a.C + c0, a.C - c0, q);
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(c0 + e < a.C ? (float)q[e] * step : 0.f);
  store_run<T, 4>(a.out, row * a.ld + c0, (int)min(a.ld - c0, 4ll), v);
}

// The same where rows are whole groups and lie as they are: a thread takes eight neighbouring elements four times
constexpr int kLine = 256 * 8 * 4;         // elements of a workgroup
template <typename T>
__device__ __forceinline__ void unpack_line_block(const UnpackArgs& a, long long block) {
  const long long total = a.groups * kPackGroup, first = block * kLine + threadIdx.x * 8;
  Pack<signed char, 8> q[4];
  int e[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long i = min(first + j * 2048, total - 8);
    q[j] = *reinterpret_cast<const Pack<signed char, 8>*>(a.codes + i);
    e[j] = a.exps[i / kPackGroup];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float step = pack_step(e[j]);
    T v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = static_cast<T>((float)q[j].v[k] * step);
    if (first + j * 2048 < total) store_run<T, 8>(a.out, first + j * 2048, 8, v);
  }
}
inline bool on_a_line(int C, const void* x, const void* codes) {
  return C % kPackGroup == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
}
inline long long unpack_blocks(const UnpackArgs& a, bool line) { return line ? ceil_div_ll(a.groups * kPackGroup, kLine) : ceil_div_ll(a.groups, kUnpackGroups); }

// Workgroup `block` of a matrix copied to rows of c.ld, zeros behind its columns; eight elements a thread
template <typename T>
__device__ __forceinline__ void widen_block(const WideCopy& c, long long block) {
  const long long i = block * 256 + threadIdx.x, wide = (c.ld + 7) / 8, row = i / wide, k = (i - row * wide) * 8;
  if (row >= c.rows) return;
  T v[8];
  load_run<T, 8>(c.from, row * c.C + k, (int)max(min(c.C - k, 8ll), 0ll), v);
  store_run<T, 8>(c.to, row * c.ld + k, (int)min(c.ld - k, 8ll), v);
}
inline long long widen_blocks(const WideCopy& c) { return ceil_div_ll(c.rows * ((c.ld + 7) / 8), 256); }

}  // namespace wc
