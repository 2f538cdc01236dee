// Matrix products with an epilogue, y = act(x wT + b + r) or act(x wT + b) + r, and what their gradients share.
#pragma once
#include "wc_common.h"

namespace wc {

// ---- activations, in fp32 ---------------------------------------------------------------------
// e^v and 1 / v by the hardware's 2^v and reciprocal: within 2 ulp, and e^v within |v| 2^-24 more, the rounding of v log2(e)
__device__ __forceinline__ float fast_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float fast_rcp(float v) { return __builtin_amdgcn_rcpf(v); }
__device__ __forceinline__ float finite(float v) { return v > 3.402823466e38f ? 3.402823466e38f : v < -3.402823466e38f ? -3.402823466e38f : v; }

// Normal distribution: the density times sqrt(2 pi), e^(-z^2 / 2), and the distribution Phi(z) = erfc(-z / sqrt 2) / 2.
// erfc(a) = e^(-a^2) t P(t) with t = 1 / (1 + 0.3 a) for a >= 0, P of degree 8 fitted to e^(a^2) erfc(a) / t on 0 <= a <= 10 in the relative
// error (2e-8 in exact arithmetic, 5e-7 in fp32), beyond which e^(-a^2) is 0 in fp32.  No cancellation for negative z, and some twenty
// instructions; 1 + erf(z / sqrt 2) has no digits left below z = -5.
struct Normal { float density, below; };
__device__ __forceinline__ Normal normal_of(float z) {
  const float a = fabsf(z) * 0.70710678f;
  const float t = fast_rcp(fmaf(0.3f, a, 1.f));
  float p = -0.12952517f;
  p = fmaf(p, t, 0.48557463f);
  p = fmaf(p, t, -0.51230263f);
  p = fmaf(p, t, 0.54774936f);
  p = fmaf(p, t, -0.094672005f);
  p = fmaf(p, t, 0.21493564f);
  p = fmaf(p, t, 0.14833656f);
  p = fmaf(p, t, 0.17071562f);
  p = fmaf(p, t, 0.16918798f);
  const float d = fast_exp(-a * a);
  const float tail = 0.5f * t * p * d;
  return {d, z < 0.f ? tail : 1.f - tail};
}
__device__ __forceinline__ float logistic(float v) { return fast_rcp(1.f + fast_exp(-v)); }
constexpr float kTanhScale = 1.59576912f;        // 2 sqrt(2 / pi): (1 + tanh(u)) / 2 is the logistic function of 2 u

// (an infinity times a zero is no number: gelu and silu of -infinity are their limit 0)
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case WC_ACT_RELU: return z < 0.f ? 0.f : z;                    // NaN stays
    case WC_ACT_GELU: return z == -__builtin_inff() ? 0.f : z * normal_of(z).below;
    case WC_ACT_GELU_TANH: return z == -__builtin_inff() ? 0.f : z * logistic(kTanhScale * (z + 0.044715f * z * z * z));
    case WC_ACT_SILU: return z == -__builtin_inff() ? 0.f : z * logistic(z);
    default: return z;
  }
}
// dy times the derivative
__device__ __forceinline__ float through(float dy, float z, int act) {
  switch (act) {
    case WC_ACT_RELU: return z > 0.f ? dy : z <= 0.f ? 0.f : z;    // a z that is no number says nothing about dy
    case WC_ACT_GELU: {
      const Normal n = normal_of(z);
      return dy * fmaf(finite(z) * n.density, 0.39894228f, n.below);
    }
    case WC_ACT_GELU_TANH: {
      const float f = finite(z), g = logistic(kTanhScale * (f + 0.044715f * f * f * f));
      const float h = g * (1.f - g);               // 0 beyond |z| = 10, where z^3 of it may be infinite
      return dy * (h == 0.f ? g : fmaf(h * f * kTanhScale, fmaf(0.134145f * f, f, 1.f), g));
    }
    case WC_ACT_SILU: {
      const float g = logistic(z);
      return dy * fmaf(finite(z) * g, 1.f - g, g);
    }
    default: return dy;
  }
}

// ---- launches -----------------------------------------------------------------------------------
// A launch has fewer than 2^32 threads along an axis.  Workgroups, of at most 512 threads, that one takes; work of more goes in several
constexpr long long kMostBlocks = (1ll << 23) - kXcds;
// launch(first, n) over workgroups first .. first + n - 1 of `blocks`
template <typename F>
int in_launches(long long blocks, F&& launch) {
  for (long long first = 0; first < blocks; first += kMostBlocks) {
    const long long left = blocks - first;
    if (int rc = launch(first, (unsigned)(left < kMostBlocks ? left : kMostBlocks))) return rc;
  }
  return WC_OK;
}

// ---- products -----------------------------------------------------------------------------------
// What becomes of a sum v of a product: v + bias[n] (+ r) is rounded to z where that is asked for, act(it) (+ r) to y.
struct LinearEpilogue {
  const void* bias;         // N values; null: none
  const void* res;          // (M, N); null: none
  void* y;                  // (M, N) of the operands' type, or fp32
  void* z;                  // (M, N); null: not asked for
  int act, res_after, y_f32;
};
// y (M, N) = the sums over the R reduction elements of A (M, R) or, outer, (R, M), and B (N, R) or, outer, (R, N)
struct LinearProduct {
  const void* a; const void* b;
  long long lda, ldb;       // elements between rows as they lie
  bool a_outer, b_outer;
  long long M, N, R;
  LinearEpilogue e;
};
inline bool linear_heavy(const LinearEpilogue& e) { return e.act != WC_ACT_NONE || e.z || e.res; }
// linear_product.hip: how a product is run - on which kernel and tiles, in how many parts of the reduction - and the launches.  Parts leave
// their sums (s, M, N) in fp32, which linear_join adds.
struct ProductTile { int m, n; };
struct ProductPlan { bool dma, few; ProductTile tile; int s; long long R_part; };
ProductPlan product_plan(const LinearProduct& p, int dtype, const LinearProduct* beside);      // beside: runs in the same launch; null: none
size_t product_parts_bytes(const LinearProduct& p, int dtype, const LinearProduct* beside);      // enough for every start of the operands and every epilogue
int product_run(const LinearProduct& p, const ProductPlan& plan, float* parts, int dtype, void* stream);
// both, in one launch where their plans allow it
int product_run_pair(const LinearProduct& p, const ProductPlan& plan, float* parts, const LinearProduct& p2, const ProductPlan& plan2, float* parts2, int dtype, void* stream);

// linear_dma.hip: products whose rows are multiples of 16 bytes, on tiles of 256 x 256 (16-bit types), 128 x 128 or 64 x 64
bool product_dma_fits(const LinearProduct& p, int dtype);
int product_dma(const LinearProduct& p, const ProductPlan& plan, float* parts, int dtype, void* stream);
bool product_dma_pairs(const ProductPlan& plan, const ProductPlan& plan2);
int product_dma_pair(const LinearProduct& p, const ProductPlan& plan, float* parts, const LinearProduct& p2, const ProductPlan& plan2, float* parts2, int dtype, void* stream);

// Matrices copied to rows that are multiples of 16 bytes, zeros behind their columns
struct WideCopy { const void* from; void* to; long long rows, C, ld; };
// dz (rows, K) = dy act'(z), rounded, and db[k] = the sum of column k before that rounding.  z of the storage type, or codes with their
// exponents; dz null: none, db null: none
struct LinearSlope {
  const void* dy; const void* z; const signed char* z_exp;
  void* dz; void* db;
  void* dz_wide; long long ld_wide;      // dz in rows of ld_wide (a multiple of 16 bytes), zeros behind K; null: none
  int act, db_f32;
  long long rows; int K;
};
// linear_gradient.hip: what stands before the products, in one launch: dz, copies, 8 bits read back (codes null: none) to rows of x_ld
struct LinearPrepare {
  bool run_slope;
  LinearSlope slope;
  WideCopy copies[2];
  int n_copies;
  const signed char* codes; const signed char* exps;
  void* x;
  long long x_rows, x_ld; int x_C;
};
size_t linear_sums_bytes(const LinearSlope& s);                     // of the columns' sums; 0: the first launch writes db itself
int linear_prepare(const LinearPrepare& p, int dtype, float* sums, void* stream);
// ... and behind them, in one launch: the parts of up to two products (s of 1: none) and the columns' sums (sums null: none)
struct LinearJoin { LinearEpilogue e; const float* parts; int s; long long M, N; };
int linear_join(const LinearJoin* joins, int n, const LinearSlope* slope, const float* sums, int dtype, void* stream);

// pack8.hip
constexpr int kPackGroup = 32;
__host__ __device__ inline long long pack_groups(long long C) { return (C + kPackGroup - 1) / kPackGroup; }
// the step of a group: 2^e from the exponent's bits, no number where the group had one
constexpr int kPackNoNumber = 127, kPackLeast = -126;
__device__ __forceinline__ float pack_step(int e) {
  return e == kPackNoNumber ? __builtin_nanf("") : __uint_as_float((unsigned)(e + 127) << 23);
}
constexpr int kPackSigns = 1, kPackGates = 2;                // of keep_sign
// what relu's gate is read from: codes of a group with an infinity or a NaN as pack8.hip leaves them for it, where 0 (times an infinity) is no number
__device__ __forceinline__ float gate_step(int e) { return e == kPackNoNumber ? __builtin_inff() : pack_step(e); }
int pack8(const void* x, signed char* codes, signed char* exps, long long rows, int C, int keep_sign, int dtype, void* stream);
int unpack8(const signed char* codes, const signed char* exps, void* x, long long rows, int C, int dtype, void* stream);
inline long long wide_row(long long C, int dtype) { const int epc = dtype == WC_F32 ? 4 : 8; return (C + epc - 1) / epc * epc; }

}  // namespace wc
