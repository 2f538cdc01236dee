// Tensors in 4 bits, the OCP microscaling formats' MXFP4: the groups of 32 neighbouring channels of a row share a scale 2^e, a value is one of
// +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} (e2m1) times it.
//
// Layout.  Rows are padded to whole stages of 128 channels, whose codes are zero: a stage is 64 bytes of a row.  codes (rows, Cp / 2) bytes, the lower
// channel in a byte's low half.  scales, e + 127, in blocks of 32 rows: (ceil(rows / 32), Cp / 128, 32, 4) bytes, so that the four scales of a
// stage are one word of a row and those of 32 rows one line of the L2: a tile of a product brings them by whole 16-byte loads.  (In rows of
// Cp / 32 bytes the same words lie a row apart, a line each.)  Scales of padding are 0.
#pragma once
#include "linear_rows.h"

namespace wc {

constexpr int kGroup4 = 32, kStage4 = 128, kRows4 = 32;
constexpr int kMostChannels4 = 1 << 22;          // rows of 256 by 2^21 bytes stay within 31-bit offsets
__host__ __device__ inline long long padded4(long long C) { return (C + kStage4 - 1) / kStage4 * kStage4; }
__host__ __device__ inline long long stages4(long long C) { return (C + kStage4 - 1) / kStage4; }
inline long long scale_bytes4(long long rows, long long C) { return ceil_div_ll(rows, kRows4) * stages4(C) * (kRows4 * 4); }
// where the scale of a row's group lies
__device__ __forceinline__ long long scale_at4(long long row, long long group, long long stages) {
  return ((row / kRows4) * stages + group / 4) * (kRows4 * 4) + (row % kRows4) * 4 + group % 4;
}

// The conversions take a scale as the exponent bits of a float: 0 is 2^-127, 255 makes every value NaN
__device__ __forceinline__ float scale4(unsigned e) { return __uint_as_float(e << 23); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// the two values of byte B of four
template <typename T, int B>
__device__ __forceinline__ Pack<T, 2> pair4(unsigned codes, float scale) {
  Pack<T, 2> r;
  if constexpr (std::is_same<T, bf16_t>::value) {
    const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B);
    r.v[0] = v[0]; r.v[1] = v[1];
  } else if constexpr (std::is_same<T, half_t>::value) {
    const f16x2 v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, B);
    r.v[0] = v[0]; r.v[1] = v[1];
  } else {
    const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, B);
    r.v[0] = v[0]; r.v[1] = v[1];
  }
  return r;
}
// the eight values of a word, each exact in T where T holds it, else T's nearest
template <typename T>
__device__ __forceinline__ void values4(unsigned codes, float scale, T (&v)[8]) {
  const Pack<T, 2> a = pair4<T, 0>(codes, scale), b = pair4<T, 1>(codes, scale), c = pair4<T, 2>(codes, scale), d = pair4<T, 3>(codes, scale);
  v[0] = a.v[0]; v[1] = a.v[1]; v[2] = b.v[0]; v[3] = b.v[1]; v[4] = c.v[0]; v[5] = c.v[1]; v[6] = d.v[0]; v[7] = d.v[1];
}

// pack4.hip
int pack4(const void* x, unsigned char* codes, unsigned char* scales, long long rows, int C, int dtype, void* stream);
int unpack4(const unsigned char* codes, const unsigned char* scales, void* x, long long rows, int C, int dtype, void* stream);

// y = act(x wT + b + r), one operand or both in 4 bits; p's a (x as it is) and b are null where they are packed
struct Operand4 { const unsigned char* codes; const unsigned char* scales; };
// linear4_few.hip: few rows of x, a pass over w for each 16 (a call takes at most kMostFew4)
constexpr int kMostFew4 = 128;
int product4_few(const LinearProduct& p, const Operand4* x, const Operand4& w, int dtype, void* stream);
// linear4_gradient.hip: dx = dz w, passes over the codes of w (K, C); parts: (linear4_gradient_parts, M, C), where those are more than one
// us, passes of 64 rows | the weight widened first: fp16 512 rows of 8192 <- 8192 97 | 133, of 25088 <- 4096 176 | 176; fp32, whose three bf16 products are faster than
// one of fp32 operands, passes of 32: 4096 rows 1674 | 4219 and 2747 | 6580 (2^20: a launch's passes)
inline int most_gradient4(int dtype) { return dtype == WC_F32 ? 1 << 20 : 512; }
int linear4_gradient_parts(long long M, long long K, long long C, int dtype);
int linear4_gradient(const void* dz, const Operand4& w, void* dx, float* parts, long long M, int K, int C, int dtype, void* stream);
// linear4_wide.hip: more rows of 16-bit x (rows of whole 16 bytes), w's codes widened in the registers.  R_part of its plan is in stages
constexpr int kMostWide4 = 2048;
bool linear4_wide_fits(const void* x, long long C, int dtype);
ProductPlan linear4_wide_plan(const LinearProduct& p);
int linear4_wide(const LinearProduct& p, const Operand4& w, const ProductPlan& plan, float* parts, int dtype, void* stream);
// linear4_dma.hip: both operands in 4 bits, on tiles.  Extents of p in channels, R padded
ProductPlan product4_plan(const LinearProduct& p);
int product4_dma(const LinearProduct& p, const Operand4& x, const Operand4& w, const ProductPlan& plan, float* parts, int dtype, void* stream);
// linear_product.hip: tiles and parts of a product in elements of 16 bits
ProductPlan product_plan4(const LinearProduct& p, bool heavy);

}  // namespace wc
