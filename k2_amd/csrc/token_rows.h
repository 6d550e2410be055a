// What the operators on rows of output logits share (token_logprobs.hip, distillation.hip): the three element types, and
// the two numbers that a row's softmax is kept as.
//
// A row of C logits x at temperature tau is kept as its largest logit m and log2 s, s = sum_i 2^d_i with
// d_i = (x_i - m) c, c = log2(e) / tau; then log p_i = ln2 (d_i - log2 s).  The difference is formed in the logits' own
// scale, before c multiplies it: it is exact or one rounding off for every pair of logits, and rows that a mask has filled
// with the type's lowest value stay rows of equal logits (c x alone would overflow).  m is the row's largest logit, or 0
// where that is -inf (a row that a mask left nothing of): then s = 0 and every p_i is 0.
#ifndef K2_AMD_CSRC_TOKEN_ROWS_H_
#define K2_AMD_CSRC_TOKEN_ROWS_H_

#include "common.h"

namespace k2amd {
namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr double kLog2E = 1.442695040888963407;
// a difference d whose 2^d is 0: where d itself is a factor beside 2^d, the products of -inf logits have to be 0, not NaN
constexpr float kNothing = -1024.0f;
constexpr int kMaxTokens = 64;        // given tokens of a row
constexpr int kMaxTop = 64;           // listed alternatives of a row
constexpr int kMaxTeacher = 256;      // entries of a teacher's list

// the bits of one 16-bit element and back (to nearest even)
struct Half {
  unsigned short bits;
};
struct Bfloat {
  unsigned short bits;
};
__device__ __forceinline__ float HalfToFloat(unsigned short u) {
  return static_cast<float>(__builtin_bit_cast(_Float16, u));
}
__device__ __forceinline__ unsigned short FloatToHalf(float f) {
  return __builtin_bit_cast(unsigned short, static_cast<_Float16>(f));
}
__device__ __forceinline__ unsigned short FloatToBfloat(float f) {
  return __builtin_bit_cast(unsigned short, static_cast<__bf16>(f));
}
__device__ __forceinline__ float ToFloat(float x) { return x; }
__device__ __forceinline__ float ToFloat(Half x) { return HalfToFloat(x.bits); }
__device__ __forceinline__ float ToFloat(Bfloat x) { return __uint_as_float((unsigned)x.bits << 16); }
__device__ __forceinline__ void FromFloat(float f, float *x) { *x = f; }
__device__ __forceinline__ void FromFloat(float f, Half *x) { x->bits = FloatToHalf(f); }
__device__ __forceinline__ void FromFloat(float f, Bfloat *x) { x->bits = FloatToBfloat(f); }

__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float Log2(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ float WaveMaxF(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
  return v;
}
__device__ __forceinline__ float WaveSumF(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// log p of an element with logit x, in the natural logarithm's scale throughout: (x - m) c could overflow where this does not
__device__ __forceinline__ float LogProb(float x, float m, float ls, float inv_tau) {
  return ls == Real<float>::NegInf() ? Real<float>::NegInf() : (x - m) * inv_tau - kLn2 * ls;
}

// The order of alternatives as one whole number: the larger logit first (a NaN before everything, -0 and 0 alike), the
// lower index first where logits are equal.  Never 0 for an element of a row.
__device__ __forceinline__ unsigned OrderOf(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long KeyOf(float x, unsigned index) {
  return ((unsigned long long)OrderOf(x) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ unsigned IndexOf(unsigned long long key) { return 0xffffffffu - (unsigned)key; }

inline bool RowsOk(long long rows, long long row_stride, int C, float temperature, int dtype) {
  if (rows < 0 || C < 1 || row_stride < 0) return false;
  if (!(temperature > 0.0f) || temperature - temperature != 0.0f) return false;
  return dtype == K2AMD_F32 || dtype == K2AMD_F16 || dtype == K2AMD_BF16;
}
// one workgroup of up to 256 work-items a row: a launch holds fewer than 2^32 work-items
inline bool RowsServed(long long rows) { return rows < (1ll << 24); }

}  // namespace
}  // namespace k2amd

#endif  // K2_AMD_CSRC_TOKEN_ROWS_H_
