// What the operators on rows of output logits share (token_logprobs.hip, distillation.hip): the three element types, how a
// wavefront holds its part of a row, and the two numbers that a row's softmax is kept as.
//
// A row of C logits x at temperature tau is kept as its largest logit m and log2 s, s = sum_i 2^d_i with
// d_i = (x_i - m) c, c = log2(e) / tau; then log p_i = (x_i - m) / tau - ln2 log2 s.  The difference is formed in the
// logits' own scale, before c multiplies it: it is exact or one rounding off for every pair of logits, and rows that a mask
// has filled with the type's lowest value stay rows of equal logits (c x alone would overflow).  m is the row's largest
// logit, or 0 where that is -inf (a row that a mask left nothing of): then s = 0 and every p_i is 0.
//
// Everything here is bound by reading the logits, 16 bytes a lane at a time.  Short rows (up to 256 vectors of 16 bytes) stay
// in the registers of 16 lanes each, four rows a wavefront: a reduction is four moves within the 16 lanes that the hardware
// moves data in, for four rows at once, and what is done once a row (its list, its results) is done for four rows at once.
// Longer rows are read along by four wavefronts without being kept, or, where their alternatives are asked for, kept in the
// registers of four wavefronts (4096 vectors) or of several workgroups.  Lane l of group w of W takes, in round u of U, vector
// (u W + w) L + l, with L = 16 or 64 lanes.
//
// Rows start at any element: the loads are unaligned ones.  80000 x 500 takes the same 17 us (bfloat16) and 32 us (float32) as
// 80000 x 501 or a tensor that starts at an odd element; 8192 x 32000 bfloat16, where every load then touches another line,
// 98 us aligned and 112 us not.  The last vector of a row whose length is no multiple of the vector's is read so that it ends
// with the row, and what the vector in front of it holds already is set to -inf in it: no byte outside the row is read,
// without a loop over elements.
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
constexpr int kMaxColumns = 1 << 20;  // columns of a row: 64 parts of what a workgroup holds in 32 bits

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
__device__ __forceinline__ unsigned Narrow(float f, const float *) { return __float_as_uint(f); }
__device__ __forceinline__ unsigned Narrow(float f, const Half *) { return FloatToHalf(f); }
__device__ __forceinline__ unsigned Narrow(float f, const Bfloat *) { return FloatToBfloat(f); }
__device__ __forceinline__ void FromFloat(float f, float *x) { *x = f; }
__device__ __forceinline__ void FromFloat(float f, Half *x) { x->bits = FloatToHalf(f); }
__device__ __forceinline__ void FromFloat(float f, Bfloat *x) { x->bits = FloatToBfloat(f); }

// `v`, as a value that the compiler knows nothing of: what is computed from it is computed here and not kept from before
__device__ __forceinline__ unsigned Anew(unsigned v) {
  asm volatile("" : "+v"(v));
  return v;
}

// 16 bytes of a row: four or eight elements
struct __align__(16) Vec {
  unsigned w[4];
};
typedef unsigned VecAnywhere __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
struct Lanes {
  static constexpr int kN = 16 / sizeof(T);
  static constexpr unsigned kNegInf = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
};
template <>
struct Lanes<Half> {
  static constexpr int kN = 8;
  static constexpr unsigned kNegInf = 0xfc00fc00u;
};
__device__ __forceinline__ float Element(const Vec &v, int e, const float *) { return __uint_as_float(v.w[e]); }
__device__ __forceinline__ float Element(const Vec &v, int e, const Half *) {
  return HalfToFloat((unsigned short)(e & 1 ? v.w[e >> 1] >> 16 : v.w[e >> 1] & 0xffffu));
}
__device__ __forceinline__ float Element(const Vec &v, int e, const Bfloat *) {
  return __uint_as_float(e & 1 ? v.w[e >> 1] & 0xffff0000u : v.w[e >> 1] << 16);
}
template <typename T>
__device__ __forceinline__ float ElementOf(const Vec &v, int e) { return Element(v, e, static_cast<const T *>(nullptr)); }
template <typename T>
__device__ __forceinline__ Vec PackOf(const float *f) {
  Vec v;
  if (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v.w[i] = Narrow(f[2 * i], static_cast<const T *>(nullptr)) | Narrow(f[(2 * i + 1) % Lanes<T>::kN], static_cast<const T *>(nullptr)) << 16;
  }
  return v;
}
// kPast: past the caches, for what is larger than they are
template <bool kPast = false>
__device__ __forceinline__ Vec LoadVec(const void *p) {
  Vec v;
  if (kPast) {
    const VecAnywhere w = __builtin_nontemporal_load(static_cast<const VecAnywhere *>(p));
    __builtin_memcpy(&v, &w, 16);
  } else {
    __builtin_memcpy(&v, p, 16);
  }
  return v;
}
template <bool kPast>
__device__ __forceinline__ void StoreVec(void *p, const Vec &v) {
  if (kPast) {
    const VecAnywhere w = {v.w[0], v.w[1], v.w[2], v.w[3]};
    __builtin_nontemporal_store(w, static_cast<VecAnywhere *>(p));
  } else {
    __builtin_memcpy(p, &v, 16);
  }
}
// Whether a backward pass over long rows reads its logits and writes their gradient past the 256 MB memory-side cache.  The
// gradient would push the logits out of it that the pass has still to read (the end of what the forward pass read), and the
// logits, read for the last time, what else there is: 8191 x 32000 bfloat16 forward and backward take 241 us instead of 287,
// 8192 x 32000 distilled 294 instead of 336.  A gradient that fits is left there for what reads it next; the pass by itself
// would be faster past the cache there too (2048 x 32000 bfloat16, 131 MB: 75 us instead of 88).
inline bool PastCache(long long rows, int C, size_t element) { return (double)rows * C * element > 268435456.0; }

// vectors of a row
template <typename T>
__host__ __device__ __forceinline__ int VecsOf(int C) { return (C + Lanes<T>::kN - 1) / Lanes<T>::kN; }

// where vector q of a row is read: its first element, or for the row's incomplete last vector what makes it end with the
// row (rows of less than a vector: 0)
template <typename T>
__device__ __forceinline__ int VecBase(int q, int C) {
  constexpr int kN = Lanes<T>::kN;
  return max(0, min(q * kN, C - kN));
}

// Vector q of row x (q < VecsOf(C)), elements that belong to the vector in front of it as -inf.  `ragged`: whether q may be the
// row's incomplete last vector.
template <typename T>
__device__ __forceinline__ Vec LoadRowVec(const T *x, int q, int C, bool ragged) {
  constexpr int kN = Lanes<T>::kN;
  Vec v;
  if (!ragged) return LoadVec(x + q * kN);
  if (C < kN) {
    float f[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) f[e] = e < C ? ToFloat(x[e < C ? e : 0]) : Real<float>::NegInf();
    return PackOf<T>(f);
  }
  const int base = VecBase<T>(q, C), skip = q * kN - base;
  v = LoadVec(x + base);
  if (skip > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) {
        if (i < skip) v.w[i] = Lanes<T>::kNegInf;
      } else {
        if (2 * i < skip) v.w[i] = (v.w[i] & 0xffff0000u) | (Lanes<T>::kNegInf & 0xffffu);
        if (2 * i + 1 < skip) v.w[i] = (v.w[i] & 0xffffu) | (Lanes<T>::kNegInf & 0xffff0000u);
      }
    }
  }
  return v;
}

// The U vectors of a row (or of the row's part that starts at vector `first`) that one of W groups of L lanes holds; -inf
// past the row's end.  lane: within the group.
template <typename T, int U, int W, int L = kWave>
struct RowPart {
  Vec v[U];

  __device__ __forceinline__ static int Vector(int u, int first, int wave, int lane) { return first + (u * W + wave) * L + lane; }
  // Vector u as a pass over the vectors reads it: the compiler would otherwise hold all vectors' elements unpacked from one
  // pass to the next (twice the registers for 16-bit types).
  __device__ __forceinline__ const Vec &Packed(int u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[u].w[i] = Anew(v[u].w[i]);
    return v[u];
  }
  // the same as Vector, and likewise not kept from one pass to the next (nor what is compared with it)
  __device__ __forceinline__ static int VectorAnew(int u, int first, int wave, int lane) {
    return (int)Anew((unsigned)Vector(u, first, wave, lane));
  }
  template <bool kPast = false>
  __device__ __forceinline__ void Load(const T *x, int C, int first, int wave, int lane) {
    const int whole = C / Lanes<T>::kN, all = VecsOf<T>(C);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = Vector(u, first, wave, lane);
      const int q_last = first + (u * W + wave) * L + L - 1;  // the same in every lane
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u].w[i] = Lanes<T>::kNegInf;
      if (q_last < whole) v[u] = LoadVec<kPast>(x + q * Lanes<T>::kN);
      else if (q < all) v[u] = LoadRowVec<T>(x, q, C, true);
    }
  }
};

// A gradient's way out.  The columns that a list names differ from the formula of all others.  In rows of up to eight vectors a
// lane all vectors go to LDS first, where the listed columns are written over them, and from there to memory in whole lines
// (`stage` holds the row): 64000 x 500 float32 with lists of 8 take 57 us and not 70, bfloat16 30 and not 44.  Longer rows are
// written to memory and the listed columns over them there, a few partial lines for many whole ones: through LDS, rows of
// 1237 halves took 15.3 us and not 12.5 (for the LDS, fewer of them at a time) and those of 32000 the same 194.
template <bool kPast, typename T, typename Gradient>
__device__ __forceinline__ void WriteVec(T *dx, const Vec &x, int q, int C, const Gradient &gradient) {
  constexpr int kN = Lanes<T>::kN;
  float g[kN];
#pragma unroll
  for (int e = 0; e < kN; ++e) g[e] = gradient(ElementOf<T>(x, e));
  if ((q + 1) * kN <= C) {
    StoreVec<kPast>(dx + (size_t)q * kN, PackOf<T>(g));
  } else {  // the incomplete last vector, which was read to end with the row
    const int base = VecBase<T>(q, C);
#pragma unroll
    for (int e = 0; e < kN; ++e)
      if (base + e >= q * kN && base + e < C) FromFloat(g[e], &dx[base + e]);
  }
}
template <typename T>
__device__ __forceinline__ void StoreStaged(const T *stage, T *dx, int q, int C) {
  constexpr int kN = Lanes<T>::kN;
  if ((q + 1) * kN <= C) {
    StoreVec<false>(dx + (size_t)q * kN, *reinterpret_cast<const Vec *>(stage + q * kN));
  } else {
    for (int i = q * kN; i < C; ++i) dx[i] = stage[i];
  }
}
template <bool kPast, typename T>
__device__ __forceinline__ void StoreZeros(T *dx, int q, int C) {
  WriteVec<kPast>(dx, Vec{{0, 0, 0, 0}}, q, C, [](float) { return 0.0f; });
}
// short rows that a workgroup has in its backward pass: what they are staged in takes 2 KB of LDS each
template <int U>
constexpr int StagedVecs() { return U <= 8 ? U * 16 : 0; }

__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float Log2(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float Exp(float x) { return Exp2(x * 1.44269504088896341f); }  // |x| 2^-23 off, relative

// Reductions over a wavefront: within rows of 16 lanes by DPP moves, across the four rows through scalar registers.  Every
// lane gets the result.
template <int kCtrl>
__device__ __forceinline__ float DppMove(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), kCtrl, 0xf, 0xf, false));
}
__device__ __forceinline__ float ReadLane(float v, int lane) {
  return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
__device__ __forceinline__ float WaveMaxF(float v) {
  v = fmaxf(v, DppMove<0xb1>(v));   // neighbours
  v = fmaxf(v, DppMove<0x4e>(v));   // pairs
  v = fmaxf(v, DppMove<0x141>(v));  // quads, mirrored within eight lanes
  v = fmaxf(v, DppMove<0x140>(v));  // eights, mirrored within sixteen
  return fmaxf(fmaxf(ReadLane(v, 0), ReadLane(v, 16)), fmaxf(ReadLane(v, 32), ReadLane(v, 48)));
}
__device__ __forceinline__ float WaveSumF(float v) {
  v += DppMove<0xb1>(v);
  v += DppMove<0x4e>(v);
  v += DppMove<0x141>(v);
  v += DppMove<0x140>(v);
  return (ReadLane(v, 0) + ReadLane(v, 16)) + (ReadLane(v, 32) + ReadLane(v, 48));
}
// The same over the L lanes of a group: 16 lanes of one row of lanes, or the wavefront.
template <int L>
__device__ __forceinline__ float GroupMax(float v) {
  if (L == kWave) return WaveMaxF(v);
  v = fmaxf(v, DppMove<0xb1>(v));
  v = fmaxf(v, DppMove<0x4e>(v));
  v = fmaxf(v, DppMove<0x141>(v));
  return fmaxf(v, DppMove<0x140>(v));
}
template <int L>
__device__ __forceinline__ float GroupSum(float v) {
  if (L == kWave) return WaveSumF(v);
  v += DppMove<0xb1>(v);
  v += DppMove<0x4e>(v);
  v += DppMove<0x141>(v);
  return v + DppMove<0x140>(v);
}
// the lanes of this lane's group among those where `predicate` holds, the group's first lane in bit 0
template <int L>
__device__ __forceinline__ unsigned long long GroupBallot(bool predicate) {
  const unsigned long long all = __ballot(predicate);
  if (L == kWave) return all;
  const int shift = (int)(threadIdx.x & (kWave - 1) & ~(unsigned)(L - 1));
  return (all >> shift) & ((1ull << (L & 63)) - 1);
}
__device__ __forceinline__ unsigned BelowLane(unsigned long long lanes) {  // how many of `lanes` are below this one
  return __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0u));
}

// log p of an element with logit x, in the natural logarithm's scale throughout: (x - m) c could overflow where this does not
__device__ __forceinline__ float LogProb(float x, float m, float ls, float inv_tau) {
  return ls == Real<float>::NegInf() ? Real<float>::NegInf() : (x - m) * inv_tau - kLn2 * ls;
}

// What is known of a stretch of logits: the largest (0 where that is -inf), s and t = sum of d 2^d for the entropy.
struct Sums {
  float m, s, t;
};
// the sums of two stretches as one
__device__ __forceinline__ Sums Join(const Sums &a, const Sums &b, float c) {
  if (a.s == 0.0f) return b;
  if (b.s == 0.0f) return a;
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = (a.m - r.m) * c, db = (b.m - r.m) * c, ea = Exp2(da), eb = Exp2(db);
  r.s = a.s * ea + b.s * eb;
  r.t = (a.t + fmaxf(da, kNothing) * a.s) * ea + (b.t + fmaxf(db, kNothing) * b.s) * eb;
  return r;
}

// the sums of the up to 64 stretches that a wavefront's lanes have (s = 0: none) as one, in every lane
__device__ __forceinline__ Sums JoinLanes(const Sums &a, float c) {
  Sums r{WaveMaxF(a.s == 0.0f ? Real<float>::NegInf() : a.m), 0.0f, 0.0f};
  if (r.m == Real<float>::NegInf()) r.m = 0.0f;
  const float d = a.s == 0.0f ? 0.0f : (a.m - r.m) * c, e = Exp2(d);
  r.s = WaveSumF(a.s * e);
  r.t = WaveSumF((a.t + fmaxf(d, kNothing) * a.s) * e);
  return r;
}

// m, s and t (kEntropy) of what a group of lanes holds, from its largest logit.  The inner loop is one fused multiply-add,
// one exponential and one addition an element: d = x c - M with M = m c rounded, which leaves every exponent off by the same
// M - m c, exactly known and below a half, and that is taken out of the sums at the end.  Rows whose m c is beyond kFar (a
// type's lowest value everywhere, a temperature of nearly 0) take the difference first.  Each row chooses for itself: where the
// rows of a wavefront differ, both forms are computed, so that no row's bits depend on what lies next to it.  (Rows that do
// not count come with -inf as their largest logit: whatever they hold, they never ask for the second form.)
constexpr float kFar = 1.0e6f;
template <bool kEntropy, typename T, int U, int W, int L>
__device__ __forceinline__ Sums SumsOf(RowPart<T, U, W, L> &part, float high, float c) {
  constexpr int kN = Lanes<T>::kN;
  Sums r{high == Real<float>::NegInf() ? 0.0f : high, 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < U; ++u) part.Packed(u);  // (here, and not in the two branches: each would get registers of its own)
  const bool far = !(fabsf(r.m * c) <= kFar);
  if (__ballot(!far) != 0) {
    const float shift = -(r.m * c);
    float s[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float d = __builtin_fmaf(ElementOf<T>(part.v[u], e), c, shift), p = Exp2(d);
        s[e & 3] += p;
        if (kEntropy) t[e & 3] += fmaxf(d, kNothing) * p;
      }
    const float off = __builtin_fmaf(r.m, c, shift), scale = Exp2(-off);
    r.s = GroupSum<L>((s[0] + s[1]) + (s[2] + s[3]));
    if (kEntropy) r.t = (GroupSum<L>((t[0] + t[1]) + (t[2] + t[3])) - off * r.s) * scale;
    r.s *= scale;
  }
  if (__ballot(far) != 0) {
    float s[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[i] = Anew(part.v[u].w[i]);
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float d = (ElementOf<T>(v, e) - r.m) * c, p = Exp2(d);
        s[e & 3] += p;
        if (kEntropy) t[e & 3] += fmaxf(d, kNothing) * p;
      }
    }
    const float s_far = GroupSum<L>((s[0] + s[1]) + (s[2] + s[3]));
    const float t_far = kEntropy ? GroupSum<L>((t[0] + t[1]) + (t[2] + t[3])) : 0.0f;
    if (far) {
      r.s = s_far;
      r.t = t_far;
    }
  }
  return r;
}

// -inf in the place of a vector's elements that are marked
template <typename T>
__device__ __forceinline__ void DropMarked(Vec *v, unsigned marked) {
  auto all_if = [&](int bit) { return (unsigned)((int)(marked << (31 - bit)) >> 31); };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned gone = sizeof(T) == 4 ? all_if(i) : (all_if(2 * i) & 0xffffu) | (all_if(2 * i + 1) & 0xffff0000u);
    v->w[i] = (gone & Lanes<T>::kNegInf) | (~gone & v->w[i]);
  }
}
// the marks of the elements of a vector that is read from column `base` on; bit 0 of `bits` is column `begin` (`base` is
// below it only in a row's last vector, which is read to end with the row); one word behind the last is readable
template <typename T>
__device__ __forceinline__ unsigned MarksOf(const unsigned *bits, int base, int begin) {
  constexpr int kN = Lanes<T>::kN;
  const int at = base - begin, from = max(at, 0), shift = from & 31;
  unsigned marked = bits[from >> 5] >> shift;
  if (shift + kN > 32) marked |= bits[(from >> 5) + 1] << (32 - shift);  // (only in a row's last vector)
  return (marked << (from - at)) & ((1u << kN) - 1);
}

// m, s and t (kEntropy) of vectors [first, end) of a row that W wavefronts read, each on its own and without keeping them:
// a lane runs along its vectors with a largest logit of its own, four vectors at a time, while the next four are on their
// way.  kMarked: without the elements marked in `bits` (of columns from first on).
template <typename T, int W, bool kEntropy, bool kMarked>
__device__ __forceinline__ Sums StreamSums(const T *x, int C, int first, int end, int wave, int lane, float c,
                                           const unsigned *bits) {
  constexpr int kN = Lanes<T>::kN, kStep = 4;
  const int whole = C / kN;
  const int rounds = (end - first + W * kWave - 1) / (W * kWave);
  Sums r{Real<float>::NegInf(), 0.0f, 0.0f};
  bool far = false;
  float reference = 0.0f;  // M: what the exponents are taken from, m c rounded
  float s[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
  Vec next[kStep];
  auto fetch = [&](int round) {
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      const int q = first + ((round + i) * W + wave) * kWave + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) next[i].w[j] = Lanes<T>::kNegInf;
      if (q < end) next[i] = LoadRowVec<T>(x, q, C, q >= whole);
    }
  };
  fetch(0);
  for (int round = 0; round < rounds; round += kStep) {
    Vec v[kStep];
#pragma unroll
    for (int i = 0; i < kStep; ++i) v[i] = next[i];
    if (round + kStep < rounds) fetch(round + kStep);
    if (kMarked) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const int q = first + ((round + i) * W + wave) * kWave + lane;
        const unsigned marked = q < end ? MarksOf<T>(bits, VecBase<T>(q, C), first * kN) : 0u;
        if (__ballot(marked != 0) != 0) DropMarked<T>(&v[i], marked);
      }
    }
    float high[2] = {r.m, Real<float>::NegInf()};
#pragma unroll
    for (int i = 0; i < kStep; ++i)
#pragma unroll
      for (int e = 0; e < kN; e += 2)
        high[e / 2 & 1] = fmaxf(fmaxf(high[e / 2 & 1], ElementOf<T>(v[i], e)), ElementOf<T>(v[i], e + 1));
    r.m = fmaxf(high[0], high[1]);
    const float before = reference;
    reference = r.m == Real<float>::NegInf() ? 0.0f : r.m * c;
    far |= !(fabsf(reference) <= kFar);
    const float down = fminf(before - reference, 0.0f), scale = Exp2(down);  // (the first reference may be below 0: s is 0 then)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kEntropy) t[i] = (t[i] + fmaxf(down, kNothing) * s[i]) * scale;
      s[i] *= scale;
    }
#pragma unroll
    for (int i = 0; i < kStep; ++i)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float d = __builtin_fmaf(ElementOf<T>(v[i], e), c, -reference), p = Exp2(d);
        s[e & 3] += p;
        if (kEntropy) t[e & 3] += fmaxf(d, kNothing) * p;
      }
  }
  if (__ballot(far) != 0) {  // differences first, as in SumsOf
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = t[i] = 0.0f;
    r.m = WaveMaxF(r.m);
    for (int round = 0; round < rounds; ++round) {
      const int q = first + (round * W + wave) * kWave + lane;
      if (q >= end) continue;
      Vec v = LoadRowVec<T>(x, q, C, q >= whole);
      if (kMarked) DropMarked<T>(&v, MarksOf<T>(bits, VecBase<T>(q, C), first * kN));
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float d = (ElementOf<T>(v, e) - r.m) * c, p = Exp2(d);
        s[e & 3] += p;
        if (kEntropy) t[e & 3] += fmaxf(d, kNothing) * p;
      }
    }
    r.s = (s[0] + s[1]) + (s[2] + s[3]);
    r.t = (t[0] + t[1]) + (t[2] + t[3]);
  } else {
    if (r.m == Real<float>::NegInf()) r.m = 0.0f;
    const float off = __builtin_fmaf(r.m, c, -reference), scale = Exp2(-off);
    r.s = (s[0] + s[1]) + (s[2] + s[3]);
    r.t = (((t[0] + t[1]) + (t[2] + t[3])) - off * r.s) * scale;
    r.s *= scale;
  }
  return JoinLanes(r, c);
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
__device__ __forceinline__ float LogitOf(unsigned long long key) {
  const unsigned order = (unsigned)(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? (order == 0xffffffffu ? 0x7fc00000u : order & 0x7fffffffu) : ~order);
}

inline bool RowsOk(long long rows, long long row_stride, int C, float temperature, int dtype) {
  if (rows < 0 || C < 1 || row_stride < 0) return false;
  if (!(temperature > 0.0f) || temperature - temperature != 0.0f) return false;
  if (!(kLog2E / (double)temperature <= 3.40282346e38)) return false;  // (c of the kernels would be infinite)
  return dtype == K2AMD_F32 || dtype == K2AMD_F16 || dtype == K2AMD_BF16;
}
inline bool RowsServed(long long rows, int C) { return rows < (1ll << 31) && C <= kMaxColumns; }

// How rows of more than 256 vectors are cut into parts, each for a workgroup of four wavefronts.
struct LongShape {
  int vecs;   // of a part
  int parts;
};
// Rows that are read along (no alternatives): whole up to kPartColumns (a lane then adds up 256 terms, in four sums; the
// marks of a part take 8 KB of LDS), unless that leaves compute units without work.
constexpr int kPartColumns = 1 << 16;
inline LongShape StreamShapeOf(long long rows, int vecs, int vec) {
  const int max_vecs = kPartColumns / vec;
  long long parts = (vecs + max_vecs - 1) / max_vecs;
  const long long wanted = (1024 + rows - 1) / rows, finest = (vecs + 1023) / 1024;
  if (parts < wanted) parts = wanted < finest ? wanted : finest;
  if (parts > 64) parts = 64;
  const int each = (int)(((vecs + parts - 1) / parts + 255) / 256 * 256);
  return LongShape{each, (vecs + each - 1) / each};
}
// Rows that are held: 16 vectors a lane hold 4096 vectors; parts of 1024 where that would leave compute units without work.
inline LongShape HeldShapeOf(long long rows, int vecs) {
  const int whole = (vecs + 4095) / 4096, fine = (vecs + 1023) / 1024;
  return fine == 1 || (rows * whole < 256 && fine <= 64) ? LongShape{1024, fine} : LongShape{4096, whole};
}
inline bool Misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }  // of what is accessed by 16 bytes

// A launch holds fewer than 2^32 work-items in x: calls with more rows are several launches.
constexpr long long kRowsPerLaunch = 1ll << 20;

}  // namespace
}  // namespace k2amd

#endif  // K2_AMD_CSRC_TOKEN_ROWS_H_
