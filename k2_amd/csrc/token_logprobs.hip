// Log-probs of given tokens, entropy and the most likely alternatives of rows of logits, and the gradient of all three
// (k2amd_token_logprobs_forward / _backward).
//
//   log p_i = (x_i - m) / tau - log s,   H = -sum_i p_i log p_i,   alternatives: the k largest logits
//   dx_i = 1/tau [ sum_{j: c_j = i} g_j - p_i sum_j g_j - gH p_i (log p_i + H) ]
//
// with c_j the given tokens and the alternatives together and g_j what reaches their log-probs.
//
// Measured on an MI355X, kernel times after some hundred passes: 80000 x 500 float32, four fifths of the rows, 8 alternatives,
// 43 us (20 us to read them; the arithmetic, half of it the selection, keeps the vector units busy for 23); 4096 x 32000 with
// 64 alternatives 98 us in bfloat16 (41 to read; the selection is two thirds of the instructions) and in float32, whose rows
// are two parts, 143 and 20 for the join; 6553 of 8191 x 32000 with entropy 83 us in bfloat16 (5.0 TB/s) and 146 in float32
// (5.8), and their gradient 156 (419 MB read, 524 MB written: 6.0 TB/s) and 331 (5.7); one row of 131072 with 20 alternatives
// 8.2 us in 16 parts and 7.2 us for their join in bfloat16, 7.0 and 18.7 in float32, in 32 parts.
#include "token_rows.h"

namespace k2amd {
namespace {

// ---- alternatives ---------------------------------------------------------------------------------
//
// The k largest of the elements that wavefronts hold in registers, without sorting them.  A lane's elements form up to four
// groups; a bisection over the groups' maxima finds a logit that at least k groups reach, by counting ballots (a comparison
// and scalar work for each step), so at least k elements reach it, and hardly more in data that is not made of ties: the
// groups with two of the k largest are few.  These elements go to LDS as whole numbers that carry value and index, and each
// one's place is the number of larger ones.  Where more than kListed reach the threshold (rows of equal logits, a mask
// that leaves a handful of tokens in front of thousands of -inf) or a NaN is among them, the wavefront lists its k
// largest class by class instead: the largest value, all its occurrences in the order of the index, the next value.
constexpr int kListed = 128;  // elements that a wavefront lists

template <int G>
__device__ __forceinline__ int GroupsReaching(const float (&group)[G], float v) {
  int n = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) n += __popcll(__ballot(group[g] >= v));
  return n;
}

// A value that at least k of the groups' maxima reach (-inf if no larger one was found), the largest of them being `high`;
// `from`: one that is known to be reached by k.
template <int G>
__device__ __forceinline__ float Threshold(const float (&group)[G], float high, int k, float from) {
  if (GroupsReaching(group, high) >= k) return high;
  float lo = from, hi = high;
  if (lo == Real<float>::NegInf()) {
    // steps of 8, 64, 4096: most rows' k-th largest lies within 8 of the largest
    lo = high - 8.0f;
    if (GroupsReaching(group, lo) < k) {
      hi = lo;
      lo = high - 64.0f;
      if (GroupsReaching(group, lo) < k) {
        hi = lo;
        lo = high - 4096.0f;
        if (!(GroupsReaching(group, lo) >= k)) return Real<float>::NegInf();
      }
    }
  }
  for (int step = 0; step < 24; ++step) {
    const float mid = 0.5f * (lo + hi);
    const int n = GroupsReaching(group, mid);
    if (n >= k) {
      lo = mid;
      if (n <= k + (k >> 1) + 2) break;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// Lists the wavefront's elements that reach `threshold`; returns how many there are (only kListed of them are listed).
template <typename T, int U, int W>
__device__ __forceinline__ int ListReaching(RowPart<T, U, W> &part, int C, int first, int wave, int lane, float threshold,
                                            unsigned long long *list) {
  constexpr int kN = Lanes<T>::kN;
  int count = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Vec &v = part.Packed(u);
    float x[kN], high = Real<float>::NegInf();
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      x[e] = ElementOf<T>(v, e);
      high = fmaxf(high, x[e]);
    }
    if (__ballot(high >= threshold) == 0) continue;
    const int q = part.VectorAnew(u, first, wave, lane), base = VecBase<T>(q, C);
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      if (__ballot(x[e] >= threshold) == 0) continue;
      const int index = base + e;
      const bool mine = x[e] >= threshold && index >= q * kN && index < C;  // (the -inf that pads a row is no element of it)
      const unsigned long long lanes = __ballot(mine);
      const int at = count + (int)BelowLane(lanes);
      if (mine && at < kListed) list[at] = KeyOf(x[e], (unsigned)index);
      count += __popcll(lanes);
    }
  }
  return count;
}

// Lists the wavefront's k largest elements (k <= kMaxTop) class by class of equal ones; returns how many.
template <typename T, int U, int W>
__device__ __forceinline__ int ListByClasses(RowPart<T, U, W> &part, int C, int first, int wave, int lane, int k,
                                             unsigned long long *list) {
  constexpr int kN = Lanes<T>::kN;
  int count = 0;
  float last = 0.0f;
  for (int round = 0; count < k; ++round) {
    // the first class: the NaNs; the second: the largest; then the largest below the last
    float high = Real<float>::NegInf();
    if (round > 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Vec &v = part.Packed(u);
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float x = ElementOf<T>(v, e);
          if (round == 1 || x < last) high = fmaxf(high, x);
        }
      }
      high = WaveMaxF(high);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (count >= k) continue;
      const int q = part.VectorAnew(u, first, wave, lane), base = VecBase<T>(q, C);
      const Vec &v = part.Packed(u);
      unsigned bits = 0;
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float x = ElementOf<T>(v, e);
        if ((round == 0 ? x != x : x == high) && base + e >= q * kN && base + e < C) bits |= 1u << e;
      }
      if (__ballot(bits != 0) == 0) continue;
      unsigned long long total = 0;
      int at = count, here = 0;
#pragma unroll
      for (int e = 0; e < kN; ++e) {  // elements in front of this lane's, in the order of the index
        const unsigned long long lanes = __ballot((bits >> e & 1u) != 0);
        at += (int)BelowLane(lanes);
        total += __popcll(lanes);
      }
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (bits >> e & 1u) {
          if (at + here < k) list[at + here] = KeyOf(ElementOf<T>(v, e), (unsigned)(base + e));
          ++here;
        }
      count = min(k, count + (int)total);
    }
    if (round > 0 && high == Real<float>::NegInf()) break;  // nothing is below
    last = high;
  }
  return count;
}

// ---- forward ----------------------------------------------------------------------------------------

struct ForwardArgs {
  long long row_stride;
  const int64_t *tokens;
  const uint8_t *mask;
  float *logprobs, *entropy, *top_logprobs;
  int64_t *top_tokens;
  float *stats;
  int C, n, k;
  float c, inv_tau;
  // rows in several parts: [rows][parts] sums and [rows][parts][k] keys, the largest first, 0 past the last
  int parts;
  float4 *part_sums;
  unsigned long long *part_keys;
};

__device__ __forceinline__ void WriteSkippedRow(const ForwardArgs &a, size_t row, int i) {
  if (i < a.n) a.logprobs[row * a.n + i] = 0.0f;
  if (i < a.k) {
    a.top_logprobs[row * a.k + i] = Real<float>::NegInf();
    a.top_tokens[row * a.k + i] = -1;
  }
  if (i == 0 && a.entropy != nullptr) a.entropy[row] = 0.0f;
  if (i == 0 && a.stats != nullptr) a.stats[2 * row] = a.stats[2 * row + 1] = 0.0f;
}

// What a row's sums say, by the first 64 work-items; x_token: the logit of work-item i's token.
__device__ __forceinline__ void WriteRow(const ForwardArgs &a, size_t row, int i, const Sums &sums, int64_t token,
                                         float x_token) {
  const float ls = Log2(sums.s);
  if (i < a.n) {
    float lp = 0.0f;
    if (token >= a.C) lp = __uint_as_float(0x7fc00000u);
    else if (token >= 0) lp = LogProb(x_token, sums.m, ls, a.inv_tau);
    a.logprobs[row * a.n + i] = lp;
  }
  if (i == 0 && a.entropy != nullptr) a.entropy[row] = sums.s == 0.0f ? 0.0f : kLn2 * (ls - sums.t / sums.s);
  if (i == 0 && a.stats != nullptr) {
    a.stats[2 * row] = sums.m;
    a.stats[2 * row + 1] = sums.s;
  }
}

// Short rows: 16 lanes each, four rows a wavefront (a wavefront a row took the same 47 us as this at first, and the selection
// four times the instructions a row).  What a row depends on (mask, tokens) is asked for first and together, then
// the row.  Every vector of a row is a group of the threshold's; each row has a threshold of its own, so that the counting is
// done in the 16 lanes of the row.  A lane collects which of its elements reach it in bits and then lists them one after the
// other, reading each again (it is in the nearest cache): the list's code is run as often as the busiest lane has elements in
// it, not once for each place of an element in a lane.
constexpr int kShort = 16, kShortRows = 16;
constexpr int kThreads = kShort * kShortRows;

__device__ __forceinline__ int RowSum(int n) {  // (the moves of GroupSum)
  n += __builtin_amdgcn_update_dpp(0, n, 0xb1, 0xf, 0xf, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x4e, 0xf, 0xf, false);
  n += __builtin_amdgcn_update_dpp(0, n, 0x141, 0xf, 0xf, false);
  return n + __builtin_amdgcn_update_dpp(0, n, 0x140, 0xf, 0xf, false);
}

// as Threshold above, for each of the wavefront's rows; reaching(v): how many of a row's groups (or elements) reach v
template <typename Reaching>
__device__ __forceinline__ float RowThreshold(float high, int k, const Reaching &reaching) {
  float lo = high, hi = high;
  bool found = reaching(high) >= k, done = found;
#pragma unroll 1
  for (int i = 0; i < 3; ++i) {
    if (__ballot(!found) == 0) continue;
    const float v = high - (i == 0 ? 8.0f : i == 1 ? 64.0f : 4096.0f);
    const bool reached = reaching(v) >= k;
    if (!found) (reached ? lo : hi) = v;
    found |= reached;
  }
  if (!found) lo = Real<float>::NegInf();
  done |= !found;
#pragma unroll 1
  for (int step = 0; step < 24 && __ballot(!done) != 0; ++step) {
    const float mid = 0.5f * (lo + hi);
    const int n = reaching(mid);
    if (!done) (n >= k ? lo : hi) = mid;
    done |= n >= k && n <= k + (k >> 1) + 2;
  }
  return lo;
}

template <typename T, int U, bool kEntropy>
__global__ __launch_bounds__(kThreads) void TokenShortKernel(const T *__restrict__ logits, long long row0, long long rows,
                                                             ForwardArgs a) {
  constexpr int kN = Lanes<T>::kN;
  __shared__ unsigned long long lists[kShortRows][kListed];
  __shared__ int listed[kShortRows];
  const int lane = threadIdx.x % kShort, in_block = threadIdx.x / kShort;
  const long long in_launch = (long long)blockIdx.x * kShortRows + in_block;
  if ((in_launch & ~3ll) >= rows) return;  // (the wavefront's first row)
  const bool there = in_launch < rows;
  const size_t row = row0 + (there ? in_launch : rows - 1);  // (lanes without a row follow along and write nothing)
  const uint8_t masked = a.mask == nullptr ? 1 : a.mask[row];
  int64_t token = lane < a.n ? a.tokens[row * a.n + lane] : -1;
  const bool live = there && masked != 0;
  const T *x = logits + row * a.row_stride;
  RowPart<T, U, 1, kShort> part;
  // (all four rows or none: a load that some lanes skip is a branch for each vector)
  part.Load(x, __ballot(live) != 0 ? a.C : 0, 0, 0, lane);
  float x_token = live && token >= 0 && token < a.C ? ToFloat(x[token]) : 0.0f;
  float group[U], high = Real<float>::NegInf();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Vec &v = part.Packed(u);
    group[u] = Real<float>::NegInf();
#pragma unroll
    for (int e = 0; e < kN; e += 2) group[u] = fmaxf(fmaxf(group[u], ElementOf<T>(v, e)), ElementOf<T>(v, e + 1));
    high = fmaxf(high, group[u]);
  }
  high = GroupMax<kShort>(high);
  const Sums sums = SumsOf<kEntropy>(part, live ? high : Real<float>::NegInf(), a.c);
  if (there && !live) {
    for (int i = lane; i < max(max(a.n, a.k), 1); i += kShort) WriteSkippedRow(a, row, i);
  } else if (there) {
    WriteRow(a, row, lane, sums, token, x_token);
    for (int i = lane + kShort; i < a.n; i += kShort) {
      token = a.tokens[row * a.n + i];
      x_token = token >= 0 && token < a.C ? ToFloat(x[token]) : 0.0f;
      WriteRow(a, row, i, sums, token, x_token);
    }
  }
  if (a.k == 0) return;

  unsigned long long *list = lists[in_block];
  if (lane == 0) listed[in_block] = 0;
  const bool odd = sums.s != sums.s;  // a NaN or +inf among them
  const float from = live && !odd ? high : Real<float>::NegInf();
  const int wanted = live && !odd ? a.k : 0;
  float threshold;
  if (2 * a.k <= VecsOf<T>(a.C)) {
    threshold = RowThreshold(from, wanted, [&](float v) {
      int n = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) n += group[u] >= v ? 1 : 0;
      return RowSum(n);
    });
  } else {
    // so many that the k-th largest of the groups' maxima says little: the elements themselves are counted (64000 x 500
    // bfloat16 with 64 alternatives by groups listed more than there is room for in nearly every row, and took 1019 us)
    threshold = RowThreshold(from, wanted, [&](float v) {
      int n = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Vec x;  // (a copy: the branch must not get vectors of its own)
#pragma unroll
        for (int i = 0; i < 4; ++i) x.w[i] = Anew(part.v[u].w[i]);
#pragma unroll
        for (int e = 0; e < kN; ++e) n += ElementOf<T>(x, e) >= v ? 1 : 0;
      }
      return RowSum(n);
    });
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  constexpr int kPerWord = 32 / kN;  // vectors whose elements share a word of bits
#pragma unroll
  for (int word = 0; word < (U + kPerWord - 1) / kPerWord; ++word) {
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < kPerWord && word * kPerWord + i < U; ++i) {
      const int u = word * kPerWord + i;
      if (__ballot(group[u] >= threshold) == 0) continue;
      const Vec &v = part.Packed(u);
      unsigned of_vector = 0;
#pragma unroll
      for (int e = 0; e < kN; ++e) of_vector |= ElementOf<T>(v, e) >= threshold ? 1u << e : 0u;
      if ((u + 1) * kShort * kN > a.C) {  // the round with the row's end: the -inf that pads a row is no element of it
        const int q = part.VectorAnew(u, 0, 0, lane), base = VecBase<T>(q, a.C);
        of_vector &= q < VecsOf<T>(a.C) ? ((1u << kN) - 1) << min(kN, q * kN - base) : 0u;
        if (base + kN > a.C) of_vector &= (1u << (a.C - base)) - 1;
      }
      bits |= of_vector << (i * kN);
    }
    if (!live || odd) bits = 0;
    int at = bits != 0 ? atomicAdd(&listed[in_block], __popc(bits)) : 0;
    while (__ballot(bits != 0) != 0) {
      if (bits != 0) {
        const int bit = __ffs((int)bits) - 1, q = part.Vector(word * kPerWord + bit / kN, 0, 0, lane);
        const int index = VecBase<T>(q, a.C) + bit % kN;
        if (at < kListed) list[at] = KeyOf(ToFloat(x[index]), (unsigned)index);
        ++at;
        bits &= bits - 1;
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // rows that list too much, or NaNs: by the whole wavefront, one after the other
  const unsigned long long again = __ballot(live && (odd || listed[in_block] > kListed));
  if (again != 0) {
    for (int g = 0; g < kWave / kShort; ++g) {
      if ((again >> (g * kShort) & 1) == 0) continue;
      const int other = in_block / 4 * 4 + g, wave_lane = threadIdx.x & (kWave - 1);
      RowPart<T, (U + 3) / 4, 1> wide;
      wide.Load(logits + (row0 + (long long)blockIdx.x * kShortRows + other) * a.row_stride, a.C, 0, 0, wave_lane);
      const int count = ListByClasses<T, (U + 3) / 4, 1>(wide, a.C, 0, 0, wave_lane, a.k, lists[other]);
      if (wave_lane == 0) listed[other] = count;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (!live) return;
  const int count = listed[in_block];
  const float ls = Log2(sums.s);
  for (int i = lane; i < count; i += kShort) {
    const unsigned long long key = list[i];
    int place = 0;
    for (int j = 0; j < count; ++j) place += list[j] > key ? 1 : 0;
    if (place < a.k) {
      a.top_tokens[row * a.k + place] = IndexOf(key);
      a.top_logprobs[row * a.k + place] = LogProb(LogitOf(key), sums.m, ls, a.inv_tau);
    }
  }
  for (int i = count + lane; i < a.k; i += kShort) {  // rows shorter than the list
    a.top_tokens[row * a.k + i] = -1;
    a.top_logprobs[row * a.k + i] = Real<float>::NegInf();
  }
}

// Long rows with alternatives: W wavefronts hold a row or a part of it.  kEntropy: whether t is summed up.
template <typename T, int U, int W, bool kEntropy>
__global__ __launch_bounds__(W *kWave) void TokenHeldKernel(const T *__restrict__ logits, long long row0, ForwardArgs a) {
  constexpr int kN = Lanes<T>::kN;
  __shared__ unsigned long long lists[W][kListed];
  __shared__ float4 wave_sums[W];      // m, s, t, the threshold that k of a wavefront's groups reach
  __shared__ float wave_low[W];        // and the one that its share of k reach
  __shared__ int listed[W];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const size_t row = row0 + blockIdx.x;
  const int first = (int)blockIdx.y * (U * W * kWave);
  if (a.mask != nullptr && a.mask[row] == 0) {
    if (wave == 0 && blockIdx.y == 0) WriteSkippedRow(a, row, lane);
    return;
  }
  const T *x = logits + row * a.row_stride;
  // (the tokens in front of the row, the logits that they point to behind it: results of loads come in order)
  const int64_t token = wave == 0 && a.parts == 1 && lane < a.n ? a.tokens[row * a.n + lane] : -1;
  RowPart<T, U, W> part;
  part.Load(x, a.C, first, wave, lane);
  const float x_token = token >= 0 && token < a.C ? ToFloat(x[token]) : 0.0f;

  // the wavefront's sums
  constexpr int kGroups = U < 4 ? U : 4;
  float group[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) group[g] = Real<float>::NegInf();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Vec &v = part.Packed(u);
#pragma unroll
    for (int e = 0; e < kN; e += 2)
      group[u % kGroups] = fmaxf(fmaxf(group[u % kGroups], ElementOf<T>(v, e)), ElementOf<T>(v, e + 1));
  }
  float high = group[0];
#pragma unroll
  for (int g = 1; g < kGroups; ++g) high = fmaxf(high, group[g]);
  high = WaveMaxF(high);
  Sums sums = SumsOf<kEntropy>(part, high, a.c);

  const bool odd = sums.s != sums.s;  // a NaN or +inf among them
  float threshold = Real<float>::NegInf(), low = threshold;
  if (!odd) {
    threshold = Threshold<kGroups>(group, high, a.k, threshold);
    low = Threshold<kGroups>(group, high, (a.k + W - 1) / W, threshold);
  }
  if (lane == 0) {
    wave_sums[wave] = make_float4(sums.m, sums.s, sums.t, threshold);
    wave_low[wave] = low;
  }
  __syncthreads();
  // k elements of the part reach every wavefront's own threshold, and the lowest of those that k / W reach in each
  float lowest = wave_low[0];
  threshold = Real<float>::NegInf();
  for (int w = 0; w < W; ++w) {
    threshold = fmaxf(threshold, wave_sums[w].w);
    lowest = fminf(lowest, wave_low[w]);
  }
  threshold = fmaxf(threshold, lowest);
  sums = Sums{wave_sums[0].x, wave_sums[0].y, wave_sums[0].z};
  for (int w = 1; w < W; ++w) sums = Join(sums, Sums{wave_sums[w].x, wave_sums[w].y, wave_sums[w].z}, a.c);
  if (wave == 0) {
    if (a.parts == 1) WriteRow(a, row, lane, sums, token, x_token);
    else if (lane == 0) a.part_sums[row * a.parts + blockIdx.y] = make_float4(sums.m, sums.s, sums.t, 0.0f);
  }
  unsigned long long *own = lists[wave];
  int count = odd ? kListed + 1 : ListReaching<T, U, W>(part, a.C, first, wave, lane, threshold, own);
  if (count > kListed)
    count = ListByClasses<T, U, W>(part, a.C, first, wave, lane, a.k, own);
  if (lane == 0) listed[wave] = count;
  __syncthreads();
  // each listed element's place
  const float ls = Log2(sums.s);
  int all = 0;
  for (int w = 0; w < W; ++w) all += listed[w];
  for (int i = lane; i < count; i += kWave) {
    const unsigned long long key = own[i];
    int place = 0;
    for (int w = 0; w < W; ++w) {
      const int n = listed[w];
      for (int j = 0; j < n; ++j) place += lists[w][j] > key ? 1 : 0;
    }
    if (place < a.k) {
      if (a.parts == 1) {
        a.top_tokens[row * a.k + place] = IndexOf(key);
        a.top_logprobs[row * a.k + place] = LogProb(LogitOf(key), sums.m, ls, a.inv_tau);
      } else {
        a.part_keys[(row * a.parts + blockIdx.y) * a.k + place] = key;
      }
    }
  }
  if (wave == 0 && lane < a.k && lane >= all) {  // rows shorter than the list
    if (a.parts == 1) {
      a.top_tokens[row * a.k + lane] = -1;
      a.top_logprobs[row * a.k + lane] = Real<float>::NegInf();
    } else {
      a.part_keys[(row * a.parts + blockIdx.y) * a.k + lane] = 0;
    }
  }
}

// Long rows without alternatives: four wavefronts read along a row or a part of it.
constexpr int kStreamWaves = 4;
template <typename T, bool kEntropy>
__global__ __launch_bounds__(kStreamWaves *kWave) void TokenStreamKernel(const T *__restrict__ logits, long long row0,
                                                                        int part_vecs, ForwardArgs a) {
  __shared__ float4 wave_sums[kStreamWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const size_t row = row0 + blockIdx.x;
  const int first = (int)blockIdx.y * part_vecs, end = min(VecsOf<T>(a.C), first + part_vecs);
  if (a.mask != nullptr && a.mask[row] == 0) {
    if (wave == 0 && blockIdx.y == 0) WriteSkippedRow(a, row, lane);
    return;
  }
  const T *x = logits + row * a.row_stride;
  Sums sums = StreamSums<T, kStreamWaves, kEntropy, false>(x, a.C, first, end, wave, lane, a.c, nullptr);
  if (lane == 0) wave_sums[wave] = make_float4(sums.m, sums.s, sums.t, 0.0f);
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < kStreamWaves; ++w) sums = Join(sums, Sums{wave_sums[w].x, wave_sums[w].y, wave_sums[w].z}, a.c);
  if (a.parts > 1) {
    if (lane == 0) a.part_sums[row * a.parts + blockIdx.y] = make_float4(sums.m, sums.s, sums.t, 0.0f);
    return;
  }
  const int64_t token = lane < a.n ? a.tokens[row * a.n + lane] : -1;
  WriteRow(a, row, lane, sums, token, token >= 0 && token < a.C ? ToFloat(x[token]) : 0.0f);
}

// Joins the parts of a row: a workgroup a row.  The keys of a part are in order, so a key's place among all is its place in
// its own part and, in every other part, the number of larger ones, by bisection.  A work-item searches four parts side by
// side for a key: steps of a search wait for one another, and it is their latency that counts where there is one row (one
// after the other the 16 parts of 131072 columns took 14 us, counted one by one 41).
constexpr int kJoinThreads = 512;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void TokenJoinKernel(const T *__restrict__ logits, long long row0, ForwardArgs a) {
  HIP_DYNAMIC_SHARED(unsigned long long, keys)
  int *places = reinterpret_cast<int *>(keys + a.parts * a.k);
  const size_t row = row0 + blockIdx.x;
  if (a.mask != nullptr && a.mask[row] == 0) return;
  const int i = threadIdx.x, lane = i & (kWave - 1), all = a.parts * a.k;
  int64_t token = -1;
  float x_token = 0.0f;
  if (i < a.n) {
    token = a.tokens[row * a.n + i];
    if (token >= 0 && token < a.C) x_token = ToFloat(logits[row * a.row_stride + token]);
  }
  Sums sums{0, 0, 0};
  if (lane < a.parts) {
    const float4 v = a.part_sums[row * a.parts + lane];
    sums = Sums{v.x, v.y, v.z};
  }
  for (int j = i; j < all; j += kJoinThreads) {
    keys[j] = a.part_keys[row * all + j];
    places[j] = j % a.k;
  }
  sums = JoinLanes(sums, a.c);
  if (i < kWave) WriteRow(a, row, i, sums, token, x_token);
  if (a.k == 0) return;
  __syncthreads();
  const float ls = Log2(sums.s);
  int highest = 1;
  while (2 * highest <= a.k) highest *= 2;
  for (int task = i; task < all * ((a.parts + 3) / 4); task += kJoinThreads) {
    const int j = task % all, first = 4 * (task / all), own = j / a.k;
    const unsigned long long key = keys[j];
    int larger[4] = {0, 0, 0, 0}, place = 0;
    for (int step = highest; step > 0; step >>= 1)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const unsigned long long *part = keys + min(first + p, a.parts - 1) * a.k;
        if (larger[p] + step <= a.k && part[larger[p] + step - 1] > key) larger[p] += step;
      }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if (first + p >= a.parts || first + p == own) continue;
      // (0, past the last of its part: behind every key, in the order of the parts)
      place += key == 0 && first + p < own ? a.k : larger[p];
    }
    atomicAdd(&places[j], place);
  }
  __syncthreads();
  for (int j = i; j < all; j += kJoinThreads) {
    const unsigned long long key = keys[j];
    const int place = places[j];
    if (place >= a.k) continue;
    a.top_tokens[row * a.k + place] = key != 0 ? (int64_t)IndexOf(key) : -1;
    a.top_logprobs[row * a.k + place] = key != 0 ? LogProb(LogitOf(key), sums.m, ls, a.inv_tau) : Real<float>::NegInf();
  }
}

// ---- backward ---------------------------------------------------------------------------------------

struct BackwardArgs {
  long long row_stride;
  const int64_t *tokens;
  const uint8_t *mask;
  const float *stats, *entropy;
  const int64_t *top_tokens;
  const float *logprobs_grad, *entropy_grad, *top_grad;
  int C, n, k;
  float c, inv_tau;
};

// dx of an element that is no entry: -p (G + gH (log p + H)) / tau, with 1 / (s tau) in the coefficients
struct SoftmaxGrad {
  float m, c, flat, slope;
  float entry;  // what an entry's own gradient is multiplied by: 1 / tau
  __device__ __forceinline__ float At(float x) const {
    const float d = (x - m) * c;
    return Exp2(d) * (flat + slope * fmaxf(d, kNothing));
  }
};

// A row's entries in LDS, lane by lane of the n that share it; returns this lane's part of the sum of their gradients.
// *wrong: whether a token of this lane's is past the vocabulary.
__device__ __forceinline__ float ReadEntries(const BackwardArgs &a, size_t row, int i, int n, int entries, int *entry,
                                             float *entry_grad, bool write, bool *wrong) {
  const int used = a.logprobs_grad != nullptr ? a.n : 0;
  float sum = 0.0f;
  *wrong = false;
  for (; i < entries; i += n) {
    const bool given = i < used;
    const int64_t token = given ? a.tokens[row * a.n + i] : a.top_tokens[row * a.k + (i - used)];
    float g = given ? a.logprobs_grad[row * a.n + i] : a.top_grad[row * a.k + (i - used)];
    if (token < 0) g = 0.0f;
    if (token >= a.C) {
      g = __uint_as_float(0x7fc00000u);
      *wrong = true;
    }
    sum += g;
    if (write) {
      entry[i] = token < 0 || token >= a.C ? -1 : (int)token;
      entry_grad[i] = g;
    }
  }
  return sum;
}

// wrong: whether one of the row's tokens is past the vocabulary
__device__ __forceinline__ SoftmaxGrad RowGradOf(const BackwardArgs &a, size_t row, float sum, bool wrong) {
  const float s = a.stats[2 * row + 1];
  const float h = a.entropy_grad != nullptr ? a.entropy[row] : 0.0f;
  const float gh = a.entropy_grad != nullptr ? a.entropy_grad[row] : 0.0f;
  SoftmaxGrad f{a.stats[2 * row], a.c, 0.0f, 0.0f, 0.0f};
  if (s != 0.0f) {
    f.entry = a.inv_tau;
    const float inv_s = a.inv_tau / s;
    f.flat = -inv_s * (sum + gh * (h - kLn2 * Log2(s)));
    f.slope = -inv_s * gh * kLn2;
  } else if (wrong) {
    // (a row without any mass: every p is 0, and no logit moves a log-prob, whatever is sent back through it, NaN included;
    // a wrong token shows all the same)
    f.flat = __uint_as_float(0x7fc00000u);
  }
  return f;
}

// The entries' columns of [begin, end) over what is at `to` (column `begin` first), entry by entry of the n work-items.
template <typename T>
__device__ __forceinline__ void WriteEntries(const T *x, T *to, const int *entry, const float *entry_grad, int entries,
                                             int begin, int end, int i, int n, const SoftmaxGrad &f) {
  for (; i < entries; i += n) {
    const int token = entry[i];
    if (token < begin || token >= end) continue;
    const float xi = ToFloat(x[token]);
    float own = 0.0f;  // a token that is listed twice takes both gradients
    for (int j = 0; j < entries; ++j)
      if (entry[j] == token) own += entry_grad[j];
    FromFloat(f.At(xi) + (f.entry != 0.0f ? own * f.entry : 0.0f), &to[token - begin]);
  }
}

__host__ __device__ __forceinline__ int EntriesOf(const BackwardArgs &a) {
  return (a.logprobs_grad != nullptr ? a.n : 0) + (a.top_grad != nullptr ? a.k : 0);
}

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void TokenShortGradKernel(const T *__restrict__ logits, T *__restrict__ logits_grad,
                                                                 long long row0, long long rows, BackwardArgs a) {
  constexpr int kStage = StagedVecs<U>();
  __shared__ Vec stages[kStage > 0 ? kShortRows * kStage : 1];
  HIP_DYNAMIC_SHARED(float, entries_lds)
  const int lane = threadIdx.x % kShort, in_block = threadIdx.x / kShort, entries = EntriesOf(a);
  // the last row first: of a batch larger than the 256 MB memory-side cache it is the tail that the forward pass left there
  const long long from_last = (long long)blockIdx.x * kShortRows + in_block;
  if ((from_last & ~3ll) >= rows) return;  // (the wavefront's first row)
  const bool there = from_last < rows;
  const size_t row = row0 + (there ? rows - 1 - from_last : 0);  // (lanes without a row follow along and write nothing)
  const bool live = there && (a.mask == nullptr || a.mask[row] != 0);
  const T *x = logits + row * a.row_stride;
  T *dx = logits_grad + row * (size_t)a.C;
  float *entry_grad = entries_lds + (size_t)in_block * 2 * entries;
  int *entry = reinterpret_cast<int *>(entry_grad + entries);
  bool wrong;
  const float part_sum = ReadEntries(a, row, lane, kShort, live ? entries : 0, entry, entry_grad, true, &wrong);
  RowPart<T, U, 1, kShort> part;
  part.Load(x, __ballot(live) != 0 ? a.C : 0, 0, 0, lane);
  const SoftmaxGrad f = RowGradOf(a, row, GroupSum<kShort>(part_sum), GroupBallot<kShort>(wrong) != 0);
  const int all = live ? VecsOf<T>(a.C) : 0;
  T *to = kStage > 0 ? reinterpret_cast<T *>(stages + in_block * kStage) : dx;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = part.Vector(u, 0, 0, lane);
    if (at < all) WriteVec<false>(to, part.v[u], at, a.C, [&](float xi) { return f.At(xi); });
    else if (there && at < VecsOf<T>(a.C)) StoreZeros<false>(dx, at, a.C);
  }
  // (what is written above, and the list, are before what follows for every lane of the wavefront)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  WriteEntries(x, to, entry, entry_grad, live ? entries : 0, 0, a.C, lane, kShort, f);
  if (kStage == 0) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = part.Vector(u, 0, 0, lane);
    if (at < all) StoreStaged(to, dx, at, a.C);
  }
}

// Longer rows: W wavefronts take U vectors a lane of the stretch of a row that blockIdx.y counts.
template <typename T, int U, int W, bool kPast>
__global__ __launch_bounds__(W *kWave) void TokenLongGradKernel(const T *__restrict__ logits, T *__restrict__ logits_grad,
                                                                long long row0, long long rows, BackwardArgs a) {
  constexpr int kN = Lanes<T>::kN;
  __shared__ int entry[kMaxTokens + kMaxTop];
  __shared__ float entry_grad[kMaxTokens + kMaxTop];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const int entries = EntriesOf(a);
  const size_t row = row0 + rows - 1 - blockIdx.x;  // (the last row first, as above)
  const int first = (int)blockIdx.y * (U * W * kWave), all = VecsOf<T>(a.C);
  const T *x = logits + row * a.row_stride;
  T *dx = logits_grad + row * (size_t)a.C;
  if (a.mask != nullptr && a.mask[row] == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = RowPart<T, U, W>::Vector(u, first, wave, lane);
      if (at < all) StoreZeros<kPast>(dx, at, a.C);
    }
    return;
  }
  // (every wavefront needs the sum; the first leaves the list)
  bool wrong;
  const float sum = WaveSumF(ReadEntries(a, row, lane, kWave, entries, entry, entry_grad, wave == 0, &wrong));
  RowPart<T, U, W> part;
  part.template Load<kPast>(x, a.C, first, wave, lane);
  const SoftmaxGrad f = RowGradOf(a, row, sum, __ballot(wrong) != 0);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = part.Vector(u, first, wave, lane);
    if (at < all) WriteVec<kPast>(dx, part.v[u], at, a.C, [&](float xi) { return f.At(xi); });
  }
  if (entries == 0) return;
  __syncthreads();
  const int begin = first * kN, end = (int)min((long long)a.C, (long long)(first + U * W * kWave) * kN);
  WriteEntries(x, dx + begin, entry, entry_grad, entries, begin, end, (int)threadIdx.x, W * kWave, f);
}

// ---- launches ---------------------------------------------------------------------------------------

template <typename T, int U>
void LaunchShort(const T *logits, long long rows, bool entropy, const ForwardArgs &a, hipStream_t stream) {
  for (long long row0 = 0; row0 < rows; row0 += kRowsPerLaunch) {
    const long long n = rows - row0 < kRowsPerLaunch ? rows - row0 : kRowsPerLaunch;
    const dim3 grid((unsigned)((n + kShortRows - 1) / kShortRows)), block(kThreads);
    if (entropy) hipLaunchKernelGGL((TokenShortKernel<T, U, true>), grid, block, 0, stream, logits, row0, n, a);
    else hipLaunchKernelGGL((TokenShortKernel<T, U, false>), grid, block, 0, stream, logits, row0, n, a);
  }
}

template <typename T, int U, int W>
void LaunchHeld(const T *logits, long long rows, bool entropy, const ForwardArgs &a, hipStream_t stream) {
  for (long long row0 = 0; row0 < rows; row0 += kRowsPerLaunch) {
    const long long n = rows - row0 < kRowsPerLaunch ? rows - row0 : kRowsPerLaunch;
    const dim3 grid((unsigned)n, (unsigned)a.parts), block(W * kWave);
    if (entropy) hipLaunchKernelGGL((TokenHeldKernel<T, U, W, true>), grid, block, 0, stream, logits, row0, a);
    else hipLaunchKernelGGL((TokenHeldKernel<T, U, W, false>), grid, block, 0, stream, logits, row0, a);
    if (a.parts > 1)
      hipLaunchKernelGGL(TokenJoinKernel<T>, dim3((unsigned)n), dim3(kJoinThreads),
                         (size_t)a.parts * a.k * (sizeof(unsigned long long) + sizeof(int)), stream, logits, row0, a);
  }
}

template <typename T>
void LaunchStream(const T *logits, long long rows, bool entropy, const ForwardArgs &a, hipStream_t stream) {
  const int part_vecs = StreamShapeOf(rows, VecsOf<T>(a.C), Lanes<T>::kN).vecs;
  for (long long row0 = 0; row0 < rows; row0 += kRowsPerLaunch) {
    const long long n = rows - row0 < kRowsPerLaunch ? rows - row0 : kRowsPerLaunch;
    const dim3 grid((unsigned)n, (unsigned)a.parts), block(kStreamWaves * kWave);
    if (entropy) hipLaunchKernelGGL((TokenStreamKernel<T, true>), grid, block, 0, stream, logits, row0, part_vecs, a);
    else hipLaunchKernelGGL((TokenStreamKernel<T, false>), grid, block, 0, stream, logits, row0, part_vecs, a);
    if (a.parts > 1)
      hipLaunchKernelGGL(TokenJoinKernel<T>, dim3((unsigned)n), dim3(kJoinThreads), 0, stream, logits, row0, a);
  }
}

int PartsOf(long long rows, int C, int k, int dtype) {
  const int vecs = dtype == K2AMD_F32 ? VecsOf<float>(C) : VecsOf<Half>(C);
  if (vecs <= 16 * kShort || rows == 0) return 1;
  return k > 0 ? HeldShapeOf(rows, vecs).parts : StreamShapeOf(rows, vecs, dtype == K2AMD_F32 ? 4 : 8).parts;
}

template <typename T>
int Forward(const void *logits_v, long long rows, ForwardArgs a, hipStream_t stream) {
  const T *logits = static_cast<const T *>(logits_v);
  const int vecs = VecsOf<T>(a.C);
  const bool entropy = a.entropy != nullptr;
  if (vecs <= 2 * kShort) LaunchShort<T, 2>(logits, rows, entropy, a, stream);
  else if (vecs <= 4 * kShort) LaunchShort<T, 4>(logits, rows, entropy, a, stream);
  else if (vecs <= 8 * kShort) LaunchShort<T, 8>(logits, rows, entropy, a, stream);
  else if (vecs <= 16 * kShort) LaunchShort<T, 16>(logits, rows, entropy, a, stream);
  else if (a.k == 0) LaunchStream<T>(logits, rows, entropy, a, stream);
  else if (HeldShapeOf(rows, vecs).vecs == 1024) LaunchHeld<T, 4, 4>(logits, rows, entropy, a, stream);
  else LaunchHeld<T, 16, 4>(logits, rows, entropy, a, stream);
  return LaunchStatus();
}

template <typename T>
int Backward(const void *logits_v, void *grad_v, long long rows, const BackwardArgs &a, hipStream_t stream) {
  const T *logits = static_cast<const T *>(logits_v);
  T *grad = static_cast<T *>(grad_v);
  const int vecs = VecsOf<T>(a.C);
  for (long long done = 0; done < rows; done += kRowsPerLaunch) {
    const long long n = rows - done < kRowsPerLaunch ? rows - done : kRowsPerLaunch, row0 = rows - done - n;
    const dim3 short_grid((unsigned)((n + kShortRows - 1) / kShortRows)), block(kThreads);
    const dim3 grid((unsigned)n, (unsigned)((vecs + 16 * kWave - 1) / (16 * kWave)));
    const size_t lds = (size_t)kShortRows * 2 * EntriesOf(a) * sizeof(float);
    if (vecs <= 2 * kShort) hipLaunchKernelGGL((TokenShortGradKernel<T, 2>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (vecs <= 4 * kShort) hipLaunchKernelGGL((TokenShortGradKernel<T, 4>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (vecs <= 8 * kShort) hipLaunchKernelGGL((TokenShortGradKernel<T, 8>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (vecs <= 16 * kShort) hipLaunchKernelGGL((TokenShortGradKernel<T, 16>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (PastCache(rows, a.C, sizeof(T))) hipLaunchKernelGGL((TokenLongGradKernel<T, 4, 4, true>), grid, block, 0, stream, logits, grad, row0, n, a);
    else hipLaunchKernelGGL((TokenLongGradKernel<T, 4, 4, false>), grid, block, 0, stream, logits, grad, row0, n, a);
  }
  return LaunchStatus();
}

}  // namespace
}  // namespace k2amd

using namespace k2amd;

extern "C" {

size_t k2amd_token_logprobs_scratch_bytes(long long rows, int C, int k, int dtype) {
  if (rows < 0 || C < 1 || k < 0 || C > kMaxColumns || k > kMaxTop) return 0;
  const size_t parts = PartsOf(rows, C, k, dtype);
  return parts <= 1 ? 0 : ((size_t)rows * parts * (sizeof(float4) + (size_t)k * sizeof(unsigned long long)) + 15) / 16 * 16;
}

int k2amd_token_logprobs_forward(const void *logits, long long row_stride, const int64_t *tokens, const uint8_t *mask,
                                 float *logprobs, float *entropy, float *top_logprobs, int64_t *top_tokens, float *stats,
                                 long long rows, int C, int n, int k, float temperature, int dtype, void *scratch,
                                 size_t scratch_bytes, void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || n < 0 || k < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows, C) || n > kMaxTokens || k > kMaxTop) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || (n > 0 && (tokens == nullptr || logprobs == nullptr)) ||
      (k > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return K2AMD_ERR_INVALID_ARGUMENT;
  const int parts = PartsOf(rows, C, k, dtype);
  if (parts > 1 && (scratch == nullptr || Misaligned(scratch) || scratch_bytes < k2amd_token_logprobs_scratch_bytes(rows, C, k, dtype)))
    return K2AMD_ERR_WORKSPACE;
  float4 *sums = static_cast<float4 *>(scratch);
  const ForwardArgs a{row_stride, tokens, mask, logprobs, entropy, top_logprobs, top_tokens, stats, C, n, k,
                      (float)(kLog2E / (double)temperature), (float)(1.0 / (double)temperature), parts, sums,
                      parts > 1 ? reinterpret_cast<unsigned long long *>(sums + rows * parts) : nullptr};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32) return Forward<float>(logits, rows, a, st);
  if (dtype == K2AMD_F16) return Forward<Half>(logits, rows, a, st);
  return Forward<Bfloat>(logits, rows, a, st);
}

int k2amd_token_logprobs_backward(const void *logits, long long row_stride, const int64_t *tokens, const uint8_t *mask,
                                  const float *stats, const float *entropy, const int64_t *top_tokens,
                                  const float *logprobs_grad, const float *entropy_grad, const float *top_grad,
                                  void *logits_grad, long long rows, int C, int n, int k, float temperature, int dtype,
                                  void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || n < 0 || k < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows, C) || n > kMaxTokens || k > kMaxTop) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || stats == nullptr || logits_grad == nullptr || (n > 0 && logprobs_grad != nullptr && tokens == nullptr) ||
      (k > 0 && top_grad != nullptr && top_tokens == nullptr) || (entropy_grad != nullptr && entropy == nullptr))
    return K2AMD_ERR_INVALID_ARGUMENT;
  const BackwardArgs a{row_stride, tokens, mask, stats, entropy, top_tokens, logprobs_grad, entropy_grad, top_grad, C, n, k,
                       (float)(kLog2E / (double)temperature), (float)(1.0 / (double)temperature)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32) return Backward<float>(logits, logits_grad, rows, a, st);
  if (dtype == K2AMD_F16) return Backward<Half>(logits, logits_grad, rows, a, st);
  return Backward<Bfloat>(logits, logits_grad, rows, a, st);
}

}  // extern "C"
