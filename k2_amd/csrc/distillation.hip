// Distillation from a teacher's listed log-probs: the loss of every row, its sum, and the gradient with respect to the
// student's logits (k2amd_distillation_forward / _sum / _backward), and which rows of a pruned lattice take part
// (k2amd_rnnt_pruned_mask).
//
// The teacher's list of a row: tokens c_j with log-probs a_j (c_j < 0: no entry).  Student: p = softmax(x / tau).
//   renormalised: q_j = exp a_j / sum exp a,      L = sum_j q_j (log q_j - log p_cj)
//                 dx_i = (p_i - sum_{c_j = i} q_j) / tau
//   with a rest:  q_j = exp a_j, q_0 = max(0, 1 - sum q), p_0 = sum of p over the tokens that are not listed,
//                 L = sum_j q_j (a_j - log p_cj) + q_0 (log q_0 - log p_0),  Q = sum q + q_0
//                 dx_i = (Q p_i - sum_{c_j = i} q_j) / tau for a listed token, (Q p_0 - q_0) (p_i / p_0) / tau otherwise.
// p_0 is summed from the tokens that are not listed, with their own maximum: 1 - (sum of the listed) would lose it where
// the student is sure, which is where q_0 / p_0 matters.  Either way the gradient is one coefficient times an exponential
// for every element, and the listed elements are then written over it.
//
// Measured on an MI355X, kernel times after some hundred passes.  80000 x 500 (four fifths of the rows count), lists of 8, with
// a rest: forward 46 us in float32 and 29 in bfloat16, backward 56 and 28.  The forward pass of a training
// loop reads while the 160 MB (80 MB) of the last gradient leave the memory-side cache: with all its arithmetic taken out it
// took 40 us and 20 us.  8192 x 32000, lists of 20: forward 102 us in bfloat16 (5.1 TB/s) and 188 in float32 (5.6), backward
// 185 and 369 (5.7 TB/s both).  2048 x 131072, lists of 64, with a rest: forward in two parts 113 us in bfloat16 and 191 in
// float32 and 8 for their join, backward 181 and 383.
#include "token_rows.h"

namespace k2amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kShort = 16;                  // lanes that hold a short row
constexpr int kShortRows = kThreads / kShort;  // short rows of a workgroup
constexpr float kSkipped = -1.0f;  // in a record's last place, which is never negative: the row has no gradient

// ---- a row's list -----------------------------------------------------------------------------------
//
// The entries lie in LDS, entry j in the care of lane j mod L of the group that has the row: its token (-1: none), the
// teacher's log-prob a and the student's logit x.
struct List {
  int *token;
  float *a, *x;
  int K;  // 0 for a row without a usable list
  __device__ __forceinline__ List(float *lds, int entries)
      : token(reinterpret_cast<int *>(lds)), a(lds + entries), x(lds + 2 * entries), K(entries) {}
};
enum ListState { kNone, kUsable, kWrong };

// The tokens and the teacher's log-probs.  A log-prob of NaN or +inf (a teacher whose logits overflowed) is as wrong as a
// token past the vocabulary: the comparisons that follow would take it for an entry without weight.
template <int L>
__device__ __forceinline__ ListState ReadList(int C, const float *top_logprobs, const int64_t *top_tokens, const List &list,
                                              int lane, bool live) {
  bool present = false, wrong = false;
  if (live)
    for (int j = lane; j < list.K; j += L) {
      const int64_t given = top_tokens[j];
      const float a = top_logprobs[j];
      const int token = given >= 0 && given < C ? (int)given : -1;
      wrong |= given >= C || (token >= 0 && !(a < -Real<float>::NegInf()));
      present |= token >= 0;
      list.token[j] = token;
      list.a[j] = token >= 0 ? a : Real<float>::NegInf();
    }
  const bool any_wrong = GroupBallot<L>(wrong) != 0, any = GroupBallot<L>(present) != 0;
  return any_wrong ? kWrong : any ? kUsable : kNone;
}

// The logit of entry j's token.
template <typename T>
__device__ __forceinline__ float ListedLogit(const T *x, const List &list, int j) {
  const int token = j < list.K ? list.token[j] : -1;
  return token >= 0 ? ToFloat(x[token]) : Real<float>::NegInf();
}
// The logits of the whole list; that of the lane's first entry is at hand.
template <typename T, int L>
__device__ __forceinline__ void ReadLogits(const T *x, const List &list, int lane, float x_first) {
  if (lane < list.K) list.x[lane] = x_first;
  for (int j = lane + L; j < list.K; j += L) list.x[j] = ListedLogit(x, list, j);
}

// Bit r: the token of this lane's entry lane + r L stands earlier in the list.  All lanes of the wavefront come here.
template <int L>
__device__ __forceinline__ unsigned RepeatedEntries(const List &list, int lane) {
  unsigned repeated = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int j = lane, r = 0; j < list.K; j += L, ++r) {
    bool again = false;
    for (int i = 0; i < j; ++i) again |= list.token[i] == list.token[j];
    if (again) repeated |= 1u << r;
  }
  return repeated;
}

// Marks the list's tokens in `bits`, columns from `begin` on, and returns whether a lane of the wavefront found its token
// marked already.
template <int L>
__device__ __forceinline__ bool MarkListed(const List &list, int lane, unsigned *bits, int begin, int end) {
  bool again = false;
  for (int j = lane; j < list.K; j += L) {
    const int token = list.token[j];
    if (token < begin || token >= end) continue;
    const unsigned bit = 1u << ((token - begin) & 31);
    again |= (atomicOr(&bits[(token - begin) >> 5], bit) & bit) != 0;
  }
  return __ballot(again) != 0;
}

template <typename T, int U, int W, int L>
__device__ __forceinline__ void DropListed(RowPart<T, U, W, L> &part, int C, int lane, const unsigned *bits) {
  constexpr int kN = Lanes<T>::kN;
  const unsigned *own = bits + lane * kN / 32;  // a round of L vectors is whole words of marks
  const int shift = lane * kN % 32;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    unsigned marked = own[u * (L * kN / 32)] >> shift & ((1u << kN) - 1);
    if ((u + 1) * L * kN > C) {  // the round with the row's last vector: read to end with the row
      const int q = part.VectorAnew(u, 0, 0, lane);
      marked = q < VecsOf<T>(C) ? MarksOf<T>(bits, VecBase<T>(q, C), 0) : 0u;
    }
    DropMarked<T>(&part.v[u], marked);
  }
}

// the largest logit of what a group of lanes holds
template <typename T, int U, int W, int L>
__device__ __forceinline__ float HighOf(RowPart<T, U, W, L> &part) {
  float high[2] = {Real<float>::NegInf(), Real<float>::NegInf()};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Vec &v = part.Packed(u);
#pragma unroll
    for (int e = 0; e < Lanes<T>::kN; e += 2)
      high[e / 2 & 1] = fmaxf(fmaxf(high[e / 2 & 1], ElementOf<T>(v, e)), ElementOf<T>(v, e + 1));
  }
  return GroupMax<L>(fmaxf(high[0], high[1]));
}

// The loss of a row and its record {logit that the elements' exponent is taken from, coefficient of 2^..., m or the
// teacher's log-sum, sum of the target / s}, from its list and the sums over all its elements (kRest: over those that are
// not listed).  All lanes of the wavefront come here; lane 0 of the group writes.
template <int L, bool kRest>
__device__ __forceinline__ void FinishRow(List list, ListState state, unsigned repeated, Sums rest, int lane, float c,
                                          float inv_tau, bool live, float *loss_out, float *record) {
  if (state != kUsable) list.K = 0;
  float a_max = Real<float>::NegInf(), m_set = Real<float>::NegInf();
  for (int j = lane; j < list.K; j += L) {
    a_max = fmaxf(a_max, list.a[j]);
    m_set = fmaxf(m_set, list.x[j]);
  }
  a_max = GroupMax<L>(a_max);
  float m = rest.m, s = rest.s;
  if (kRest) {
    m_set = GroupMax<L>(m_set);
    m = rest.s == 0.0f ? m_set : fmaxf(rest.m, m_set);
    if (m == Real<float>::NegInf()) m = 0.0f;
    float s_set = 0.0f;
    for (int j = lane, r = 0; j < list.K; j += L, ++r)
      if (!(repeated >> r & 1u)) s_set += Exp2((list.x[j] - m) * c);  // (absent entries: -inf)
    s = GroupSum<L>(s_set) + (rest.s == 0.0f ? 0.0f : rest.s * Exp2((rest.m - m) * c));
  }
  const float ls = Log2(s);
  // the teacher: its log-sum, or which entry is (the first of) the largest
  float lse = 0.0f, at = Real<float>::NegInf();
  if (kRest) {
    for (int j = lane; j < list.K; j += L)
      if (list.a[j] == a_max) at = fmaxf(at, -(float)j);
    at = GroupMax<L>(at);
  } else {
    float sum = 0.0f;
    for (int j = lane; j < list.K; j += L) sum += Exp(list.a[j] - a_max);
    lse = a_max + kLn2 * Log2(GroupSum<L>(sum));
  }
  float others = 0.0f, loss = 0.0f;
  for (int j = lane; j < list.K; j += L) {
    const float a = list.a[j];
    const float q = a > Real<float>::NegInf() ? Exp(a - lse) : 0.0f;
    if (-(float)j != at) others += q;
    if (q > 0.0f) loss += q * ((a - lse) - LogProb(list.x[j], m, ls, inv_tau));
  }
  loss = GroupSum<L>(loss);
  float mass = 1.0f, p0 = 0.0f, q0 = 0.0f;
  if (kRest) {
    others = GroupSum<L>(others);
    // 1 - sum q, the largest by expm1: exact where the list holds nearly everything
    if (rest.s != 0.0f) q0 = fmaxf(0.0f, -expm1f(a_max) - others);
    mass = others + Exp(a_max) + q0;
    if (rest.s != 0.0f) {
      const float log_p0 = (rest.m - m) * inv_tau + kLn2 * (Log2(rest.s) - ls);
      p0 = Exp(log_p0);
      if (q0 > 0.0f) loss += q0 * (kLn2 * Log2(q0) - log_p0);
    }
  }
  if (lane != 0) return;
  // no list (without a rest, one of impossible tokens alone is none): nothing to learn; an index past the vocabulary or a
  // log-prob that is none is a mistake of the caller's and shows as NaN
  const bool skipped = !live || state == kNone || (state == kUsable && !kRest && a_max == Real<float>::NegInf());
  const float nan = __uint_as_float(0x7fc00000u);
  *loss_out = skipped ? 0.0f : state == kWrong ? nan : loss;
  if (record == nullptr) return;
  float4 r = make_float4(rest.m, rest.s == 0.0f ? 0.0f : (kRest ? (mass * p0 - q0) / rest.s : 1.0f / rest.s), kRest ? m : lse,
                         s == 0.0f ? 0.0f : mass / s);
  if (state == kWrong) r = make_float4(nan, nan, nan, nan);
  if (skipped) r = make_float4(0.0f, 0.0f, 0.0f, kSkipped);
  *reinterpret_cast<float4 *>(record) = r;
}

// ---- forward ----------------------------------------------------------------------------------------

struct ForwardArgs {
  long long row_stride;
  const float *top_logprobs;
  const int64_t *top_tokens;
  const uint8_t *mask;
  float *row_losses, *records;
  int C, K;
  float c, inv_tau;
  // rows in several parts: [rows][parts] m and s
  int parts;
  float2 *part_sums;
};

// Short rows: 16 lanes each.  What the row depends on (mask, list) is asked for first and together, then the row and the
// listed logits: two round trips to memory before the arithmetic, not four.
template <typename T, int U, bool kRest>
__global__ __launch_bounds__(kThreads) void DistillShortKernel(const T *__restrict__ logits, long long row0, long long rows,
                                                               ForwardArgs a) {
  constexpr int kWords = U * kShort * Lanes<T>::kN / 32 + 1;
  __shared__ unsigned listed[kRest ? kShortRows : 1][kRest ? kWords : 1];
  HIP_DYNAMIC_SHARED(float, lists)
  const int lane = threadIdx.x % kShort, group = threadIdx.x / kShort;
  const long long in_launch = (long long)blockIdx.x * kShortRows + group;
  if ((in_launch & ~3ll) >= rows) return;  // (the wavefront's first row)
  const bool there = in_launch < rows;
  const size_t row = row0 + (there ? in_launch : rows - 1);  // (a group without a row follows along and writes nothing)
  const uint8_t masked = a.mask == nullptr ? 1 : a.mask[row];
  List list(lists + (size_t)group * 3 * a.K, a.K);
  ListState state = ReadList<kShort>(a.C, a.top_logprobs + row * a.K, a.top_tokens + row * a.K, list, lane, there);
  const bool live = there && masked != 0;
  if (!live) state = kNone;
  if (state != kUsable) list.K = 0;
  const T *x = logits + row * a.row_stride;
  RowPart<T, U, 1, kShort> part;
  // (all four rows or none: a load that some lanes skip is a branch for each vector)
  part.Load(x, __ballot(state == kUsable) != 0 ? a.C : 0, 0, 0, lane);
  const float x_first = ListedLogit(x, list, lane);
  unsigned repeated = 0;
  if (kRest) {
    for (int i = lane; i < kWords; i += kShort) listed[group][i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (MarkListed<kShort>(list, lane, listed[group], 0, a.C)) repeated = RepeatedEntries<kShort>(list, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    DropListed(part, a.C, lane, listed[group]);
  }
  const float high = HighOf(part);
  const Sums sums = SumsOf<false>(part, state == kUsable ? high : Real<float>::NegInf(), a.c);
  ReadLogits<T, kShort>(x, list, lane, x_first);
  // (lane 0 of a group writes: one without a row is given another)
  FinishRow<kShort, kRest>(list, state, repeated, sums, there ? lane : lane + kShort, a.c, a.inv_tau, live, a.row_losses + row,
                           a.records == nullptr ? nullptr : a.records + 4 * row);
}

// Longer rows: four wavefronts read along a row or a part of it; the first has the list.
template <typename T, bool kRest>
__global__ __launch_bounds__(kThreads) void DistillLongKernel(const T *__restrict__ logits, long long row0, int part_vecs,
                                                              ForwardArgs a) {
  constexpr int kN = Lanes<T>::kN;
  __shared__ float lists[3 * kMaxTeacher];
  __shared__ float2 wave_sums[kWaves];
  HIP_DYNAMIC_SHARED(unsigned, listed)
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const size_t row = row0 + blockIdx.x;
  const int first = (int)blockIdx.y * part_vecs, end = min(VecsOf<T>(a.C), first + part_vecs);
  const bool live = a.mask == nullptr || a.mask[row] != 0, whole = a.parts == 1;
  const T *x = logits + row * a.row_stride;
  List list(lists, a.K);
  if (!live) {
    if (wave == 0 && whole)
      FinishRow<kWave, kRest>(list, kNone, 0, Sums{0, 0, 0}, lane, a.c, a.inv_tau, false, a.row_losses + row,
                              a.records == nullptr ? nullptr : a.records + 4 * row);
    return;
  }
  ListState state = kNone;
  unsigned repeated = 0;
  if (wave == 0 && (kRest || whole)) {
    state = ReadList<kWave>(a.C, a.top_logprobs + row * a.K, a.top_tokens + row * a.K, list, lane, true);
    if (state != kUsable) list.K = 0;
  }
  if (kRest) {
    for (int i = threadIdx.x; i < part_vecs * kN / 32 + 1; i += kThreads) listed[i] = 0;
    __syncthreads();
    if (wave == 0) {
      const int begin = first * kN;
      const bool again = MarkListed<kWave>(list, lane, listed, begin, min(a.C, begin + part_vecs * kN));
      if (again && whole) repeated = RepeatedEntries<kWave>(list, lane);
    }
    __syncthreads();
  }
  Sums sums = StreamSums<T, kWaves, false, kRest>(x, a.C, first, end, wave, lane, a.c, listed);
  if (lane == 0) wave_sums[wave] = make_float2(sums.m, sums.s);
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < kWaves; ++w) sums = Join(sums, Sums{wave_sums[w].x, wave_sums[w].y, 0.0f}, a.c);
  if (whole) {
    ReadLogits<T, kWave>(x, list, lane, ListedLogit(x, list, lane));
    FinishRow<kWave, kRest>(list, state, repeated, sums, lane, a.c, a.inv_tau, true, a.row_losses + row,
                            a.records == nullptr ? nullptr : a.records + 4 * row);
  } else if (lane == 0) {
    a.part_sums[row * a.parts + blockIdx.y] = make_float2(sums.m, sums.s);
  }
}

// Joins the parts of a row: a wavefront a row.
template <typename T, bool kRest>
__global__ __launch_bounds__(kWave) void DistillJoinKernel(const T *__restrict__ logits, long long row0, ForwardArgs a) {
  __shared__ float lists[3 * kMaxTeacher];
  const int lane = threadIdx.x;
  const size_t row = row0 + blockIdx.x;
  const bool live = a.mask == nullptr || a.mask[row] != 0;
  List list(lists, a.K);
  Sums sums{0, 0, 0};
  if (live && lane < a.parts) {
    const float2 v = a.part_sums[row * a.parts + lane];
    sums = Sums{v.x, v.y, 0.0f};
  }
  const ListState state = ReadList<kWave>(a.C, a.top_logprobs + row * a.K, a.top_tokens + row * a.K, list, lane, live);
  if (state != kUsable) list.K = 0;
  const T *x = logits + row * a.row_stride;
  ReadLogits<T, kWave>(x, list, lane, ListedLogit(x, list, lane));
  const unsigned repeated = kRest ? RepeatedEntries<kWave>(list, lane) : 0;
  sums = JoinLanes(sums, a.c);
  FinishRow<kWave, kRest>(list, state, repeated, sums, lane, a.c, a.inv_tau, live, a.row_losses + row,
                          a.records == nullptr ? nullptr : a.records + 4 * row);
}

// ---- backward ---------------------------------------------------------------------------------------

// What one row's gradient is scaled by: what reaches its loss, and the reduction's factor.
struct LossScale {
  const float *loss_grad;       // one value for every rows_per_loss rows
  unsigned rows_per_loss;
  const float *inverse_count;   // of the rows that count, where the loss is their mean, or null
  float factor;
  __device__ __forceinline__ float At(size_t row) const {
    const float g = loss_grad[(unsigned)row / rows_per_loss] * factor;
    return inverse_count != nullptr ? g * inverse_count[0] : g;
  }
};

struct BackwardArgs {
  long long row_stride;
  const float *top_logprobs;
  const int64_t *top_tokens;
  const float *records;
  LossScale scale;
  int C, K;
  float c;
};

// One row's gradient: coefficient * 2^((x - from) c) for an element that is not listed, p - (sum of its entries' q) else.
template <bool kRest>
struct RowGrad {
  float from, coefficient, m, share, lse, g;
  bool skipped;
  __device__ __forceinline__ RowGrad(const float4 &r, float scale)
      : from(r.x), coefficient(r.y * scale), m(kRest ? r.z : r.x), share(r.w), lse(kRest ? 0.0f : r.z), g(scale),
        skipped(r.w == kSkipped) {}
  __device__ __forceinline__ float Unlisted(float x, float c) const { return coefficient * Exp2((x - from) * c); }
  __device__ __forceinline__ float Listed(float x, float q, float c) const { return g * (share * Exp2((x - m) * c) - q); }
};

// The listed columns of [begin, end) over what is at `to` (column `begin` first), entry j by work-item j mod n; x_first: the
// logit of its first entry.
template <typename T, bool kRest>
__device__ __forceinline__ void WriteListed(const T *x, T *to, const int *token, const float *q, int K, int begin, int end, int i,
                                            int n, float x_first, const RowGrad<kRest> &f, float c) {
  for (int j = i; j < K; j += n) {
    const int at = token[j];
    if (at < begin || at >= end) continue;
    float sum = 0.0f;  // a token that is listed twice takes both
    for (int l = 0; l < K; ++l)
      if (token[l] == at) sum += q[l];
    FromFloat(f.Listed(j == i ? x_first : ToFloat(x[at]), sum, c), &to[at - begin]);
  }
}

template <typename T, int U, bool kRest>
__global__ __launch_bounds__(kThreads) void DistillShortGradKernel(const T *__restrict__ logits, T *__restrict__ logits_grad,
                                                                   long long row0, long long rows, BackwardArgs a) {
  constexpr int kStage = StagedVecs<U>();
  __shared__ Vec stages[kStage > 0 ? kShortRows * kStage : 1];
  HIP_DYNAMIC_SHARED(float, lists)
  const int lane = threadIdx.x % kShort, group = threadIdx.x / kShort;
  // the last row first: of a batch larger than the 256 MB memory-side cache it is the tail that the forward pass left there
  const long long from_last = (long long)blockIdx.x * kShortRows + group;
  if ((from_last & ~3ll) >= rows) return;  // (the wavefront's first row)
  const bool there = from_last < rows;
  const size_t row = row0 + (there ? rows - 1 - from_last : 0);  // (a group without a row follows along and writes nothing)
  const T *x = logits + row * a.row_stride;
  T *dx = logits_grad + row * (size_t)a.C;
  // asked for together: the record, the list; then the row and the first listed logits
  const float4 record = *reinterpret_cast<const float4 *>(a.records + 4 * row);
  const float scale = a.scale.At(row);
  int64_t given = -1;
  float teacher = 0.0f;
  if (lane < a.K) {
    given = a.top_tokens[row * a.K + lane];
    teacher = a.top_logprobs[row * a.K + lane];
  }
  const RowGrad<kRest> f(record, scale);
  const bool live = there && !f.skipped;
  RowPart<T, U, 1, kShort> part;
  part.Load(x, __ballot(live) != 0 ? a.C : 0, 0, 0, lane);
  const bool usable = live && given >= 0 && given < a.C;
  const float x_first = usable ? ToFloat(x[given]) : 0.0f;
  int *token = reinterpret_cast<int *>(lists) + (size_t)group * 2 * a.K;
  float *q = lists + (size_t)group * 2 * a.K + a.K;
  if (lane < a.K) {
    token[lane] = usable ? (int)given : -1;
    q[lane] = Exp(teacher - f.lse);
  }
  for (int j = lane + kShort; j < a.K; j += kShort) {
    given = a.top_tokens[row * a.K + j];
    token[j] = live && given >= 0 && given < a.C ? (int)given : -1;
    q[j] = Exp(a.top_logprobs[row * a.K + j] - f.lse);
  }
  const int all = live ? VecsOf<T>(a.C) : 0;
  T *to = kStage > 0 ? reinterpret_cast<T *>(stages + group * kStage) : dx;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = part.Vector(u, 0, 0, lane);
    if (at < all) WriteVec<false>(to, part.v[u], at, a.C, [&](float xi) { return f.Unlisted(xi, a.c); });
    else if (there && at < VecsOf<T>(a.C)) StoreZeros<false>(dx, at, a.C);
  }
  // (what is written above, and the list, are before what follows for every lane of the wavefront)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  WriteListed(x, to, token, q, live ? a.K : 0, 0, a.C, lane, kShort, x_first, f, a.c);
  if (kStage == 0) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = part.Vector(u, 0, 0, lane);
    if (at < all) StoreStaged(to, dx, at, a.C);
  }
}

template <typename T, int U, int W, bool kRest, bool kPast>
__global__ __launch_bounds__(W *kWave) void DistillLongGradKernel(const T *__restrict__ logits, T *__restrict__ logits_grad,
                                                                  long long row0, long long rows, BackwardArgs a) {
  constexpr int kN = Lanes<T>::kN;
  __shared__ int token[kMaxTeacher];
  __shared__ float q[kMaxTeacher];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const size_t row = row0 + rows - 1 - blockIdx.x;  // (the last row first, as above)
  const int first = (int)blockIdx.y * (U * W * kWave), all = VecsOf<T>(a.C);
  const T *x = logits + row * a.row_stride;
  T *dx = logits_grad + row * (size_t)a.C;
  const RowGrad<kRest> f(*reinterpret_cast<const float4 *>(a.records + 4 * row), a.scale.At(row));
  RowPart<T, U, W> part;
  part.template Load<kPast>(x, f.skipped ? 0 : a.C, first, wave, lane);
  for (int j = threadIdx.x; j < a.K; j += W * kWave) {
    const int64_t given = a.top_tokens[row * a.K + j];
    token[j] = given >= 0 && given < a.C && !f.skipped ? (int)given : -1;
    q[j] = Exp(a.top_logprobs[row * a.K + j] - f.lse);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = part.Vector(u, first, wave, lane);
    if (at >= all) continue;
    if (f.skipped) StoreZeros<kPast>(dx, at, a.C);
    else WriteVec<kPast>(dx, part.v[u], at, a.C, [&](float xi) { return f.Unlisted(xi, a.c); });
  }
  __syncthreads();
  const int i = threadIdx.x, begin = first * kN, end = (int)min((long long)a.C, (long long)(first + U * W * kWave) * kN);
  const int mine = i < a.K ? token[i] : -1;
  WriteListed(x, dx + begin, token, q, a.K, begin, end, i, W * kWave, mine >= begin && mine < end ? ToFloat(x[mine]) : 0.0f, f,
              a.c);
}

// ---- sums, masks and launches -----------------------------------------------------------------------

// Sums of rows_per_sum values each, and how many rows count, in a fixed order and in double, eight values on their way at a time
// in each work-item.  Up to kOneChunk of them are one workgroup's (4.9 us at 8192); more are cut into chunks of kChunk, for a
// workgroup each, which a wavefront joins in a second launch (80000 in chunks of 16384 took 14.4 us, five workgroups going
// twice to memory).
constexpr int kOneChunk = 16384, kChunk = 2048, kSumThreads = 1024, kChunkThreads = kChunk / 8;

struct SumOutput {
  float *sums, *inverse_count;
  int mean;
  float factor;
  __device__ __forceinline__ void Write(size_t i, double sum, double count) const {
    count = count > 1 ? count : 1;
    sums[i] = (float)(sum * factor / (mean ? count : 1.0));
    if (inverse_count != nullptr) inverse_count[i] = (float)(1.0 / count);
  }
};

__global__ __launch_bounds__(kSumThreads) void RowChunkSumKernel(const float *__restrict__ values,
                                                                 const uint8_t *__restrict__ mask, int rows_per_sum,
                                                                 double *__restrict__ partial, SumOutput out) {
  __shared__ double lds[2 * kSumThreads / kWave];
  // (64 bits: up to 2^31 - 1 rows, and the end of the last chunk and the step past it lie beyond them)
  const long long first = (long long)blockIdx.x * kChunk;
  const long long last = gridDim.x == 1 ? rows_per_sum : min((long long)rows_per_sum, first + kChunk);
  const size_t base = (size_t)blockIdx.y * rows_per_sum;
  double sum = 0, count = 0;
  for (long long i = first + threadIdx.x; i < last; i += 8 * (int)blockDim.x) {
    float v[8];
    uint8_t m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long at = i + j * (int)blockDim.x;
      v[j] = at < last ? values[base + at] : 0.0f;
      m[j] = at < last ? (mask != nullptr ? mask[base + at] : 1) : 0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum += v[j];
      count += m[j] != 0 ? 1.0 : 0.0;
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, kWave);
    count += __shfl_xor(count, off, kWave);
  }
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  if (lane == 0) {
    lds[2 * wave] = sum;
    lds[2 * wave + 1] = count;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < (int)blockDim.x / kWave; ++w) {
    sum += lds[2 * w];
    count += lds[2 * w + 1];
  }
  if (gridDim.x == 1) {
    out.Write(blockIdx.y, sum, count);
  } else {
    partial[2 * ((size_t)blockIdx.y * gridDim.x + blockIdx.x)] = sum;
    partial[2 * ((size_t)blockIdx.y * gridDim.x + blockIdx.x) + 1] = count;
  }
}

__global__ __launch_bounds__(kWave) void RowSumKernel(const double *__restrict__ partial, int chunks, SumOutput out) {
  double sum = 0, count = 0;
  for (int i = threadIdx.x; i < chunks; i += kWave) {
    sum += partial[2 * ((size_t)blockIdx.x * chunks + i)];
    count += partial[2 * ((size_t)blockIdx.x * chunks + i) + 1];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, kWave);
    count += __shfl_xor(count, off, kWave);
  }
  if (threadIdx.x == 0) out.Write(blockIdx.x, sum, count);
}

__global__ void PrunedMaskKernel(const int64_t *__restrict__ ranges, const int64_t *__restrict__ boundary,
                                 uint8_t *__restrict__ mask, int Tn, int R, long long rows) {
  const long long row = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= rows) return;
  const long long frame = row / R;
  const int64_t b = frame / Tn, t = frame - b * Tn, s = ranges[row];
  mask[row] = t >= boundary[4 * b + 1] && t < boundary[4 * b + 3] && s >= boundary[4 * b] && s <= boundary[4 * b + 2];
}

int PartsOf(long long rows, int C, int dtype) {
  const int each = dtype == K2AMD_F32 ? Lanes<float>::kN : Lanes<Half>::kN, vecs = (C + each - 1) / each;
  return vecs <= 16 * kShort || rows == 0 ? 1 : StreamShapeOf(rows, vecs, each).parts;
}

template <typename T, bool kRest>
int ForwardOf(const T *logits, long long rows, const ForwardArgs &a, hipStream_t stream) {
  const int vecs = VecsOf<T>(a.C);
  const LongShape shape = StreamShapeOf(rows, vecs, Lanes<T>::kN);
  const size_t marks = kRest ? (size_t)(shape.vecs * Lanes<T>::kN / 32 + 1) * sizeof(unsigned) : 0;
  for (long long row0 = 0; row0 < rows; row0 += kRowsPerLaunch) {
    const long long n = rows - row0 < kRowsPerLaunch ? rows - row0 : kRowsPerLaunch;
    const dim3 short_grid((unsigned)((n + kShortRows - 1) / kShortRows)), block(kThreads), grid((unsigned)n, (unsigned)a.parts);
    const size_t lds = (size_t)kShortRows * 3 * a.K * sizeof(float);
    if (vecs <= 2 * kShort) hipLaunchKernelGGL((DistillShortKernel<T, 2, kRest>), short_grid, block, lds, stream, logits, row0, n, a);
    else if (vecs <= 4 * kShort) hipLaunchKernelGGL((DistillShortKernel<T, 4, kRest>), short_grid, block, lds, stream, logits, row0, n, a);
    else if (vecs <= 8 * kShort) hipLaunchKernelGGL((DistillShortKernel<T, 8, kRest>), short_grid, block, lds, stream, logits, row0, n, a);
    else if (vecs <= 16 * kShort) hipLaunchKernelGGL((DistillShortKernel<T, 16, kRest>), short_grid, block, lds, stream, logits, row0, n, a);
    else hipLaunchKernelGGL((DistillLongKernel<T, kRest>), grid, block, marks, stream, logits, row0, shape.vecs, a);
    if (a.parts > 1) hipLaunchKernelGGL((DistillJoinKernel<T, kRest>), dim3((unsigned)n), dim3(kWave), 0, stream, logits, row0, a);
  }
  return LaunchStatus();
}

template <typename T, bool kRest>
int BackwardOf(const T *logits, T *grad, long long rows, const BackwardArgs &a, hipStream_t stream) {
  const int vecs = VecsOf<T>(a.C);
  const bool past = PastCache(rows, a.C, sizeof(T));
  for (long long done = 0; done < rows; done += kRowsPerLaunch) {
    const long long n = rows - done < kRowsPerLaunch ? rows - done : kRowsPerLaunch, row0 = rows - done - n;
    const dim3 short_grid((unsigned)((n + kShortRows - 1) / kShortRows)), block(kThreads);
    const dim3 grid((unsigned)n, (unsigned)((vecs + 16 * kWave - 1) / (16 * kWave)));
    const size_t lds = (size_t)kShortRows * 2 * a.K * sizeof(float);
    if (vecs <= 2 * kShort) hipLaunchKernelGGL((DistillShortGradKernel<T, 2, kRest>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (vecs <= 4 * kShort) hipLaunchKernelGGL((DistillShortGradKernel<T, 4, kRest>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (vecs <= 8 * kShort) hipLaunchKernelGGL((DistillShortGradKernel<T, 8, kRest>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (vecs <= 16 * kShort) hipLaunchKernelGGL((DistillShortGradKernel<T, 16, kRest>), short_grid, block, lds, stream, logits, grad, row0, n, a);
    else if (past) hipLaunchKernelGGL((DistillLongGradKernel<T, 4, 4, kRest, true>), grid, block, 0, stream, logits, grad, row0, n, a);
    else hipLaunchKernelGGL((DistillLongGradKernel<T, 4, 4, kRest, false>), grid, block, 0, stream, logits, grad, row0, n, a);
  }
  return LaunchStatus();
}

template <typename T>
int Forward(const void *logits, long long rows, int rest, const ForwardArgs &a, hipStream_t stream) {
  const T *x = static_cast<const T *>(logits);
  return rest ? ForwardOf<T, true>(x, rows, a, stream) : ForwardOf<T, false>(x, rows, a, stream);
}

template <typename T>
int Backward(const void *logits, void *grad, long long rows, int rest, const BackwardArgs &a, hipStream_t stream) {
  const T *x = static_cast<const T *>(logits);
  T *dx = static_cast<T *>(grad);
  return rest ? BackwardOf<T, true>(x, dx, rows, a, stream) : BackwardOf<T, false>(x, dx, rows, a, stream);
}

long long SumChunks(long long rows_per_sum) { return rows_per_sum <= kOneChunk ? 1 : (rows_per_sum + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace k2amd

using namespace k2amd;

extern "C" {

size_t k2amd_distillation_scratch_bytes(long long rows, int C, int dtype) {
  if (rows < 0 || C < 1 || C > kMaxColumns) return 0;
  const size_t parts = PartsOf(rows, C, dtype);
  return parts <= 1 ? 0 : ((size_t)rows * parts * sizeof(float2) + 15) / 16 * 16;
}

int k2amd_distillation_forward(const void *logits, long long row_stride, const float *top_logprobs,
                               const int64_t *top_tokens, const uint8_t *mask, float *row_losses, float *records,
                               long long rows, int C, int K, int rest, float temperature, int dtype, void *scratch,
                               size_t scratch_bytes, void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || K < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows, C) || K > kMaxTeacher) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || row_losses == nullptr || Misaligned(records) || (K > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return K2AMD_ERR_INVALID_ARGUMENT;
  const int parts = PartsOf(rows, C, dtype);
  if (parts > 1 && (scratch == nullptr || Misaligned(scratch) || scratch_bytes < k2amd_distillation_scratch_bytes(rows, C, dtype)))
    return K2AMD_ERR_WORKSPACE;
  const ForwardArgs a{row_stride, top_logprobs, top_tokens, mask, row_losses, records, C, K,
                      (float)(kLog2E / (double)temperature), (float)(1.0 / (double)temperature), parts,
                      static_cast<float2 *>(scratch)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32) return Forward<float>(logits, rows, rest, a, st);
  if (dtype == K2AMD_F16) return Forward<Half>(logits, rows, rest, a, st);
  return Forward<Bfloat>(logits, rows, rest, a, st);
}

int k2amd_distillation_backward(const void *logits, long long row_stride, const float *top_logprobs,
                                const int64_t *top_tokens, const float *records, const float *loss_grad,
                                long long rows_per_loss, const float *inverse_count, float factor, void *logits_grad,
                                long long rows, int C, int K, int rest, float temperature, int dtype, void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || K < 0 || rows_per_loss < 1) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows, C) || K > kMaxTeacher) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || records == nullptr || loss_grad == nullptr || logits_grad == nullptr || Misaligned(records) ||
      (K > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return K2AMD_ERR_INVALID_ARGUMENT;
  const BackwardArgs a{row_stride, top_logprobs, top_tokens, records,
                       LossScale{loss_grad, (unsigned)(rows_per_loss < rows ? rows_per_loss : rows), inverse_count, (float)((double)factor / (double)temperature)}, C, K,
                       (float)(kLog2E / (double)temperature)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32) return Backward<float>(logits, logits_grad, rows, rest, a, st);
  if (dtype == K2AMD_F16) return Backward<Half>(logits, logits_grad, rows, rest, a, st);
  return Backward<Bfloat>(logits, logits_grad, rows, rest, a, st);
}

size_t k2amd_distillation_sum_scratch_bytes(long long num_sums, long long rows_per_sum) {
  if (num_sums < 0 || rows_per_sum < 0) return 0;
  const size_t chunks = (size_t)SumChunks(rows_per_sum);
  return chunks <= 1 ? 0 : (size_t)num_sums * chunks * 2 * sizeof(double);
}

int k2amd_distillation_sum(const float *row_losses, const uint8_t *mask, float *sums, float *inverse_count,
                           long long num_sums, long long rows_per_sum, int mean, float factor, void *scratch,
                           size_t scratch_bytes, void *stream) {
  if (num_sums < 0 || rows_per_sum < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (num_sums > 65535 || rows_per_sum >= (1ll << 31)) return K2AMD_ERR_UNSUPPORTED;
  if (num_sums == 0) return K2AMD_OK;
  if (sums == nullptr || (rows_per_sum > 0 && row_losses == nullptr)) return K2AMD_ERR_INVALID_ARGUMENT;
  const int chunks = (int)SumChunks(rows_per_sum);
  if (chunks > 1 && (scratch == nullptr || Misaligned(scratch) ||
                     scratch_bytes < k2amd_distillation_sum_scratch_bytes(num_sums, rows_per_sum)))
    return K2AMD_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const SumOutput out{sums, inverse_count, mean, factor};
  hipLaunchKernelGGL(RowChunkSumKernel, dim3((unsigned)chunks, (unsigned)num_sums), dim3(chunks == 1 ? kSumThreads : kChunkThreads), 0, st, row_losses, mask,
                     (int)rows_per_sum, static_cast<double *>(scratch), out);
  if (chunks > 1)
    hipLaunchKernelGGL(RowSumKernel, dim3((unsigned)num_sums), dim3(kWave), 0, st, static_cast<const double *>(scratch), chunks,
                       out);
  return LaunchStatus();
}

int k2amd_rnnt_pruned_mask(const int64_t *ranges, const int64_t *boundary, uint8_t *mask, int B, int T, int R, void *stream) {
  if (B < 0 || T < 0 || R < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  const long long rows = (long long)B * T * R;
  if (rows >= (1ll << 31)) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (ranges == nullptr || boundary == nullptr || mask == nullptr) return K2AMD_ERR_INVALID_ARGUMENT;
  hipLaunchKernelGGL(PrunedMaskKernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     ranges, boundary, mask, T, R, rows);
  return LaunchStatus();
}

}  // extern "C"
