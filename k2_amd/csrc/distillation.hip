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
#include "token_rows.h"

namespace k2amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr float kSkipped = -1.0f;  // in a record's last place, which is never negative: the row has no gradient
constexpr int kSegment = 65536;  // columns whose membership of the list is kept as bits in LDS at a time

__device__ __forceinline__ float BlockMax(float v, float *lds) {
  v = WaveMaxF(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) v = fmaxf(v, lds[w]);
  return v;
}
__device__ __forceinline__ float BlockSum(float v, float *lds) {
  v = WaveSumF(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kWaves; ++w) v += lds[w];
  return v;
}

// One workgroup a row.
template <typename T, bool kRest>
__global__ __launch_bounds__(kThreads) void DistillForwardKernel(
    const T *__restrict__ logits, long long row_stride, const float *__restrict__ top_logprobs,
    const int64_t *__restrict__ top_tokens, const uint8_t *__restrict__ mask, float *__restrict__ row_losses,
    float *__restrict__ records, int C, int K, float c, float inv_tau) {
  __shared__ float lds[kWaves];
  __shared__ int entry[kMaxTeacher];
  __shared__ unsigned listed[kRest ? kSegment / 32 : 1];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const bool live = mask == nullptr || mask[row] != 0;
  // the list: entry j in work-item j
  int token = -1;
  float a = Real<float>::NegInf();
  bool wrong = false;
  if (live && tid < K) {
    const int64_t given = top_tokens[row * K + tid];
    wrong = given >= C;
    if (given >= 0 && !wrong) {
      token = (int)given;
      a = top_logprobs[row * K + tid];
    }
    entry[tid] = token;
  }
  const float present = BlockSum(token >= 0 || wrong ? 1.0f : 0.0f, lds);
  const float bad = BlockSum(wrong ? 1.0f : 0.0f, lds);
  const float a_max = BlockMax(a, lds);
  // no list (without a rest, one of impossible tokens alone is none): nothing to learn; an index past the vocabulary is a
  // mistake of the caller's and shows as NaN
  if (!live || present == 0.0f || bad != 0.0f || (!kRest && a_max == Real<float>::NegInf())) {
    const float v = live && bad != 0.0f ? __uint_as_float(0x7fc00000u) : 0.0f;
    if (tid == 0) row_losses[row] = v;
    if (records != nullptr && tid < 4) records[4 * row + tid] = v == 0.0f && tid == 3 ? kSkipped : v;
    return;
  }
  const T *x = logits + row * row_stride;
  const float xj = token >= 0 ? ToFloat(x[token]) : Real<float>::NegInf();
  bool first = token >= 0;  // a token listed twice is one token of the set
  if (kRest)
    for (int j = 0; j < tid && j < K; ++j)
      if (entry[j] == token) first = false;

  // the sum over the row, or over what is not listed
  float m_rest = Real<float>::NegInf(), s_rest = 0.0f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int lo = 0; lo < C; lo += kSegment) {
      const int hi = min(C, lo + kSegment);
      if (kRest) {
        __syncthreads();
        for (int i = tid; i < (hi - lo + 31) / 32; i += kThreads) listed[i] = 0;
        __syncthreads();
        if (token >= lo && token < hi) atomicOr(&listed[(token - lo) >> 5], 1u << ((token - lo) & 31));
        __syncthreads();
      }
      for (int i = lo + tid; i < hi; i += kThreads) {
        if (kRest && (listed[(i - lo) >> 5] >> ((i - lo) & 31) & 1u)) continue;
        const float v = ToFloat(x[i]);
        if (pass == 0) m_rest = fmaxf(m_rest, v);
        else s_rest += Exp2((v - m_rest) * c);
      }
    }
    if (pass == 0) {
      m_rest = BlockMax(m_rest, lds);
      if (m_rest == Real<float>::NegInf()) m_rest = 0.0f;
    } else {
      s_rest = BlockSum(s_rest, lds);
    }
  }
  float m = m_rest, s = s_rest;
  if (kRest) {
    const float m_set = BlockMax(first ? xj : Real<float>::NegInf(), lds);
    m = s_rest == 0.0f ? m_set : fmaxf(m_rest, m_set);
    if (m == Real<float>::NegInf()) m = 0.0f;
    const float s_set = BlockSum(first ? Exp2((xj - m) * c) : 0.0f, lds);
    s = s_set + (s_rest == 0.0f ? 0.0f : s_rest * Exp2((m_rest - m) * c));
  }
  const float ls = Log2(s);

  // the teacher
  float lse = 0.0f, q0 = 0.0f;
  if (!kRest) lse = a_max + logf(BlockSum(token >= 0 ? expf(a - a_max) : 0.0f, lds));
  const float q = token >= 0 && a > Real<float>::NegInf() ? expf(a - lse) : 0.0f;
  float mass = BlockSum(q, lds);
  if (kRest) {
    // 1 - sum q, the largest by expm1: exact where the list holds nearly everything
    const float at = BlockMax(token >= 0 && a == a_max ? -(float)tid : -(float)kThreads, lds);
    const float others = BlockSum(at == -(float)tid ? 0.0f : q, lds);
    q0 = s_rest == 0.0f ? 0.0f : fmaxf(0.0f, -expm1f(a_max) - others);
    mass += q0;
  }
  float loss = 0.0f;
  if (q > 0.0f) {
    loss = q * ((a - lse) - LogProb(xj, m, ls, inv_tau));
  }
  loss = BlockSum(loss, lds);
  float p0 = 0.0f;
  if (kRest && s_rest != 0.0f) {
    const float log_p0 = kLn2 * ((m_rest - m) * c + Log2(s_rest) - ls);
    p0 = expf(log_p0);
    if (q0 > 0.0f) loss += q0 * (logf(q0) - log_p0);
  }
  if (tid == 0) {
    row_losses[row] = loss;
    if (records != nullptr) {
      float *r = records + 4 * row;
      r[0] = m_rest;
      r[1] = s_rest == 0.0f ? 0.0f : (kRest ? (mass * p0 - q0) / s_rest : 1.0f / s_rest);
      r[2] = kRest ? m : lse;
      r[3] = s == 0.0f ? 0.0f : mass / s;
    }
  }
}

// What one row's gradient is scaled by: what reaches its loss, and the reduction's factor.
struct LossScale {
  const float *loss_grad;       // one value for every rows_per_loss rows
  long long rows_per_loss;
  const float *inverse_count;   // of the rows that count, where the loss is their mean, or null
  float factor;
  __device__ __forceinline__ float At(size_t row) const {
    float g = loss_grad[row / rows_per_loss] * factor;
    return inverse_count != nullptr ? g * inverse_count[0] : g;
  }
};

template <typename T, bool kRest>
__global__ __launch_bounds__(kThreads) void DistillBackwardKernel(
    const T *__restrict__ logits, long long row_stride, const float *__restrict__ top_logprobs,
    const int64_t *__restrict__ top_tokens, const float *__restrict__ records, LossScale scale,
    T *__restrict__ logits_grad, int C, int K, float c) {
  __shared__ int entry[kMaxTeacher];
  __shared__ float entry_q[kMaxTeacher];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x;
  T *dx = logits_grad + row * C;
  const float base = records[4 * row + 1], third = records[4 * row + 2], share = records[4 * row + 3];
  if (share == kSkipped) {
    for (int i = tid; i < C; i += kThreads) FromFloat(0.0f, &dx[i]);
    return;
  }
  const T *x = logits + row * row_stride;
  const float g = scale.At(row), m_rest = records[4 * row];
  if (tid < K) {
    const int64_t token = top_tokens[row * K + tid];
    const float a = top_logprobs[row * K + tid];
    entry[tid] = token >= 0 && token < C ? (int)token : -1;
    entry_q[tid] = a > Real<float>::NegInf() ? expf(a - (kRest ? 0.0f : third)) : 0.0f;
  }
  for (int i = tid; i < C; i += kThreads) FromFloat(g * base * Exp2((ToFloat(x[i]) - m_rest) * c), &dx[i]);
  __syncthreads();
  if (tid < K && entry[tid] >= 0) {
    float q = 0.0f;
    for (int j = 0; j < K; ++j)
      if (entry[j] == entry[tid]) q += entry_q[j];
    const float p = share * Exp2((ToFloat(x[entry[tid]]) - (kRest ? third : m_rest)) * c);
    FromFloat(g * (p - q), &dx[entry[tid]]);
  }
}

// Sums of rows_per_sum values each, and how many rows count, in a fixed order: chunks of kChunk values a workgroup, in
// double, then one workgroup a sum over its chunks.
constexpr int kChunk = 8192;

__global__ __launch_bounds__(kThreads) void RowChunkSumKernel(const float *__restrict__ values,
                                                              const uint8_t *__restrict__ mask, long long rows_per_sum,
                                                              double *__restrict__ partial) {
  __shared__ double lds[2 * kWaves];
  const long long first = (long long)blockIdx.x * kChunk, last = min(rows_per_sum, first + (long long)kChunk);
  const size_t base = (size_t)blockIdx.y * rows_per_sum;
  double sum = 0, count = 0;
  for (long long i = first + threadIdx.x; i < last; i += kThreads) {
    sum += values[base + i];
    if (mask == nullptr || mask[base + i] != 0) count += 1;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, kWave);
    count += __shfl_xor(count, off, kWave);
  }
  if ((threadIdx.x & (kWave - 1)) == 0) {
    lds[threadIdx.x / kWave] = sum;
    lds[kWaves + threadIdx.x / kWave] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) {
      sum += lds[w];
      count += lds[kWaves + w];
    }
    double *out = partial + 2 * ((size_t)blockIdx.y * gridDim.x + blockIdx.x);
    out[0] = sum;
    out[1] = count;
  }
}

__global__ __launch_bounds__(kWave) void RowSumKernel(const double *__restrict__ partial, int chunks, int mean, float factor,
                                                      float *__restrict__ sums, float *__restrict__ inverse_count) {
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
  if (threadIdx.x == 0) {
    count = count > 1 ? count : 1;
    sums[blockIdx.x] = (float)(sum * factor / (mean ? count : 1.0));
    if (inverse_count != nullptr) inverse_count[blockIdx.x] = (float)(1.0 / count);
  }
}

__global__ void PrunedMaskKernel(const int64_t *__restrict__ ranges, const int64_t *__restrict__ boundary,
                                 uint8_t *__restrict__ mask, int Tn, int R, long long rows) {
  const long long row = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= rows) return;
  const long long frame = row / R;
  const int64_t b = frame / Tn, t = frame - b * Tn, s = ranges[row];
  mask[row] = t >= boundary[4 * b + 1] && t < boundary[4 * b + 3] && s >= boundary[4 * b] && s <= boundary[4 * b + 2];
}

template <typename T>
int Forward(const void *logits, long long row_stride, const float *top_logprobs, const int64_t *top_tokens,
            const uint8_t *mask, float *row_losses, float *records, long long rows, int C, int K, int rest,
            float temperature, hipStream_t stream) {
  const float c = (float)(kLog2E / (double)temperature);
  const dim3 grid((unsigned)rows), block(kThreads);
  if (rest)
    hipLaunchKernelGGL((DistillForwardKernel<T, true>), grid, block, 0, stream, (const T *)logits, row_stride, top_logprobs,
                       top_tokens, mask, row_losses, records, C, K, c, (float)(1.0 / (double)temperature));
  else
    hipLaunchKernelGGL((DistillForwardKernel<T, false>), grid, block, 0, stream, (const T *)logits, row_stride, top_logprobs,
                       top_tokens, mask, row_losses, records, C, K, c, (float)(1.0 / (double)temperature));
  return LaunchStatus();
}

template <typename T>
int Backward(const void *logits, long long row_stride, const float *top_logprobs, const int64_t *top_tokens,
             const float *records, LossScale scale, void *logits_grad, long long rows, int C, int K,
             int rest, float temperature, hipStream_t stream) {
  const float c = (float)(kLog2E / (double)temperature);
  const dim3 grid((unsigned)rows), block(kThreads);
  if (rest)
    hipLaunchKernelGGL((DistillBackwardKernel<T, true>), grid, block, 0, stream, (const T *)logits, row_stride, top_logprobs,
                       top_tokens, records, scale, (T *)logits_grad, C, K, c);
  else
    hipLaunchKernelGGL((DistillBackwardKernel<T, false>), grid, block, 0, stream, (const T *)logits, row_stride, top_logprobs,
                       top_tokens, records, scale, (T *)logits_grad, C, K, c);
  return LaunchStatus();
}

long long SumChunks(long long rows_per_sum) { return (rows_per_sum + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace k2amd

using namespace k2amd;

extern "C" {

int k2amd_distillation_forward(const void *logits, long long row_stride, const float *top_logprobs,
                               const int64_t *top_tokens, const uint8_t *mask, float *row_losses, float *records,
                               long long rows, int C, int K, int rest, float temperature, int dtype, void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || K < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows, C) || K > kMaxTeacher) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || row_losses == nullptr || (K > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return K2AMD_ERR_INVALID_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32)
    return Forward<float>(logits, row_stride, top_logprobs, top_tokens, mask, row_losses, records, rows, C, K, rest, temperature, st);
  if (dtype == K2AMD_F16)
    return Forward<Half>(logits, row_stride, top_logprobs, top_tokens, mask, row_losses, records, rows, C, K, rest, temperature, st);
  return Forward<Bfloat>(logits, row_stride, top_logprobs, top_tokens, mask, row_losses, records, rows, C, K, rest, temperature, st);
}

int k2amd_distillation_backward(const void *logits, long long row_stride, const float *top_logprobs,
                                const int64_t *top_tokens, const float *records, const float *loss_grad, long long rows_per_loss, const float *inverse_count, float factor,
                                void *logits_grad, long long rows, int C, int K, int rest, float temperature, int dtype,
                                void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || K < 0 || rows_per_loss < 1) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows, C) || K > kMaxTeacher) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || records == nullptr || loss_grad == nullptr || logits_grad == nullptr ||
      (K > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return K2AMD_ERR_INVALID_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const LossScale scale{loss_grad, rows_per_loss, inverse_count, (float)((double)factor / (double)temperature)};
  if (dtype == K2AMD_F32)
    return Backward<float>(logits, row_stride, top_logprobs, top_tokens, records, scale, logits_grad, rows, C, K, rest, temperature, st);
  if (dtype == K2AMD_F16)
    return Backward<Half>(logits, row_stride, top_logprobs, top_tokens, records, scale, logits_grad, rows, C, K, rest, temperature, st);
  return Backward<Bfloat>(logits, row_stride, top_logprobs, top_tokens, records, scale, logits_grad, rows, C, K, rest, temperature, st);
}

size_t k2amd_distillation_sum_scratch_bytes(long long sums, long long rows_per_sum) {
  if (sums < 0 || rows_per_sum < 0) return 0;
  return (size_t)sums * (size_t)SumChunks(rows_per_sum) * 2 * sizeof(double);
}

int k2amd_distillation_sum(const float *row_losses, const uint8_t *mask, float *sums, float *inverse_count,
                           long long num_sums, long long rows_per_sum, int mean, float factor, void *scratch,
                           size_t scratch_bytes, void *stream) {
  if (num_sums < 0 || rows_per_sum < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (num_sums > 65535 || SumChunks(rows_per_sum) > (1 << 20)) return K2AMD_ERR_UNSUPPORTED;
  if (num_sums == 0) return K2AMD_OK;
  if (sums == nullptr || (rows_per_sum > 0 && row_losses == nullptr)) return K2AMD_ERR_INVALID_ARGUMENT;
  if (scratch_bytes < k2amd_distillation_sum_scratch_bytes(num_sums, rows_per_sum) || (rows_per_sum > 0 && scratch == nullptr))
    return K2AMD_ERR_WORKSPACE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int chunks = (int)SumChunks(rows_per_sum);
  if (chunks > 0)
    hipLaunchKernelGGL(RowChunkSumKernel, dim3((unsigned)chunks, (unsigned)num_sums), dim3(kThreads), 0, st, row_losses, mask,
                       rows_per_sum, (double *)scratch);
  hipLaunchKernelGGL(RowSumKernel, dim3((unsigned)num_sums), dim3(kWave), 0, st, (const double *)scratch, chunks, mean, factor,
                     sums, inverse_count);
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
