// Log-probs of given tokens, entropy and the most likely alternatives of rows of logits, and the gradient of all three
// (k2amd_token_logprobs_forward / _backward).
//
//   log p_i = (x_i - m) / tau - log s,   H = -sum_i p_i log p_i,   alternatives: the k largest logits
//   dx_i = 1/tau [ sum_{j: c_j = i} g_j - p_i sum_j g_j - gH p_i (log p_i + H) ]
//
// with c_j the given tokens and the alternatives together and g_j what reaches their log-probs.
#include "token_rows.h"

namespace k2amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

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
__device__ __forceinline__ unsigned long long BlockMaxKey(unsigned long long v, unsigned long long *lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, kWave));
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) v = max(v, lds[w]);
  return v;
}

// One workgroup a row: a pass for the maximum, one for the sums, one for each alternative.
template <typename T>
__global__ __launch_bounds__(kThreads) void TokenForwardKernel(
    const T *__restrict__ logits, long long row_stride, const int64_t *__restrict__ tokens,
    const uint8_t *__restrict__ mask, float *__restrict__ logprobs, float *__restrict__ entropy,
    float *__restrict__ top_logprobs, int64_t *__restrict__ top_tokens, float *__restrict__ stats, int C, int n, int k,
    float c, float inv_tau) {
  __shared__ float lds[kWaves];
  __shared__ unsigned long long lds_key[kWaves];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x;
  if (mask != nullptr && mask[row] == 0) {
    if (tid < n) logprobs[row * n + tid] = 0.0f;
    if (tid < k) {
      top_logprobs[row * k + tid] = Real<float>::NegInf();
      top_tokens[row * k + tid] = -1;
    }
    if (tid == 0 && entropy != nullptr) entropy[row] = 0.0f;
    if (tid == 0 && stats != nullptr) stats[2 * row] = stats[2 * row + 1] = 0.0f;
    return;
  }
  const T *x = logits + row * row_stride;
  float m = Real<float>::NegInf();
  for (int i = tid; i < C; i += kThreads) m = fmaxf(m, ToFloat(x[i]));
  m = BlockMax(m, lds);
  if (m == Real<float>::NegInf()) m = 0.0f;
  float s = 0.0f, t = 0.0f;
  for (int i = tid; i < C; i += kThreads) {
    const float d = (ToFloat(x[i]) - m) * c, e = Exp2(d);
    s += e;
    t += fmaxf(d, kNothing) * e;
  }
  s = BlockSum(s, lds);
  t = BlockSum(t, lds);
  const float ls = Log2(s);
  if (tid < n) {
    const int64_t token = tokens[row * n + tid];
    float lp = 0.0f;
    if (token >= C) lp = __uint_as_float(0x7fc00000u);
    else if (token >= 0) lp = LogProb(ToFloat(x[token]), m, ls, inv_tau);
    logprobs[row * n + tid] = lp;
  }
  if (tid == 0 && entropy != nullptr) entropy[row] = s == 0.0f ? 0.0f : kLn2 * (ls - t / s);
  if (tid == 0 && stats != nullptr) {
    stats[2 * row] = m;
    stats[2 * row + 1] = ls;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int i = tid; i < C; i += kThreads) {
      const unsigned long long key = KeyOf(ToFloat(x[i]), (unsigned)i);
      if (key < last) best = max(best, key);
    }
    last = BlockMaxKey(best, lds_key);
    if (tid == 0) {
      const bool some = last != 0;
      top_logprobs[row * k + j] = some ? LogProb(ToFloat(x[IndexOf(last)]), m, ls, inv_tau) : Real<float>::NegInf();
      top_tokens[row * k + j] = some ? (int64_t)IndexOf(last) : -1;
    }
  }
}

// One workgroup a row: the softmax part of every element, then the entries' own elements over it.
template <typename T>
__global__ __launch_bounds__(kThreads) void TokenBackwardKernel(
    const T *__restrict__ logits, long long row_stride, const int64_t *__restrict__ tokens,
    const uint8_t *__restrict__ mask, const float *__restrict__ stats, const float *__restrict__ entropy,
    const int64_t *__restrict__ top_tokens, const float *__restrict__ logprobs_grad,
    const float *__restrict__ entropy_grad, const float *__restrict__ top_grad, T *__restrict__ logits_grad, int C, int n,
    int k, float c, float inv_tau) {
  __shared__ int entry[kMaxTokens + kMaxTop];
  __shared__ float entry_grad[kMaxTokens + kMaxTop];
  __shared__ float lds[kWaves];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x;
  T *dx = logits_grad + row * C;
  if (mask != nullptr && mask[row] == 0) {
    for (int i = tid; i < C; i += kThreads) FromFloat(0.0f, &dx[i]);
    return;
  }
  const T *x = logits + row * row_stride;
  const int used = (logprobs_grad != nullptr ? n : 0), both = used + (top_grad != nullptr ? k : 0);
  float g = 0.0f;
  if (tid < both) {
    int64_t token;
    if (tid < used) {
      token = tokens[row * n + tid];
      g = logprobs_grad[row * n + tid];
    } else {
      token = top_tokens[row * k + (tid - used)];
      g = top_grad[row * k + (tid - used)];
    }
    if (token < 0) g = 0.0f;
    if (token >= C) g = __uint_as_float(0x7fc00000u);
    entry[tid] = token < 0 || token >= C ? -1 : (int)token;
    entry_grad[tid] = g;
  }
  const float sum = BlockSum(g, lds);
  const float m = stats[2 * row], ls = stats[2 * row + 1];
  const float h = entropy_grad != nullptr ? entropy[row] : 0.0f, gh = entropy_grad != nullptr ? entropy_grad[row] : 0.0f;
  const float none = ls == Real<float>::NegInf() ? 0.0f : 1.0f;  // a row without any mass: every p is 0
  auto softmax_part = [&](float xi) {
    const float d = fmaxf((xi - m) * c, kNothing) - (none != 0.0f ? ls : 0.0f);
    const float p = none * Exp2(d);
    return -p * (sum + gh * (kLn2 * d + h));
  };
  for (int i = tid; i < C; i += kThreads) FromFloat(softmax_part(ToFloat(x[i])) * inv_tau, &dx[i]);
  __syncthreads();
  if (tid < both && entry[tid] >= 0) {
    float own = 0.0f;
    for (int j = 0; j < both; ++j)
      if (entry[j] == entry[tid]) own += entry_grad[j];
    FromFloat((softmax_part(ToFloat(x[entry[tid]])) + own) * inv_tau, &dx[entry[tid]]);
  }
}

template <typename T>
int Forward(const void *logits, long long row_stride, const int64_t *tokens, const uint8_t *mask, float *logprobs,
            float *entropy, float *top_logprobs, int64_t *top_tokens, float *stats, long long rows, int C, int n, int k,
            float temperature, hipStream_t stream) {
  hipLaunchKernelGGL((TokenForwardKernel<T>), dim3((unsigned)rows), dim3(kThreads), 0, stream, (const T *)logits, row_stride,
                     tokens, mask, logprobs, entropy, top_logprobs, top_tokens, stats, C, n, k,
                     (float)(kLog2E / (double)temperature), (float)(1.0 / (double)temperature));
  return LaunchStatus();
}

template <typename T>
int Backward(const void *logits, long long row_stride, const int64_t *tokens, const uint8_t *mask, const float *stats,
             const float *entropy, const int64_t *top_tokens, const float *logprobs_grad, const float *entropy_grad,
             const float *top_grad, void *logits_grad, long long rows, int C, int n, int k, float temperature,
             hipStream_t stream) {
  hipLaunchKernelGGL((TokenBackwardKernel<T>), dim3((unsigned)rows), dim3(kThreads), 0, stream, (const T *)logits, row_stride,
                     tokens, mask, stats, entropy, top_tokens, logprobs_grad, entropy_grad, top_grad, (T *)logits_grad, C, n,
                     k, (float)(kLog2E / (double)temperature), (float)(1.0 / (double)temperature));
  return LaunchStatus();
}

}  // namespace
}  // namespace k2amd

using namespace k2amd;

extern "C" {

int k2amd_token_logprobs_forward(const void *logits, long long row_stride, const int64_t *tokens, const uint8_t *mask,
                                 float *logprobs, float *entropy, float *top_logprobs, int64_t *top_tokens, float *stats,
                                 long long rows, int C, int n, int k, float temperature, int dtype, void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || n < 0 || k < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows) || n > kMaxTokens || k > kMaxTop) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || (n > 0 && (tokens == nullptr || logprobs == nullptr)) ||
      (k > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
    return K2AMD_ERR_INVALID_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32)
    return Forward<float>(logits, row_stride, tokens, mask, logprobs, entropy, top_logprobs, top_tokens, stats, rows, C, n, k, temperature, st);
  if (dtype == K2AMD_F16)
    return Forward<Half>(logits, row_stride, tokens, mask, logprobs, entropy, top_logprobs, top_tokens, stats, rows, C, n, k, temperature, st);
  return Forward<Bfloat>(logits, row_stride, tokens, mask, logprobs, entropy, top_logprobs, top_tokens, stats, rows, C, n, k, temperature, st);
}

int k2amd_token_logprobs_backward(const void *logits, long long row_stride, const int64_t *tokens, const uint8_t *mask,
                                  const float *stats, const float *entropy, const int64_t *top_tokens,
                                  const float *logprobs_grad, const float *entropy_grad, const float *top_grad,
                                  void *logits_grad, long long rows, int C, int n, int k, float temperature, int dtype,
                                  void *stream) {
  if (!RowsOk(rows, row_stride, C, temperature, dtype) || n < 0 || k < 0) return K2AMD_ERR_INVALID_ARGUMENT;
  if (!RowsServed(rows) || n > kMaxTokens || k > kMaxTop) return K2AMD_ERR_UNSUPPORTED;
  if (rows == 0) return K2AMD_OK;
  if (logits == nullptr || stats == nullptr || logits_grad == nullptr || (n > 0 && logprobs_grad != nullptr && tokens == nullptr) ||
      (k > 0 && top_grad != nullptr && top_tokens == nullptr) || (entropy_grad != nullptr && entropy == nullptr))
    return K2AMD_ERR_INVALID_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == K2AMD_F32)
    return Backward<float>(logits, row_stride, tokens, mask, stats, entropy, top_tokens, logprobs_grad, entropy_grad, top_grad, logits_grad, rows, C, n, k, temperature, st);
  if (dtype == K2AMD_F16)
    return Backward<Half>(logits, row_stride, tokens, mask, stats, entropy, top_tokens, logprobs_grad, entropy_grad, top_grad, logits_grad, rows, C, n, k, temperature, st);
  return Backward<Bfloat>(logits, row_stride, tokens, mask, stats, entropy, top_tokens, logprobs_grad, entropy_grad, top_grad, logits_grad, rows, C, n, k, temperature, st);
}

}  // extern "C"
