// Log probabilities of given tokens, entropy and top tokens of logit rows (gfx950).
//
// Mathematics.  With m the largest logit of a row, n how many are equal to it and
// R = sum over the smaller ones of exp(x - m) plus n - 1, log sum exp(x) is m +
// log1p(R): a given token's log probability is (x - m) - log1p(R), the entropy
// log1p(R) + sum (m - x) exp(x - m) / (1 + R), all terms of one sign, so that a
// row that is nearly decided keeps its digits.
#include "w8a8_internal.h"

namespace w8a8 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

template <typename T> __device__ inline float logit(const void* x, int64_t i) {
  if constexpr (std::is_same<T, float>::value)
    return static_cast<const float*>(x)[i];
  else
    return to_f32(static_cast<const T*>(x)[i]);
}

// The order of logits: by value, NaN above all, equal ones by their number.
__device__ inline uint64_t rank_of(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // one zero
  const uint32_t order = x != x ? ~0u : (u >> 31) ? ~u : u | 0x80000000u;
  return static_cast<uint64_t>(order) << 32 | static_cast<uint32_t>(~i);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(TokenLogprobs p) {
  __shared__ float red[3][kWaves];
  __shared__ uint64_t best[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  float top = -INFINITY;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) top = fmaxf(top, logit<T>(x, i));
  for (int w = 1; w < 64; w <<= 1) top = fmaxf(top, __shfl_xor(top, w));
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red[0][w]);
  __syncthreads();
  float sum = 0.0f, spread = 0.0f, equal = 0.0f;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
    const float d = logit<T>(x, i) - top;
    const float e = expf(d);
    if (d == 0.0f) {
      equal += 1.0f;
    } else {
      sum += e;
      spread -= e == 0.0f ? 0.0f : d * e;
    }
  }
  for (int w = 1; w < 64; w <<= 1) {
    sum += __shfl_xor(sum, w);
    spread += __shfl_xor(spread, w);
    equal += __shfl_xor(equal, w);
  }
  if (lane == 0) {
    red[0][wave] = sum;
    red[1][wave] = spread;
    red[2][wave] = equal;
  }
  __syncthreads();
  sum = spread = equal = 0.0f;
  for (int w = 0; w < kWaves; ++w) {
    sum += red[0][w];
    spread += red[1][w];
    equal += red[2][w];
  }
  const float rest = sum + (equal - 1.0f);
  const float norm = equal == 0.0f ? NAN : log1pf(rest);
  if (threadIdx.x == 0 && p.entropy != nullptr) p.entropy[row] = norm + spread / (1.0f + rest);
  for (int i = threadIdx.x; i < p.given; i += kThreads) {
    const int64_t token = p.tokens[row * p.ld_tokens + i];
    float y = token == -1 ? 0.0f : NAN;
    if (token >= 0 && token < p.vocab) y = (logit<T>(x, token) - top) - norm;
    p.logprobs[row * p.given + i] = y;
  }
  uint64_t last = ~uint64_t{0};
  for (int k = 0; k < p.top; ++k) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
      const uint64_t r = rank_of(logit<T>(x, i), i);
      if (r < last && r > mine) mine = r;
    }
    for (int w = 1; w < 64; w <<= 1) mine = max(mine, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(mine), w)));
    __syncthreads();
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) mine = max(mine, best[w]);
    last = mine;
    if (threadIdx.x == 0) {
      const int token = static_cast<int>(~static_cast<uint32_t>(mine));
      p.top_tokens[row * p.top + k] = token;
      p.top_logprobs[row * p.top + k] = (logit<T>(x, token) - top) - norm;
    }
  }
}

}  // namespace

int64_t token_logprobs_workspace(int64_t, int64_t, int64_t, int) { return 0; }

hipError_t launch_token_logprobs(const TokenLogprobs& p, int dtype, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(p.rows));
  if (dtype == kF32)
    hipLaunchKernelGGL((logprobs_kernel<float>), grid, dim3(kThreads), 0, st, p);
  else if (dtype == kF16)
    hipLaunchKernelGGL((logprobs_kernel<__half>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((logprobs_kernel<__hip_bfloat16>), grid, dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace w8a8
