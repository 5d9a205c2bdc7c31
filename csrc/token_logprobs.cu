// Log-probability of a given token, entropy and the most likely tokens of each
// row of logits.
//
//   m = max x,  Z = sum e^(x - m),  S = sum e^(x - m) (x - m)
//   logprob = x[id] - m - log Z,    entropy = log Z - S / Z
//
// A term with e^(x - m) = 0 adds nothing to S (x = -inf included). A row
// without a finite maximum (all -inf, a +inf or a NaN) has no distribution:
// its log-probabilities and entropy are NaN. In the order of the top tokens a
// NaN counts as larger than every number; equal logits go by index.

#include "ragged.cuh"

namespace afd {

namespace {

constexpr int kThreads = 256;

// Floats in an order that unsigned integers have, NaN last.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float block_sum(float v, float* sh) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  float r = 0.f;
  for (int w = 0; w < kThreads / 32; ++w) r += sh[w];
  return r;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v,
                                                        unsigned long long* sh) {
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  unsigned long long r = 0;
  for (int w = 0; w < kThreads / 32; ++w) r = max(r, sh[w]);
  return r;
}

// One CTA per row, and one more pass over the row per top token.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(TokenLogprobsArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ float fsh[kThreads / 32];
  __shared__ unsigned long long ush[kThreads / 32];
  const int r = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)r * a.row;
  auto key = [&](int i) {
    return ((unsigned long long)order_of(to_f(x[i])) << 32) | (uint32_t)~i;
  };
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < a.V; i += kThreads) best = max(best, key(i));
  best = block_max(best, ush);
  const float m = to_f(x[~(uint32_t)best]);
  const bool none = !(m > -INFINITY && m < INFINITY);
  float z = 0.f, s = 0.f;
  for (int i = threadIdx.x; i < a.V; i += kThreads) {
    const float d = to_f(x[i]) - m, e = expf(d);
    z += e;
    s += e > 0.f ? e * d : 0.f;
  }
  z = block_sum(z, fsh);
  s = block_sum(s, fsh);
  const float lz = logf(z);
  if (threadIdx.x == 0) {
    const int64_t id = a.ids[r];
    const bool ok = !none && id >= 0 && id < a.V;
    a.logprob[r] = ok ? to_f(x[id]) - m - lz : NAN;
    a.entropy[r] = none ? NAN : lz - s / z;
  }
  for (int k = 0; k < a.top_k; ++k) {
    if (threadIdx.x == 0) {
      const uint32_t i = ~(uint32_t)best;
      a.top_ids[(size_t)r * a.top_k + k] = i;
      a.top_logprobs[(size_t)r * a.top_k + k] = none ? NAN : to_f(x[i]) - m - lz;
    }
    unsigned long long next = 0;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const unsigned long long c = key(i);
      if (c < best) next = max(next, c);
    }
    best = block_max(next, ush);
  }
}

}  // namespace

int launch_token_logprobs(const TokenLogprobsArgs& a, cudaStream_t s) {
  if (a.R == 0) return 0;
  const dim3 grid((unsigned)a.R);
  cudaError_t e;
  if (a.elem == kElemBf16)
    e = launch_k(token_logprobs_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, s, a);
  else if (a.elem == kElemF16)
    e = launch_k(token_logprobs_kernel<__half>, grid, dim3(kThreads), 0, s, a);
  else
    e = launch_k(token_logprobs_kernel<float>, grid, dim3(kThreads), 0, s, a);
  return e == cudaSuccess ? 0 : 4000 + (int)e;
}

}  // namespace afd
