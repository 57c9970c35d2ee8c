// Log probabilities of given tokens, with entropy and top alternatives, from logits (fdllm_logprobs);
// the reference reduces logits on the host (runners.py:877-881).  Per row of x, in fp32:
//   m = max x,  S0 = sum e^(x - m),  S1 = sum e^(x - m) (x - m)
//   lse = m + log S0,  logprob = x[target] - lse,  entropy = log S0 - S1 / S0
// and the `top` largest by (value descending, id ascending).
#include "paged.h"

namespace fdllm {

namespace {

// Order of the alternatives as one unsigned key: the value's rank in the high word (NaN as -inf), the
// complemented id in the low word, so that the largest key is the largest value's lowest id.
__device__ __forceinline__ unsigned long long rank_key(float x, int id) {
  uint32_t b = __float_as_uint(x == x ? x + 0.f : -INFINITY);  // + 0: -0 ranks as 0
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | static_cast<uint32_t>(~id);
}

template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const LogprobArgs a) {
  __shared__ float red[3][8];
  __shared__ unsigned long long best[8];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.ld;
  float m = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
    const float v = to_f<T>(x[i]);
    nan |= v != v;
    m = fmaxf(m, v);
  }
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[0][warp] = m;
  nan = __syncthreads_or(nan);
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[0][w]);
  float s0 = 0.f, s1 = 0.f;
  for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
    const float d = to_f<T>(x[i]) - m, e = expf(d);
    s0 += e;
    s1 += e > 0.f ? e * d : 0.f;
  }
  for (int o = 16; o > 0; o >>= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
  }
  if (lane == 0) red[1][warp] = s0, red[2][warp] = s1;
  __syncthreads();
  s0 = s1 = 0.f;
  for (int w = 0; w < 8; ++w) s0 += red[1][w], s1 += red[2][w];
  const bool bad = nan || m == INFINITY || m == -INFINITY;
  const float ls = bad ? NAN : logf(s0), lse = m + ls;
  if (threadIdx.x == 0) {
    if (a.targets != nullptr) {
      const int t = a.targets[row];
      const bool ok = t >= 0 && t < a.vocab;
      if (!ok) report_error(a.err, kErrTokenRange);
      a.logprob[row] = ok ? to_f<T>(x[t]) - lse : NAN;
    }
    if (a.entropy != nullptr) a.entropy[row] = ls - s1 / s0;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long b = 0;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
      const unsigned long long c = rank_key(to_f<T>(x[i]), i);
      if (c < last && c > b) b = c;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long c = __shfl_xor_sync(0xffffffffu, b, o);
      b = c > b ? c : b;
    }
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    for (int w = 0; w < 8; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (threadIdx.x == 0) {
      const int id = static_cast<int>(~static_cast<uint32_t>(b));
      a.top_ids[static_cast<size_t>(row) * a.top + k] = id;
      a.top_logprobs[static_cast<size_t>(row) * a.top + k] = to_f<T>(x[id]) - lse;
    }
  }
}

}  // namespace

int launch_logprobs(const LogprobArgs& a, int dtype, cudaStream_t s) {
  return dtype == 1 ? launch_k(logprobs_kernel<bf16>, dim3(a.rows), dim3(256), 0, s, a)
                    : launch_k(logprobs_kernel<float>, dim3(a.rows), dim3(256), 0, s, a);
}

}  // namespace fdllm
