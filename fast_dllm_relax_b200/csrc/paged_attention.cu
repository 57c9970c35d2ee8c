// Attention over a paged 8-bit KV cache (fdllm_paged_attention) on CUDA cores, for fp32 queries.  Reference semantics: runtime.py:63-73 (every query row attends the cached rows), with the
// cache's values code * scale.
//
// One CTA of four warps per (token row, query head).  Each warp walks its share of the keys with the
// running maximum m and sum l of the softmax, a lane holding HD / 32 of the head's columns:
//   s_t = scale (q . k_t),  o = o 2^(m - m') + 2^(s_t - m') v_t   (base-2 exponents, fp32)
// and the warps' (m, l, o) are joined through shared memory.
#include "paged.h"

namespace fdllm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_simt_kernel(const PagedAttnArgs a) {
  constexpr int W = HD / 32;
  __shared__ float sm[4], sl[4], so[4][HD];
  pdl_trigger();
  pdl_wait();
  const int tok = blockIdx.x, head = blockIdx.y, kvh = head / (a.hq / a.hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int req = paged_req_of(a.reqs, a.n, tok);
  const PagedReq r = a.reqs[req];
  const int lim = paged_key_limit(r.len, r.start + tok - r.tok0, a.causal_block);
  const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(tok) * a.ldq + head * HD;
  float qr[W], o[W], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    qr[i] = to_f<T>(q[lane + 32 * i]) * a.scale * kLog2e;
    o[i] = 0.f;
  }
  for (int t = warp; t < lim; t += 4) {
    const int id = max(paged_page_id(a.table[static_cast<size_t>(req) * a.table_ld + t / a.page_size], a.pages, a.err), 0);
    const size_t unit = static_cast<size_t>(id) * a.hkv + kvh;
    const size_t row = (unit * a.page_size + t % a.page_size) * HD;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += qr[i] * f32x2_from_e4m3x2(a.k[row + lane + 32 * i]).x;
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.k_scale[unit];
    const float m2 = fmaxf(m, s), c = exp2f(m - m2), p = exp2f(s - m2), pv = p * a.v_scale[unit];
    l = l * c + p;
    m = m2;
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] = o[i] * c + pv * f32x2_from_e4m3x2(a.v[row + lane + 32 * i]).x;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < W; ++i) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  for (int d = threadIdx.x; d < HD; d += blockDim.x) {
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - mx);
      num += f * so[w][d];
      den += f * sl[w];
    }
    static_cast<T*>(a.out)[(static_cast<size_t>(tok) * a.hq + head) * HD + d] = from_f<T>(den > 0.f ? num / den : 0.f);
  }
}

template <typename T>
int launch_simt(const PagedAttnArgs& a, cudaStream_t s) {
  const dim3 grid(a.total_rows, a.hq);
  switch (a.hd) {
    case 32: return launch_k(paged_attn_simt_kernel<T, 32>, grid, dim3(128), 0, s, a);
    case 64: return launch_k(paged_attn_simt_kernel<T, 64>, grid, dim3(128), 0, s, a);
    default: return launch_k(paged_attn_simt_kernel<T, 128>, grid, dim3(128), 0, s, a);
  }
}

}  // namespace

int launch_paged_attention_simt(const PagedAttnArgs& a, cudaStream_t s) { return launch_simt<float>(a, s); }

}  // namespace fdllm
