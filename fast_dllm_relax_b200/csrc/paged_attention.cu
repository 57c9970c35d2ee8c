// Attention over a paged 8-bit KV cache (fdllm_paged_attention) on CUDA cores, for fp32 queries.  Reference
// semantics: runtime.py:63-73 (every query row attends the cached rows), with the cache's values code * scale.
//
// One CTA of four warps per (token row, query head); the warps take the keys 32 at a time in turn.  A lane scores
// one key (the query is in shared memory, the key's row 16 bytes a load), the warp moves its running maximum m and
// sum l once per 32 keys, and then a lane holds HD / 32 of the head's columns:
//   s_t = scale (q . k_t),  o = o 2^(m - m') + sum_t 2^(s_t - m') v_t   (base-2 exponents, fp32)
// with the 32 value rows' loads in flight together.  The warps' (m, l, o) are joined through shared memory.
// Bound by latency at the sizes it serves (parity checks): 4 requests of 8 to 32 rows over 65 to 515 keys, 4/2 heads
// of 64, take 16.5 us; one key at a time with the warp's lanes over its columns took 89.
#include "paged.h"

namespace fdllm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// W consecutive codes at p, widened.
template <int W>
__device__ __forceinline__ void load_codes(const uint8_t* p, float* x) {
  if constexpr (W == 4) {
    const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(p));
    const float2 a = f32x2_from_e4m3x2(static_cast<uint16_t>(u)), b = f32x2_from_e4m3x2(static_cast<uint16_t>(u >> 16));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  } else if constexpr (W == 2) {
    const float2 a = f32x2_from_e4m3x2(__ldg(reinterpret_cast<const uint16_t*>(p)));
    x[0] = a.x, x[1] = a.y;
  } else {
    x[0] = f32x2_from_e4m3x2(__ldg(p)).x;
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_simt_kernel(const PagedAttnArgs a) {
  constexpr int W = HD / 32;
  __shared__ float sm[4], sl[4], so[4][HD];
  __shared__ alignas(16) float sq[HD];
  pdl_trigger();
  pdl_wait();
  const int tok = blockIdx.x, head = blockIdx.y, kvh = head / (a.hq / a.hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int req = paged_req_of(a.reqs, a.n, tok);
  const PagedReq r = a.reqs[req];
  const int lim = paged_key_limit(r.len, r.start + tok - r.tok0, a.causal_block);
  const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(tok) * a.ldq + head * HD;
  for (int d = threadIdx.x; d < HD; d += blockDim.x) sq[d] = to_f<T>(q[d]) * a.scale * kLog2e;
  __syncthreads();
  float o[W], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] = 0.f;
  const int* table = a.table + static_cast<size_t>(req) * a.table_ld;
  for (int c0 = 32 * warp; c0 < lim; c0 += 128) {
    const int key = min(c0 + lane, lim - 1);  // lanes past the range repeat its last key, with weight 0
    const int id = max(paged_page_id(table[key >> a.page_shift], a.pages, a.err), 0);
    const int unit = id * a.hkv + kvh;
    const uint8_t* kp = a.k + ((static_cast<size_t>(unit) << a.page_shift) + (key & (a.page_size - 1))) * HD;
    uint4 u[HD / 16];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(kp) + i);
    const float ks = __ldg(a.k_scale + unit), vs = __ldg(a.v_scale + unit);
    // the value rows: this half-warp's 16 keys are in one page
    float v[32][W];
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const int ut = __shfl_sync(0xffffffffu, unit, t), kt = min(c0 + t, lim - 1);
      load_codes<W>(a.v + ((static_cast<size_t>(ut) << a.page_shift) + (kt & (a.page_size - 1))) * HD + lane * W, v[t]);
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 qv = *reinterpret_cast<const float4*>(&sq[16 * i + 4 * j]);
        const float2 x = f32x2_from_e4m3x2(static_cast<uint16_t>(w[j])), y = f32x2_from_e4m3x2(static_cast<uint16_t>(w[j] >> 16));
        s0 = fmaf(x.x, qv.x, s0);
        s1 = fmaf(x.y, qv.y, s1);
        s0 = fmaf(y.x, qv.z, s0);
        s1 = fmaf(y.y, qv.w, s1);
      }
    }
    const float s = c0 + lane < lim ? (s0 + s1) * ks : -INFINITY;
    float mx = s;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float m2 = fmaxf(m, mx), c = exp2f(m - m2), p = exp2f(s - m2), pv = s == -INFINITY ? 0.f : p * vs;
    l = l * c + p;
    m = m2;
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] *= c;
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const float pt = __shfl_sync(0xffffffffu, pv, t);
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = fmaf(pt, v[t][i], o[i]);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < W; ++i) so[warp][lane * W + i] = o[i];
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
