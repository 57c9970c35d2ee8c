// Attention over a paged 8-bit KV cache (fdllm_paged_attention) on CUDA cores, for fp32 queries.  Reference
// semantics: runtime.py:63-73 (every query row attends the cached rows), with the cache's values code * scale.
//
// One CTA of eight warps per token row and up to four query heads of a KV head, which share the widening of its codes;
// the warps take the keys 32 at a time in turn.  A lane scores one key (the queries are in shared memory, the key's row
// 16 bytes a load), the warp moves its running maximum m and sum l of a head once per 32 keys, and then a lane holds
// HD / 32 of the heads' columns:
//   s_t = scale (q . k_t),  o = o 2^(m - m') + sum_t 2^(s_t - m') v_t   (base-2 exponents, fp32)
// with the 32 value rows' loads in flight together.  The warps' (m, l, o) are joined through shared memory.
// Bound by latency at the sizes it serves (parity checks): 4 requests of 8 to 32 rows over 65 to 515 keys, 4/2 heads of
// 64, take 10.3 us (a CTA of four warps a query head: 16.5), 3 of 32 rows over up to 609 keys, 12/2 heads of 128, 21.7
// (34.2).
#include "paged.h"

namespace fdllm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;

// W consecutive codes, and the same widened.
template <int W>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p) {
  if constexpr (W == 4) return __ldg(reinterpret_cast<const uint32_t*>(p));
  else if constexpr (W == 2) return __ldg(reinterpret_cast<const uint16_t*>(p));
  else return __ldg(p);
}
template <int W>
__device__ __forceinline__ void widen(uint32_t u, float* x) {
  const float2 a = f32x2_from_e4m3x2(static_cast<uint16_t>(u));
  x[0] = a.x;
  if constexpr (W > 1) x[1] = a.y;
  if constexpr (W > 2) {
    const float2 b = f32x2_from_e4m3x2(static_cast<uint16_t>(u >> 16));
    x[2] = b.x, x[3] = b.y;
  }
}

// NH query heads a CTA.  Past the KV head's last query head a CTA repeats it and writes nothing.
template <int HD, int NH>
__global__ void __launch_bounds__(32 * kWarps, 2) paged_attn_simt_kernel(const PagedAttnArgs a) {
  constexpr int W = HD / 32;
  __shared__ float sm[kWarps][NH], sl[kWarps][NH], so[kWarps][NH][HD];
  __shared__ alignas(16) float sq[NH][HD];
  pdl_trigger();
  pdl_wait();
  const int G = a.hq / a.hkv, sets = (G + NH - 1) / NH;  // CTAs to a KV head
  const int tok = blockIdx.x, kvh = blockIdx.y / sets, head0 = kvh * G + (blockIdx.y - kvh * sets) * NH, end = (kvh + 1) * G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int req = paged_req_of(a.reqs, a.n, tok);
  const PagedReq r = a.reqs[req];
  const int lim = paged_key_limit(r.len, r.start + tok - r.tok0, a.causal_block);
  const float* q = static_cast<const float*>(a.q) + static_cast<size_t>(tok) * a.ldq;
  for (int i = threadIdx.x; i < NH * HD; i += 32 * kWarps) {
    const int h = i / HD, d = i - h * HD;
    sq[h][d] = q[min(head0 + h, end - 1) * HD + d] * a.scale * kLog2e;
  }
  __syncthreads();
  float o[NH][W], m[NH], l[NH];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) o[h][i] = 0.f;
  }
  const int* table = a.table + static_cast<size_t>(req) * a.table_ld;
  for (int c0 = 32 * warp; c0 < lim; c0 += 32 * kWarps) {
    const int key = min(c0 + lane, lim - 1);  // lanes past the range repeat its last key, with weight 0
    const int id = max(paged_page_id(table[key >> a.page_shift], a.pages, a.err), 0);
    const int unit = id * a.hkv + kvh;
    const uint8_t* kp = a.k + ((static_cast<size_t>(unit) << a.page_shift) + (key & (a.page_size - 1))) * HD;
    uint4 u[HD / 16];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(kp) + i);
    const float ks = __ldg(a.k_scale + unit), vs = __ldg(a.v_scale + unit);
    uint32_t v[32];
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const int ut = __shfl_sync(0xffffffffu, unit, t), kt = min(c0 + t, lim - 1);
      v[t] = load_codes<W>(a.v + ((static_cast<size_t>(ut) << a.page_shift) + (kt & (a.page_size - 1))) * HD + lane * W);
    }
    float s0[NH], s1[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) s0[h] = s1[h] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[4];
        widen<4>(w[j], x);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const float4 qv = *reinterpret_cast<const float4*>(&sq[h][16 * i + 4 * j]);
          s0[h] = fmaf(x[0], qv.x, s0[h]);
          s1[h] = fmaf(x[1], qv.y, s1[h]);
          s0[h] = fmaf(x[2], qv.z, s0[h]);
          s1[h] = fmaf(x[3], qv.w, s1[h]);
        }
      }
    }
    float pv[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const float s = c0 + lane < lim ? (s0[h] + s1[h]) * ks : -INFINITY;
      float mx = s;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float m2 = fmaxf(m[h], mx), c = exp2f(m[h] - m2), p = exp2f(s - m2);
      pv[h] = s == -INFINITY ? 0.f : p * vs;
      l[h] = l[h] * c + p;
      m[h] = m2;
#pragma unroll
      for (int i = 0; i < W; ++i) o[h][i] *= c;
    }
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      float x[W];
      widen<W>(v[t], x);
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float pt = __shfl_sync(0xffffffffu, pv[h], t);
#pragma unroll
        for (int i = 0; i < W; ++i) o[h][i] = fmaf(pt, x[i], o[h][i]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
    if (lane == 0) sm[warp][h] = m[h], sl[warp][h] = l[h];
#pragma unroll
    for (int i = 0; i < W; ++i) so[warp][h][lane * W + i] = o[h][i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NH * HD; i += 32 * kWarps) {
    const int h = i / HD, d = i - h * HD;
    if (head0 + h >= end) break;
    float mx = sm[0][h];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm[w][h]);
    float num = 0.f, den = 0.f;  // den: 0 without keys, NaN where a score is not a number
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm[w][h] == -INFINITY ? 0.f : exp2f(sm[w][h] - mx);
      num += f * so[w][h][d];
      den += f * sl[w][h];
    }
    static_cast<float*>(a.out)[(static_cast<size_t>(tok) * a.hq + head0 + h) * HD + d] = den == 0.f ? 0.f : num / den;
  }
}

template <int HD>
int launch_hd(const PagedAttnArgs& a, cudaStream_t s) {
  const int G = a.hq / a.hkv, nh = (G + (G + 3) / 4 - 1) / ((G + 3) / 4);  // as even as sets of up to four come
  const dim3 grid(a.total_rows, a.hkv * ((G + nh - 1) / nh)), block(32 * kWarps);
  switch (nh) {
    case 1: return launch_k(paged_attn_simt_kernel<HD, 1>, grid, block, 0, s, a);
    case 2: return launch_k(paged_attn_simt_kernel<HD, 2>, grid, block, 0, s, a);
    case 3: return launch_k(paged_attn_simt_kernel<HD, 3>, grid, block, 0, s, a);
    default: return launch_k(paged_attn_simt_kernel<HD, 4>, grid, block, 0, s, a);
  }
}

}  // namespace

int launch_paged_attention_simt(const PagedAttnArgs& a, cudaStream_t s) {
  return a.hd == 32 ? launch_hd<32>(a, s) : a.hd == 64 ? launch_hd<64>(a, s) : launch_hd<128>(a, s);
}

}  // namespace fdllm
