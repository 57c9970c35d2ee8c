// Appending keys and values to a paged 8-bit cache, with the position rotation applied on the way
// (fdllm_paged_append): no counterpart in the reference, whose callback writes rotated K/V rows into a
// contiguous buffer (runtime.py:51-60); the rotation is model/cuda.py:303-316 in fp32.
//
//   k'   = (k1 cos - k2 sin, k2 cos + k1 sin)             halves of a head, fp32
//   s    = max(2^e, s_old if the page keeps rows)         per page and head; 2^e the least power of two
//                                                         (e >= -64) with max |finite new value| <= 448 2^e
//   code = e4m3(value / s),  kept codes = e4m3(code_old * s_old / s)
//
// A power of two makes both divisions exact, so a value is rounded once, and a kept code only loses
// bits where it becomes subnormal.
#include "paged.h"

namespace fdllm {

namespace {

constexpr int kMinScaleExp = -64;

// The least e >= kMinScaleExp with amax <= 448 * 2^e, for finite amax >= 0: amax = m 2^x, 448 = 1.75 2^8.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int x = static_cast<int>(b >> 23) - 127;  // -127 for zero and subnormals: clamped below
  const int e = x - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return max(e, kMinScaleExp);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // NaN and infinities do not move the scale
}

template <typename TT>
__device__ __forceinline__ float table_at(const void* t, size_t i) { return to_f<TT>(static_cast<const TT*>(t)[i]); }

// Value d of the rotated (or plain, V) row.
template <typename T, typename TT>
__device__ __forceinline__ float new_value(const T* row, int d, int hd, bool rotate, const PagedAppendArgs& a, int pos) {
  const float x = to_f<T>(row[d]);
  if (!rotate) return x;
  const int half = hd >> 1, i = d < half ? d : d - half;
  const size_t at = static_cast<size_t>(pos) * half + i;
  const float c = table_at<TT>(a.cos, at), s = table_at<TT>(a.sin, at);
  const float y = to_f<T>(row[d < half ? d + half : d - half]);
  return d < half ? x * c - y * s : x * c + y * s;
}

// One CTA per (page unit, KV head, K or V), then one per token row for the queries.
template <typename T, typename TT>
__global__ void __launch_bounds__(128) paged_append_kernel(const PagedAppendArgs a) {
  __shared__ float red[4];
  pdl_trigger();
  pdl_wait();
  const int hd = a.hd;
  const int kv_blocks = a.n_units * a.hkv * 2;
  if (static_cast<int>(blockIdx.x) >= kv_blocks) {  // queries
    const int tok = blockIdx.x - kv_blocks;
    const PagedReq r = a.reqs[paged_req_of(a.reqs, a.n, tok)];
    const int pos = r.start + tok - r.tok0;
    const T* src = static_cast<const T*>(a.q_in) + static_cast<size_t>(tok) * a.ldq;
    T* dst = static_cast<T*>(a.q_out) + static_cast<size_t>(tok) * a.hq * hd;
    for (int i = threadIdx.x; i < a.hq * hd; i += blockDim.x)
      dst[i] = from_f<T>(new_value<T, TT>(src + i / hd * hd, i % hd, hd, true, a, pos));
    return;
  }
  const int is_v = blockIdx.x & 1, head = (blockIdx.x >> 1) % a.hkv;
  const PagedPageUnit u = a.units[(blockIdx.x >> 1) / a.hkv];
  const PagedReq r = a.reqs[u.req];
  const int id = paged_page_id(a.table[static_cast<size_t>(u.req) * a.table_ld + u.slot], a.pages, a.err);
  if (id < 0) return;
  const int ps = a.page_size, base = u.slot * ps;
  const int w0 = max(r.start - base, 0), w1 = min(r.start + r.rows - base, ps);  // page rows written
  const int live = min(max(r.live - base, 0), ps);                                // page rows that held values
  const size_t unit = static_cast<size_t>(id) * a.hkv + head;
  uint8_t* codes = (is_v ? a.v : a.k) + unit * ps * hd;
  float* scale = (is_v ? a.v_scale : a.k_scale) + unit;
  const int ld = is_v ? a.ldv : a.ldk;
  const T* src = static_cast<const T*>(is_v ? a.v_in : a.k_in) +
                 static_cast<size_t>(r.tok0 + base + w0 - r.start) * ld + head * hd;
  const int nw = (w1 - w0) * hd, pos0 = base + w0;

  float amax = 0.f;
  for (int i = threadIdx.x; i < nw; i += blockDim.x)
    amax = fmaxf(amax, finite_abs(new_value<T, TT>(src + static_cast<size_t>(i / hd) * ld, i % hd, hd, !is_v, a, pos0 + i / hd)));
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  const float s_old = *scale;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const bool keeps = w0 > 0 || live > w1;  // rows below w0 held values: start <= live
  float s = pow2f(scale_exponent(amax));
  if (keeps && s_old > s) s = s_old;
  const float inv = 1.f / s;
  if (threadIdx.x == 0) *scale = s;
  for (int i = threadIdx.x; i < nw; i += blockDim.x) {
    const float x = new_value<T, TT>(src + static_cast<size_t>(i / hd) * ld, i % hd, hd, !is_v, a, pos0 + i / hd);
    codes[w0 * hd + i] = static_cast<uint8_t>(e4m3x2_from_f32(x * inv, 0.f) & 0xFF);
  }
  if (keeps && s != s_old) {
    const float f = s_old / s;
    const int n0 = w0 * hd, n1 = max(live - w1, 0) * hd;
    for (int i = threadIdx.x; i < n0 + n1; i += blockDim.x) {
      uint8_t* c = codes + (i < n0 ? i : w1 * hd + i - n0);
      *c = static_cast<uint8_t>(e4m3x2_from_f32(f32x2_from_e4m3x2(*c).x * f, 0.f) & 0xFF);
    }
  }
}

}  // namespace

int launch_paged_append(const PagedAppendArgs& a, int dtype, cudaStream_t s) {
  const int grid = a.n_units * a.hkv * 2 + (a.q_in != nullptr ? a.total_rows : 0);
  if (dtype == 1)
    return a.table_f32 ? launch_k(paged_append_kernel<bf16, float>, dim3(grid), dim3(128), 0, s, a)
                       : launch_k(paged_append_kernel<bf16, bf16>, dim3(grid), dim3(128), 0, s, a);
  return launch_k(paged_append_kernel<float, float>, dim3(grid), dim3(128), 0, s, a);
}

}  // namespace fdllm
