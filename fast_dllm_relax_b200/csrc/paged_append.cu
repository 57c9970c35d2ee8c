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
// bits where it becomes subnormal.  A page that keeps a larger scale of its own, which need not be one (a cache that
// another program filled), takes the rounded quotients.
//
// Bound: HBM (every input read once, every output written once).  One launch, two kinds of CTAs:
//   - a page, KV head and K or V: a thread holds up to two 8-column chunk pairs (K) or four chunks (V) of the
//     page's new rows in registers, so the values are read and rotated once, reduced to the page's maximum across
//     the CTA, and coded from the registers;
//   - up to 16 token rows of one request for the queries: a thread holds its position's 8 cosines and sines and
//     applies them to every head of its share.
// Measured: 8 prompts of 4096 tokens, 12/2 heads of 128, bf16, 254 MB: 50.4 us, 5.0 TB/s; with 84 registers a thread,
// so 640 threads an SM, 55.7.  32 block steps of 32 rows 4.8 us (fp32 8.1), 8 rows inside each of 32 blocks 3.1, one
// token 2.4.
#include <algorithm>

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

// Eight consecutive values, 16-byte aligned (bf16) or 32 bytes in two loads (fp32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<bf16>(const bf16* p, float (&x)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void store8(bf16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// (x, y) = (x cos - y sin, y cos + x sin), eight columns of the two halves.
__device__ __forceinline__ void rotate8(float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i] * c[i] - y[i] * s[i];
    y[i] = y[i] * c[i] + x[i] * s[i];
    x[i] = a;
  }
}

// 1 / s for a power of two; for another scale 1, and the values become their quotients here: by the inverse in 64 bits,
// whose 2^-53 leaves a quotient of few bits, as one half way between two codes is, as it is.
template <int N>
__device__ __forceinline__ float inverse_scale(float s, float (&x)[N][8]) {
  if ((__float_as_uint(s) & 0x7FFFFFu) == 0) return 1.f / s;
  const double inv = 1.0 / s;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[j][i] = static_cast<float>(x[j][i] * inv);
  return 1.f;
}

__device__ __forceinline__ uint2 code8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = e4m3x2_from_f32(x[4 * h] * inv, x[4 * h + 1] * inv) |
           static_cast<uint32_t>(e4m3x2_from_f32(x[4 * h + 2] * inv, x[4 * h + 3] * inv)) << 16;
  return make_uint2(w[0], w[1]);
}

// The new scale of a page from its new rows' maximum (over this thread's part); every thread gets it.
__device__ __forceinline__ float page_scale(float amax, bool keeps, float s_old, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
  amax = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) amax = fmaxf(amax, red[w]);
  const float s = pow2f(scale_exponent(amax));
  return keeps && s_old > s ? s_old : s;
}

// 64 registers: 1024 threads an SM, whose loads cover a unit's own chain of latencies (plan, page id, rows, maximum).
template <typename T, typename TT>
__global__ void __launch_bounds__(512, 2) paged_append_kernel(const PagedAppendArgs a) {
  __shared__ float red[16];
  pdl_trigger();
  pdl_wait();
  const int hd = a.hd, half = hd >> 1, tid = threadIdx.x;
  const int kv_blocks = a.n_units * a.hkv * 2;
  const TT* cos_t = static_cast<const TT*>(a.cos);
  const TT* sin_t = static_cast<const TT*>(a.sin);

  if (static_cast<int>(blockIdx.x) >= kv_blocks) {  // ---- queries
    const PagedPageUnit u = a.q_units[blockIdx.x - kv_blocks];  // (request, first token of it)
    const PagedReq r = a.reqs[u.req];
    const int lanes = half >> 3;                       // threads to a head row: 8 columns of each half
    const int groups = blockDim.x / lanes, g = tid / lanes, d = (tid % lanes) * 8;
    const int n_tok = min(kPagedQTokens, r.rows - u.slot);
    const int split = max(1, groups / n_tok);          // groups to a token, a share of its heads each
    const int step = groups / split;
    if (g >= step * split) return;
    for (int t = g / split; t < n_tok; t += step) {
      const int tok = r.tok0 + u.slot + t;
      const size_t at = static_cast<size_t>(r.start + u.slot + t) * half + d;
      float c[8], s[8];
      load8<TT>(cos_t + at, c);
      load8<TT>(sin_t + at, s);
      const T* src = static_cast<const T*>(a.q_in) + static_cast<size_t>(tok) * a.ldq + d;
      T* dst = static_cast<T*>(a.q_out) + static_cast<size_t>(tok) * a.hq * hd + d;
#pragma unroll 2
      for (int h = g % split; h < a.hq; h += split) {
        float x[8], y[8];
        load8<T>(src + h * hd, x);
        load8<T>(src + h * hd + half, y);
        rotate8(x, y, c, s);
        store8(dst + h * hd, x);
        store8(dst + h * hd + half, y);
      }
    }
    return;
  }

  // ---- a page's keys or values of one head
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
  const int n_rows = w1 - w0;
  const bool keeps = w0 > 0 || live > w1;  // rows below w0 held values: start <= live
  const float s_old = *scale;
  float s;
  if (is_v) {
    const int per = hd >> 3, items = n_rows * per;  // chunks: at most four a thread (page_size * hd / 8 <= 4 blockDim)
    float x[4][8], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid + j * blockDim.x;
      if (i < items) load8<T>(src + static_cast<size_t>(i / per) * ld + (i % per) * 8, x[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tid + j * static_cast<int>(blockDim.x) < items)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(x[j][e]));
    s = page_scale(amax, keeps, s_old, red);
    const float inv = inverse_scale(s, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid + j * blockDim.x;
      if (i < items) *reinterpret_cast<uint2*>(codes + w0 * hd + i * 8) = code8(x[j], inv);
    }
  } else {
    const int per = half >> 3, items = n_rows * per;  // chunk pairs: at most two a thread
    float x[2][8], y[2][8], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = tid + j * blockDim.x;
      if (i < items) {
        const T* p = src + static_cast<size_t>(i / per) * ld + (i % per) * 8;
        load8<T>(p, x[j]);
        load8<T>(p + half, y[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = tid + j * blockDim.x;
      if (i < items) {
        float c[8], sn[8];
        const size_t at = static_cast<size_t>(base + w0 + i / per) * half + (i % per) * 8;
        load8<TT>(cos_t + at, c);
        load8<TT>(sin_t + at, sn);
        rotate8(x[j], y[j], c, sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(finite_abs(x[j][e]), finite_abs(y[j][e])));
      }
    }
    s = page_scale(amax, keeps, s_old, red);
    const float inv = inverse_scale(s, x);
    (void)inverse_scale(s, y);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = tid + j * blockDim.x;
      if (i < items) {
        uint8_t* dst = codes + (w0 + i / per) * hd + (i % per) * 8;
        *reinterpret_cast<uint2*>(dst) = code8(x[j], inv);
        *reinterpret_cast<uint2*>(dst + half) = code8(y[j], inv);
      }
    }
  }
  if (tid == 0) *scale = s;
  if (keeps && s != s_old) {  // kept rows, four codes at a time
    const float f = s_old / s;
    const int n0 = w0 * hd / 4, n1 = max(live - w1, 0) * hd / 4;
    for (int i = tid; i < n0 + n1; i += blockDim.x) {
      uint32_t* c = reinterpret_cast<uint32_t*>(codes) + (i < n0 ? i : w1 * hd / 4 + i - n0);
      const float2 lo = f32x2_from_e4m3x2(static_cast<uint16_t>(*c)), hi = f32x2_from_e4m3x2(static_cast<uint16_t>(*c >> 16));
      *c = e4m3x2_from_f32(lo.x * f, lo.y * f) | static_cast<uint32_t>(e4m3x2_from_f32(hi.x * f, hi.y * f)) << 16;
    }
  }
}

}  // namespace

int launch_paged_append(const PagedAppendArgs& a, int dtype, cudaStream_t s) {
  const int grid = a.n_units * a.hkv * 2 + (a.q_in != nullptr ? a.n_q_units : 0);
  const int block = std::max(64, std::min(512, a.page_size * 4));  // two chunk pairs of a full page a thread at head_dim 128
  if (dtype == 1)
    return a.table_f32 ? launch_k(paged_append_kernel<bf16, float>, dim3(grid), dim3(block), 0, s, a)
                       : launch_k(paged_append_kernel<bf16, bf16>, dim3(grid), dim3(block), 0, s, a);
  return launch_k(paged_append_kernel<float, float>, dim3(grid), dim3(block), 0, s, a);
}

}  // namespace fdllm
