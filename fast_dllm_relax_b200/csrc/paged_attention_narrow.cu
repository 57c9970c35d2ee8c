// Attention over a paged 8-bit KV cache for few query rows (fdllm_paged_attention, bf16): single tokens
// and small steps.  Semantics as in paged_attention.cu.
//
// The query rows of one request and KV head are its (token, query head) pairs; a tile has 8 * NT of them.
// A CTA takes one item of the plan: a tile and a range of keys.  Its four warps take the range's 16-key
// chunks in turn (a chunk lies in one page: one page id and one scale pair), each on its own:
//   S^T = K Q^T     m16n8k16: keys are the M side, so that 8 query rows fill the tensor tile
//   P^T = 2^(a S + log2 vs - B)      a = scale log2(e) ks, B the column's base
//   O^T += V^T P^T  head columns are the M side; P^T is S^T's accumulator, packed and transposed in
//                   registers (movmatrix)
// in f16: e4m3 codes are exact in it, a query row scaled by a power of two loses nothing above 2^-22 of
// its largest element, and P^T keeps 11 bits.  Folding the page's value scale into the exponent keeps P
// inside f16's range whatever the scales are; the row sum l takes 2^-log2(vs) back out.  The base moves
// only when a weight passes 2^15 (then to 2^8), which one vote a chunk finds, so the maximum costs no
// shuffles; weights down to 2^-32 of the largest are kept.
//
// Bound: HBM (one byte a cached value).  K and V codes go from global memory straight to the fragments'
// registers: a thread of the K fragment owns HD / 4 consecutive columns of rows g and g + 8, of the V
// fragment HD / 8 consecutive columns of its four keys (the MMA's reduction and row orders are free as long
// as both operands agree), so the loads are 16 bytes wide and whole rows are read.  The next chunk's loads
// are in flight while a chunk is computed, the page id of the one after it too.
//
// A tile whose keys are split over several items joins them through the workspace: the last item to arrive
// (a counter) adds the partials in item order, so the result does not depend on the arrival order.
#include "paged.h"

namespace fdllm {

namespace {

constexpr int kWarps = 4;
constexpr int kChunk = 16;  // keys
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTrip = 15.f, kSeat = 8.f;  // P may reach 2^kTrip; a moved base puts the maximum at 2^kSeat

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lo_pair(uint32_t w) { return f16x2_from_e4m3x2(static_cast<uint16_t>(w)); }
__device__ __forceinline__ uint32_t hi_pair(uint32_t w) { return f16x2_from_e4m3x2(static_cast<uint16_t>(w >> 16)); }

// N consecutive words from p.
template <int N>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* p) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
    }
  } else if constexpr (N == 2) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = u.x, w[1] = u.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// One chunk's codes as the fragments need them, and its page's scales.
template <int HD>
struct Chunk {
  static constexpr int KW = HD / 16, VW = HD / 32;  // words a key row of the K and of the V fragment
  uint32_t k[2][KW], v[4][VW];
  float ks, vs;
};

template <int HD, int NT>
__global__ void __launch_bounds__(32 * kWarps) paged_attn_narrow_kernel(const PagedAttnArgs a) {
  constexpr int R = 8 * NT, KS = HD / 16;  // query rows; MMA steps of a score, and of the head columns
  extern __shared__ float smem[];          // queries at first, then the warps' partial O [kWarps][R][HD]
  __shared__ float s_base[kWarps][R], s_sum[kWarps][R], s_unscale[R];
  __shared__ int s_last;
  pdl_trigger();
  pdl_wait();
  const PagedItem it = a.items[blockIdx.x];
  const PagedReq r = a.reqs[it.req];
  const int G = a.hq / a.hkv, rows = min(r.rows * G - it.row0, R);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // queries: f16 rows scaled by a power of two that puts the largest element into [2^7, 2^8)
  __half* sq = reinterpret_cast<__half*>(smem);
  for (int i = warp; i < R; i += kWarps) {
    const int row = it.row0 + i;
    const bool ok = i < rows;
    const bf16* src = static_cast<const bf16*>(a.q) + static_cast<size_t>(r.tok0 + (ok ? row / G : 0)) * a.ldq +
                      static_cast<size_t>(it.head * G + (ok ? row % G : 0)) * HD;
    float x[HD / 32], m = 0.f;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
      x[j] = ok ? to_f<bf16>(src[lane + 32 * j]) : 0.f;
      m = fmaxf(m, fabsf(x[j]));
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // exponent of m, kept where both the scale and its inverse are normal floats
    const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -110), 110);
    const float up = m > 0.f ? __uint_as_float(static_cast<uint32_t>(127 + 7 - e) << 23) : 1.f;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) sq[i * (HD + 8) + lane + 32 * j] = __float2half_rn(x[j] * up);
    if (lane == 0) s_unscale[i] = a.scale * kLog2e / up;
  }
  __syncthreads();
  uint32_t qf[KS][NT][2];  // B fragments: columns are query rows, the reduction order is the K fragment's
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint2 u = *reinterpret_cast<const uint2*>(sq + (n * 8 + g) * (HD + 8) + t * (HD / 4) + 4 * s);
      qf[s][n][0] = u.x, qf[s][n][1] = u.y;
    }
  float unscale[NT][2];
  int lim[NT][2], lim_min = 0x7FFFFFFF;  // keys each of this thread's columns attends
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = n * 8 + 2 * t + c;
      unscale[n][c] = s_unscale[i];
      lim[n][c] = i < rows ? min(it.key1, paged_key_limit(r.len, r.start + (it.row0 + i) / G, a.causal_block)) : it.key1;
      lim_min = min(lim_min, lim[n][c]);
    }
  lim_min = __reduce_min_sync(0xffffffffu, lim_min);
  __syncthreads();  // the queries' shared memory becomes the partials'

  float o[KS][NT][4], base[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    base[n][0] = base[n][1] = -INFINITY;
    sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
  }

  const int* table = a.table + static_cast<size_t>(it.req) * a.table_ld;
  auto page_of = [&](int key) { return key < it.key1 ? paged_page_id(table[key >> a.page_shift], a.pages, a.err) : 0; };
  auto fetch = [&](Chunk<HD>& c, int key, int page) {
    const size_t unit = static_cast<size_t>(max(page, 0)) * a.hkv + it.head;
    const size_t row0 = (unit << a.page_shift) + (key & (a.page_size - 1));
    const uint8_t* kp = a.k + row0 * HD + t * (HD / 4);
    const uint8_t* vp = a.v + row0 * HD + g * (HD / 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) load_words<Chunk<HD>::KW>(c.k[h], kp + (g + 8 * h) * HD);
#pragma unroll
    for (int j = 0; j < 4; ++j) load_words<Chunk<HD>::VW>(c.v[j], vp + (2 * t + (j & 1) + 8 * (j >> 1)) * HD);
    c.ks = __ldg(a.k_scale + unit);
    c.vs = __ldg(a.v_scale + unit);
  };

  int key = it.key0 + warp * kChunk;
  Chunk<HD> cur;
  if (key < it.key1) fetch(cur, key, page_of(key));
  int next_page = page_of(key + kWarps * kChunk);
  for (; key < it.key1; key += kWarps * kChunk) {
    Chunk<HD> next;
    const int nk = key + kWarps * kChunk;
    if (nk < it.key1) fetch(next, nk, next_page);
    next_page = page_of(nk + kWarps * kChunk);

    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const uint32_t a0 = lo_pair(cur.k[0][st]), a1 = lo_pair(cur.k[1][st]);
      const uint32_t a2 = hi_pair(cur.k[0][st]), a3 = hi_pair(cur.k[1][st]);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(s[n], a0, a1, a2, a3, qf[st][n][0], qf[st][n][1]);
    }
    const float lv = __log2f(cur.vs), inv_vs = exp2_approx(-lv);
    bool trip = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = fmaf(s[n][e], unscale[n][e & 1] * cur.ks, lv);
        if (key + kChunk > lim_min && key + g + (e >> 1) * 8 >= lim[n][e & 1]) x = -INFINITY;
        s[n][e] = x;
        trip |= x > base[n][e & 1] + kTrip;
      }
    if (__any_sync(0xffffffffu, trip)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = fmaxf(s[n][c], s[n][c + 2]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          if (m > base[n][c] + kTrip) {
            const float f = exp2_approx(base[n][c] - (m - kSeat));
            base[n][c] = m - kSeat;
            sum[n][c] *= f;
#pragma unroll
            for (int i = 0; i < KS; ++i) o[i][n][c] *= f, o[i][n][c + 2] *= f;
          }
        }
    }
    uint32_t p[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float b = base[n][e & 1];
        s[n][e] = exp2_approx(s[n][e] - (b == -INFINITY ? 0.f : b));
      }
      sum[n][0] += (s[n][0] + s[n][2]) * inv_vs;
      sum[n][1] += (s[n][1] + s[n][3]) * inv_vs;
      p[n][0] = transpose_8x8(pack_f16x2(s[n][0], s[n][1]));
      p[n][1] = transpose_8x8(pack_f16x2(s[n][2], s[n][3]));
    }
    if (key + kChunk > it.key1) {  // rows past the range hold anything: their weight is 0, their values must be
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (key + 2 * t + (j & 1) + 8 * (j >> 1) >= it.key1)
#pragma unroll
          for (int w = 0; w < Chunk<HD>::VW; ++w) cur.v[j][w] = 0;
    }
    // head columns (HD / 8) g + 2 i (fragment rows g) and + 1 (rows g + 8): bytes of the words w = i / 2
#pragma unroll
    for (int w = 0; w < Chunk<HD>::VW; ++w) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t ab = __byte_perm(cur.v[0][w], cur.v[1][w], h == 0 ? 0x5140 : 0x7362);
        const uint32_t cd = __byte_perm(cur.v[2][w], cur.v[3][w], h == 0 ? 0x5140 : 0x7362);
        const uint32_t a0 = lo_pair(ab), a1 = hi_pair(ab), a2 = lo_pair(cd), a3 = hi_pair(cd);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[2 * w + h][n], a0, a1, a2, a3, p[n][0], p[n][1]);
      }
    }
    cur = next;
  }

  // join the warps: O relative to the largest base of a row
  float* so = smem + warp * R * HD;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = n * 8 + 2 * t + c;
      float l = sum[n][c];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (g == 0) s_base[warp][row] = base[n][c], s_sum[warp][row] = l;
#pragma unroll
      for (int i = 0; i < KS; i += 2)
        *reinterpret_cast<float4*>(so + row * HD + g * (HD / 8) + 2 * i) =
            make_float4(o[i][n][c], o[i][n][c + 2], o[i + 1][n][c], o[i + 1][n][c + 2]);
    }
  __syncthreads();
  constexpr int C4 = HD / 4;
  bf16* out = static_cast<bf16*>(a.out);
  auto write_out = [&](int i, int c4, float4 v, float inv) {
    const int row = it.row0 + i;
    bf16* dst = out + (static_cast<size_t>(r.tok0 + row / G) * a.hq + it.head * G + row % G) * HD + 4 * c4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
  };
  float4* part = a.part + it.part;  // this item's partial: [R][C4] columns, then [R] (base, sum, -, -)
  for (int i = threadIdx.x; i < rows * C4; i += 32 * kWarps) {
    const int row = i / C4, c4 = i % C4;
    float m = s_base[0][row];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_base[w][row]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float b = s_base[w][row], f = b == -INFINITY ? 0.f : exp2f(b - m);
      const float4 v = *reinterpret_cast<const float4*>(smem + (w * R + row) * HD + 4 * c4);
      l += f * s_sum[w][row];
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
    }
    if (it.splits == 1) {
      write_out(row, c4, acc, l != 0.f ? 1.f / l : 0.f);
    } else {
      part[row * C4 + c4] = acc;
      if (c4 == 0) part[R * C4 + row] = make_float4(m, l, 0.f, 0.f);
    }
  }
  if (it.splits == 1) return;

  // the tile's last item adds the partials
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(&a.arrived[it.tile], 1u) == static_cast<unsigned>(it.splits - 1);
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  constexpr int kPart = R * C4 + R;
  const float4* first = part - static_cast<size_t>(it.split) * kPart;
  for (int i = threadIdx.x; i < rows * C4; i += 32 * kWarps) {
    const int row = i / C4, c4 = i % C4;
    float m = -INFINITY;
    for (int s = 0; s < it.splits; ++s) m = fmaxf(m, __ldcg(&first[s * kPart + R * C4 + row]).x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 8
    for (int s = 0; s < it.splits; ++s) {
      const float4 b = __ldcg(&first[s * kPart + R * C4 + row]), v = __ldcg(&first[s * kPart + row * C4 + c4]);
      const float f = b.x == -INFINITY ? 0.f : exp2f(b.x - m);
      l += f * b.y;
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
    }
    write_out(row, c4, acc, l != 0.f ? 1.f / l : 0.f);
  }
  if (threadIdx.x == 0) a.arrived[it.tile] = 0;  // ready for the next call
}

template <int HD, int NT>
constexpr size_t smem_bytes() {
  return sizeof(float) * kWarps * 8 * NT * HD;
}

template <int HD>
int launch_hd(const PagedAttnArgs& a, int nt, int n_items, cudaStream_t s) {
  const dim3 grid(n_items), block(32 * kWarps);
  switch (nt) {
    case 1: return launch_k(paged_attn_narrow_kernel<HD, 1>, grid, block, smem_bytes<HD, 1>(), s, a);
    case 2: return launch_k(paged_attn_narrow_kernel<HD, 2>, grid, block, smem_bytes<HD, 2>(), s, a);
    default: return launch_k(paged_attn_narrow_kernel<HD, 3>, grid, block, smem_bytes<HD, 3>(), s, a);
  }
}

}  // namespace

int init_paged_attention_attributes() {
  cudaError_t e = cudaFuncSetAttribute(paged_attn_narrow_kernel<128, 3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem_bytes<128, 3>()));
  return e;
}

int launch_paged_attention_narrow(const PagedAttnArgs& a, int nt, int n_items, cudaStream_t s) {
  switch (a.hd) {
    case 32: return launch_hd<32>(a, nt, n_items, s);
    case 64: return launch_hd<64>(a, nt, n_items, s);
    default: return launch_hd<128>(a, nt, n_items, s);
  }
}

}  // namespace fdllm
