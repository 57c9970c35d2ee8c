// Attention over a paged 8-bit KV cache at head sizes 32 and 64 (fdllm_paged_attention, bf16).  Semantics as in
// paged_attention.cu.
//
// The query rows of one request and KV head are its (token, query head) pairs; a tile has 8 * NT of them.
// A CTA takes one item of the plan: a tile and a range of keys.  Its four compute warps take the range's 16-key
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
// Bound: HBM (one byte a cached value).  A producer warp keeps a ring of 64-key stages full with TMA copies
// of whole pages (their rows of this KV head are contiguous), so the bytes in flight do not depend on the
// compute warps' registers or progress; page ids and scales are read 32 pages at a time.  A thread of
// the K fragment owns HD / 4 consecutive columns of rows g and g + 8, of the V fragment HD / 8 consecutive
// columns of its four keys (the MMA's reduction and row orders are free as long as both operands agree).
//
// A tile whose keys are split over several items joins them through the workspace: the last item to arrive
// (a counter) adds the partials in item order, so the result does not depend on the arrival order.
//
// Measured, 8/8 heads of 64: 64 tokens over 1000 keys each 21.2 us, 3.1 TB/s (latency: 512 CTAs of eight stages, a
// chain of item, page ids, scales and copies before the first); 56 prompts of 5 to 734 rows 74 us, where the 3000
// tiles' prologues and joins take more than their products.
#include "paged.h"

namespace fdllm {

namespace {

constexpr int kWarps = 4;
constexpr int kChunk = 16;  // keys a warp takes at a time
constexpr int kStageKeys = kWarps * kChunk;
constexpr int kStages = 4;
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

// N consecutive words of shared memory from byte offset `off` of row `row` of a tile of HD-byte rows.
template <int HD, int N>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* tile, int row, int off) {
  const uint8_t* p = tile + row * HD + off;
  if constexpr (N == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// Dynamic shared memory: the ring (kStages of K then V tiles, 1024-byte aligned), reused for the warps'
// partial O at the end; before it the queries.
template <int HD, int NT>
struct Smem {
  static constexpr int kTile = kStageKeys * HD;  // bytes of a K or V tile
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kJoin = kWarps * 8 * NT * HD * 4;
  static constexpr int kQ = 8 * NT * (HD + 8) * 2;
  static constexpr int kBytes = 1024 + (kRing > kJoin ? kRing : kJoin) + kQ;
};

template <int HD, int NT>
__device__ __forceinline__ void run(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v) {
  constexpr int R = 8 * NT, KS = HD / 16;  // query rows; MMA steps of a score, and of the head columns
  using S = Smem<HD, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __half* sq = reinterpret_cast<__half*>(ring + (S::kRing > S::kJoin ? S::kRing : S::kJoin));
  __shared__ float s_base[kWarps][R], s_sum[kWarps][R], s_unscale[R];
  __shared__ float2 s_scale[kStages][kStageKeys / 16];  // (K, V) scales of a stage's pages
  __shared__ uint64_t s_full[kStages], s_empty[kStages];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s_full[i], 32);
      mbar_init(&s_empty[i], kWarps);
    }
    mbar_fence_init();
  }
  pdl_trigger();
  pdl_wait();
  const PagedItem it = a.items[blockIdx.x];
  const int G = a.hq / a.hkv;
  __syncthreads();

  if (warp == kWarps) {
    // ---------------- producer: pages of the key range, kStages stages ahead ----------------
    const int ps = a.page_size, per_stage = max(kStageKeys >> a.page_shift, 1), box = min(ps, kStageKeys);
    const int* table = a.table + static_cast<size_t>(it.req) * a.table_ld;
    int batch = -32, row = 0;  // first page of the 32 whose ids and scales the lanes hold; a page's first pool row
    float2 sc = make_float2(1.f, 1.f);
    const uint64_t policy = l2_policy_evict_first();  // a step reads a cached row once
    int issued = 0;
    for (int key = it.key0; key < it.key1; key += kStageKeys, ++issued) {
      const int page0 = key >> a.page_shift, st = issued % kStages;
      if (page0 + per_stage > batch + 32) {  // uniform
        batch = page0;
        const int p = page0 + lane;
        if (static_cast<long long>(p) * ps < it.key1) {
          const int id = max(paged_page_id(table[p], a.pages, a.err), 0);
          const size_t unit = static_cast<size_t>(id) * a.hkv + it.head;
          row = static_cast<int>(unit << a.page_shift);
          sc = make_float2(__ldg(a.k_scale + unit), __ldg(a.v_scale + unit));
        }
      }
      const int from = page0 - batch + (lane < per_stage ? lane : 0);
      const int src = __shfl_sync(0xffffffffu, row, from) + (key & (ps - 1));  // (key within a page: pages over 64 rows)
      const float2 s2 = make_float2(__shfl_sync(0xffffffffu, sc.x, from), __shfl_sync(0xffffffffu, sc.y, from));
      const bool live = lane < per_stage && static_cast<long long>(page0 + lane) * ps < it.key1;
      if (!__all_sync(0xffffffffu, mbar_wait(&s_empty[st], ((issued / kStages) & 1u) ^ 1u))) {
        report_wait(a.err, kErrTimeoutProducer, 31, a.total_rows, it.splits);
        break;
      }
      if (live) {
        s_scale[st][lane] = s2;
        uint8_t* dst = ring + st * 2 * S::kTile + lane * box * HD;
        mbar_arrive_expect_tx(&s_full[st], 2 * box * HD);
        tma_load_2d(dst, &tm_k, &s_full[st], 0, a.layer_row + src, policy);
        tma_load_2d(dst + S::kTile, &tm_v, &s_full[st], 0, a.layer_row + src, policy);
      } else {
        mbar_arrive(&s_full[st]);
      }
      __syncwarp();
    }
    for (int j = max(0, issued - kStages); j < issued; ++j)  // every copy landed before leaving
      if (!mbar_wait(&s_full[j % kStages], (j / kStages) & 1u)) break;
  }

  float o[KS][NT][4], base[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    base[n][0] = base[n][1] = -INFINITY;
    sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
  }
  if (warp < kWarps) {
    // queries: f16 rows scaled by a power of two that puts the largest element into [2^7, 2^8)
    float x[R / kWarps][HD / 32];  // a warp's rows together: one latency
#pragma unroll
    for (int k = 0; k < R / kWarps; ++k) {
      const int i = warp + k * kWarps, row = it.row0 + min(i, it.rows - 1), t = row / G;
      const bf16* src = static_cast<const bf16*>(a.q) + static_cast<size_t>(it.tok0 + t) * a.ldq +
                        static_cast<size_t>(it.head * G + row - t * G) * HD;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) x[k][j] = i < it.rows ? to_f<bf16>(src[lane + 32 * j]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < R / kWarps; ++k) {
      const int i = warp + k * kWarps;
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) m = fmaxf(m, fabsf(x[k][j]));
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      // exponent of m, kept where both the scale and its inverse are normal floats; an infinite row has no weights
      int e = max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -110);
      if (m == 0.f) e = 7;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 7 - e) << 23);
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) sq[i * (HD + 8) + lane + 32 * j] = __float2half_rn(x[k][j] * up);
      if (lane == 0)
        s_unscale[i] = m < INFINITY ? a.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e - 7) << 23) : NAN;
    }
    named_sync(1, 32 * kWarps);
    uint32_t qf[KS][NT][2];  // B fragments: columns are query rows, the reduction order is the K fragment's
    float unscale[NT][2];
    int lim[NT][2], lim_min = 0x7FFFFFFF;  // keys each of this thread's columns attends
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint2 u = *reinterpret_cast<const uint2*>(sq + (n * 8 + g) * (HD + 8) + t * (HD / 4) + 4 * s);
        qf[s][n][0] = u.x, qf[s][n][1] = u.y;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = n * 8 + 2 * t + c;
        unscale[n][c] = s_unscale[i];
        lim[n][c] = i < it.rows ? min(it.key1, paged_key_limit(it.len, it.start + (it.row0 + i) / G, a.causal_block)) : it.key1;
        lim_min = min(lim_min, lim[n][c]);
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);

    int j = 0;
    for (int key0 = it.key0; key0 < it.key1; key0 += kStageKeys, ++j) {
      const int st = j % kStages, key = key0 + warp * kChunk;
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[st], (j / kStages) & 1u))) {
        report_wait(a.err, kErrTimeoutEpilogue, 32, a.total_rows, it.splits);
        break;
      }
      const uint8_t* tile = ring + st * 2 * S::kTile + warp * kChunk * HD;
      if (key < it.key1) {
        float s[NT][4], s_odd[NT][4];  // two chains of accumulation, half the latency
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = s_odd[n][e] = 0.f;
        {
          uint32_t k[2][HD / 16];
#pragma unroll
          for (int h = 0; h < 2; ++h) load_words<HD, HD / 16>(k[h], tile, g + 8 * h, t * (HD / 4));
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const uint32_t a0 = lo_pair(k[0][i]), a1 = lo_pair(k[1][i]), a2 = hi_pair(k[0][i]), a3 = hi_pair(k[1][i]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(i & 1 ? s_odd[n] : s[n], a0, a1, a2, a3, qf[i][n][0], qf[i][n][1]);
          }
        }
        uint32_t v[4][HD / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          load_words<HD, HD / 32>(v[i], tile + S::kTile, 2 * t + (i & 1) + 8 * (i >> 1), g * (HD / 8));
        const float2 sc = s_scale[st][(warp * kChunk) >> min(a.page_shift, 6)];
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[st]);  // everything of the stage is in registers
        const float lv = __log2f(sc.y), inv_vs = exp2_approx(-lv);
        bool trip = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = fmaf(s[n][e] + s_odd[n][e], unscale[n][e & 1] * sc.x, lv);
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
          for (int i = 0; i < 4; ++i)
            if (key + 2 * t + (i & 1) + 8 * (i >> 1) >= it.key1)
#pragma unroll
              for (int w = 0; w < HD / 32; ++w) v[i][w] = 0;
        }
        // head columns (HD / 8) g + 2 i (fragment rows g) and + 1 (rows g + 8): bytes of the words w = i / 2
#pragma unroll
        for (int w = 0; w < HD / 32; ++w) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t ab = __byte_perm(v[0][w], v[1][w], h == 0 ? 0x5140 : 0x7362);
            const uint32_t cd = __byte_perm(v[2][w], v[3][w], h == 0 ? 0x5140 : 0x7362);
            const uint32_t a0 = lo_pair(ab), a1 = hi_pair(ab), a2 = lo_pair(cd), a3 = hi_pair(cd);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[2 * w + h][n], a0, a1, a2, a3, p[n][0], p[n][1]);
          }
        }
      } else {
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[st]);
      }
    }
  }
  __syncthreads();  // every copy has landed and been read: the ring becomes the partials'
  float* smem = reinterpret_cast<float*>(ring);

  // join the warps: O relative to the largest base of a row
  float* so = smem + warp * R * HD;
  if (warp < kWarps) {
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
  }
  __syncthreads();
  constexpr int C4 = HD / 4;
  bf16* out = static_cast<bf16*>(a.out);
  auto write_out = [&](int i, int c4, float4 v, float inv) {
    const int row = it.row0 + i;
    bf16* dst = out + (static_cast<size_t>(it.tok0 + row / G) * a.hq + it.head * G + row % G) * HD + 4 * c4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
  };
  float4* part = a.part + it.part;  // this item's partial: [R][C4] columns, then [R] (base, sum, -, -)
  for (int i = threadIdx.x; i < it.rows * C4; i += 32 * (kWarps + 1)) {
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
#pragma unroll 1
  for (int i = threadIdx.x; i < it.rows * C4; i += 32 * (kWarps + 1)) {
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

// One launch for all classes, each a range of the grid.
template <int HD>
__global__ void __launch_bounds__(32 * (kWarps + 1), kPagedNarrowCtas)
    paged_attn_narrow_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap tm_k,
                             const __grid_constant__ CUtensorMap tm_v) {
  const int i = blockIdx.x;
  if (i < a.class_end[2]) run<HD, 3>(a, tm_k, tm_v);
  else if (i < a.class_end[1]) run<HD, 2>(a, tm_k, tm_v);
  else run<HD, 1>(a, tm_k, tm_v);
}

}  // namespace

int init_paged_attention_attributes() {
  const cudaError_t e = cudaFuncSetAttribute(paged_attn_narrow_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             Smem<32, 3>::kBytes);
  return e != cudaSuccess ? e
                          : cudaFuncSetAttribute(paged_attn_narrow_kernel<64>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<64, 3>::kBytes);
}

int launch_paged_attention_narrow(const PagedAttnArgs& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  const dim3 grid(a.class_end[0]), block(32 * (kWarps + 1));
  return a.hd == 32 ? launch_k(paged_attn_narrow_kernel<32>, grid, block, Smem<32, 3>::kBytes, s, a, k, v)
                    : launch_k(paged_attn_narrow_kernel<64>, grid, block, Smem<64, 3>::kBytes, s, a, k, v);
}

}  // namespace fdllm
