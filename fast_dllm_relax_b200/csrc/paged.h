// Paged 8-bit KV cache: the plan's layout within its int32 words (built on the host by paged.cu,
// read by the append and attention kernels) and the kernels' launch arguments.
#pragma once

#ifdef __CUDACC__
#include <cuda_fp16.h>

#include "common.cuh"
#endif
#include "kernels.h"

namespace fdllm {

// One request of a plan: kPagedReqWords words at words[kPagedReqWords * i].
constexpr int kPagedReqWords = 8;
struct PagedReq {
  int tok0;   // its first token row
  int rows;   // its token rows
  int start;  // cache position of its first token row
  int live;   // cache rows that hold values before the call
  int len;    // cached length the call attends: max(live, start + rows)
  int pad[3];
};
static_assert(sizeof(PagedReq) == 4 * kPagedReqWords, "plan request layout");

// A CTA's share of an append, two words: one page that it writes, or up to kPagedQTokens token rows whose
// queries it rotates.
constexpr int kPagedQTokens = 16;
struct PagedPageUnit {
  int req;
  int slot;  // page number within the request / first token row within it
};

constexpr int kMaxPagedSplits = 32;  // key shares of a tile (a lane each in the join)

// One share of an attention call (bf16): query rows [row0, ..) of a request and KV head (row = token * G +
// query head within the group) over keys [key0, key1).  The items of one tile (same rows) are consecutive.
constexpr int kPagedItemWords = 16;
struct alignas(16) PagedItem {
  int req, head;        // head: KV head
  int row0, rows;       // rows [row0, row0 + rows) of the request and KV head
  int key0, key1;       // key0 a multiple of 128
  int tok0, start, len; // the request's (PagedReq)
  int split, splits;    // this share's number and how many the tile has
  int tile;             // arrival counter
  int part;             // its partial in the workspace, in 16-byte units (splits > 1)
  int pad[3];
};
static_assert(sizeof(PagedItem) == 4 * kPagedItemWords, "plan item layout");

// Item classes, the largest tiles first in the plan: tiles of 16, 32 and 48 query rows (keys on the MMA's M side) and of
// up to 128 (rows on it) at head_dim 128, of 8, 16 and 24 at the others (mma.sync).
constexpr int kPagedClasses = 4;
constexpr int kPagedWide = 3;
constexpr int kPagedNarrowCtas = 3;  // CTAs on an SM at the other head sizes

// fdllm_paged_plan::priv
enum PagedPriv : int {
  kPagedPageUnits = 0,  // number of page units
  kPagedPageOff = 1,    // word offset of the page units
  kPagedTiles = 2,      // arrival counters needed
  kPagedParts = 3,      // workspace for partials, in 16-byte units
  kPagedItems = 4,      // [kPagedClasses] numbers of items
  kPagedItemOff = kPagedItems + kPagedClasses,  // word offset of the items, class after class from the last
  kPagedQUnits,         // number of query units
  kPagedQOff,           // word offset of the query units
  kPagedShape,          // [4] the handle's heads, KV heads, head_dim and dtype
  kPagedPrivEnd = kPagedShape + 4,
};

struct PagedAppendArgs {
  const PagedReq* reqs;
  const PagedPageUnit *units, *q_units;
  int n_units, n_q_units, n, total_rows;
  const int* table;
  int table_ld;
  uint8_t *k, *v;          // this layer's codes [pages, hkv, page_size, hd]
  float *k_scale, *v_scale;  // this layer's scales [pages, hkv]
  int pages, page_size;
  int hq, hkv, hd;
  const void *q_in, *k_in, *v_in;
  int ldq, ldk, ldv;
  const void *cos, *sin;   // fp32 tables, or the handle's in its dtype (table_f32 = 0)
  int table_f32;
  int rope_rows;
  void* q_out;
  int* err;
};

struct PagedAttnArgs {
  const PagedReq* reqs;
  int n, total_rows;
  const int* table;
  int table_ld;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  int pages, page_size, page_shift;  // page_size = 1 << page_shift
  int hq, hkv, hd;
  int causal_block;
  const void* q;
  int ldq;
  float scale;
  void* out;
  const PagedItem* items;
  int class_end[kPagedClasses];  // class c is the CTAs [class_end[c + 1], class_end[c])
  int layer_row;       // first row of this layer in the pool's maps (rows of head_dim codes)
  float4* part;        // partials of split tiles
  unsigned* arrived;   // [tiles] items done (zero between launches)
  int* err;
};

constexpr int kMaxTopLogprobs = 32;

struct LogprobArgs {
  const void* logits;
  int rows, vocab;
  long long ld;
  const int* targets;
  int top;
  float *logprob, *entropy;
  int* top_ids;
  float* top_logprobs;
  float4* part;               // [rows][parts] partial statistics
  unsigned long long* keys;   // [rows][parts][top] partial alternatives
  unsigned* arrived;          // [rows] parts done (zero between launches)
  int* err;
};

int launch_paged_append(const PagedAppendArgs& a, int dtype, cudaStream_t s);
int launch_paged_attention_simt(const PagedAttnArgs& a, cudaStream_t s);  // fp32
// bf16, all items in one launch (class_end[0] of them): head_dim 32 and 64; 128
int launch_paged_attention_narrow(const PagedAttnArgs& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s);
int launch_paged_attention_mma(const PagedAttnArgs& a, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s);
// CTAs a row is split into, and chunks each.
int logprobs_parts(int rows, int vocab, int dtype, int num_sms, int* part_chunks);
int launch_logprobs(const LogprobArgs& a, int dtype, int parts, int part_chunks, cudaStream_t s);

#ifdef __CUDACC__
// ---- float8 e4m3 (1 sign, 4 exponent, 3 mantissa bits; largest 448, no infinities) --------------
__device__ __forceinline__ uint16_t e4m3x2_from_f32(float lo, float hi) {  // nearest even, saturating
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t f16x2_from_e4m3x2(uint16_t c) {  // exact
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

__device__ __forceinline__ float2 f32x2_from_e4m3x2(uint16_t c) {
  const uint32_t h = f16x2_from_e4m3x2(c);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

static_assert(kPagedPrivEnd <= 17, "fdllm_paged_plan::priv");

// The request that owns token row `tok`: the last one with tok0 <= tok (empty requests share the
// tok0 of the next one, so the last is the owner).
__device__ __forceinline__ int paged_req_of(const PagedReq* reqs, int n, int tok) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (reqs[mid].tok0 <= tok) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Page id of a table entry, bounds-checked: outside [0, pages) records the error and gives -1.
__device__ __forceinline__ int paged_page_id(int id, int pages, int* err) {
  if (id >= 0 && id < pages) return id;
  report_error(err, kErrCacheRange);
  return -1;
}

// Cache rows the token row at position `pos` attends.
__device__ __forceinline__ int paged_key_limit(int len, int pos, int causal_block) {
  if (causal_block <= 0) return len;
  const long long lim = (static_cast<long long>(pos / causal_block) + 1) * causal_block;
  return lim < len ? static_cast<int>(lim) : len;
}

// What the rows of an item need.
template <int PR>
struct PagedRows {
  float unscale[PR];  // scale log2(e) over the power of two that the staged query is multiplied by
  int out[PR];        // (token, head) row of the output
  int lim[PR];        // cache rows it attends within the item's range (padding rows: the range's end)
};

// The query rows of an item as two e4m3 terms Qh + Ql (128-byte rows with the 128-byte swizzle), by 256 threads: 2 to 16
// a row, as many as fit, each with consecutive columns.  kPad: padding rows get zeros, else they are left as they are.
// A row is scaled by the power of two that puts its largest element into [2^7, 2^8).  (A warp a row, one column group a
// lane, took twice the time at 128 rows: its five shuffles and its row's bookkeeping came once a row and warp.)
template <int PR, bool kPad>
__device__ __forceinline__ void paged_stage_queries(const PagedAttnArgs& a, const PagedItem& it, uint8_t* qh, uint8_t* ql,
                                                    PagedRows<PR>& rows, int tid) {
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int kLanes = PR <= 16 ? 16 : PR <= 32 ? 8 : PR <= 48 ? 4 : 2, U = 16 / kLanes;  // threads a row, 16-byte loads
  static_assert(PR * kLanes <= 256 && (PR * kLanes) % 32 == 0, "whole warps");
  const int n = tid / kLanes, part = tid % kLanes, G = a.hq / a.hkv;
  if (n < PR) {
    const int row = it.row0 + min(n, it.rows - 1), t = row / G, h = it.head * G + row - t * G;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.q) + static_cast<long long>(it.tok0 + t) * a.ldq +
                                                      static_cast<long long>(h) * 128) + part * U;
    uint4 u[U];
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = n < it.rows ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t m2 = 0u;  // the largest magnitudes of the even and the odd columns
#pragma unroll
    for (int i = 0; i < U; ++i)
      m2 = __vmaxu2(__vmaxu2(m2, __vmaxu2(u[i].x & 0x7FFF7FFFu, u[i].y & 0x7FFF7FFFu)),
                    __vmaxu2(u[i].z & 0x7FFF7FFFu, u[i].w & 0x7FFF7FFFu));
    uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    // exponent of the maximum (a bf16's bits), kept where both the scale and its inverse are normal floats; a row that
    // is not finite has no weights: its scores become NaN below (the codes saturate)
    const bool finite = m < 0x7F80u;
    int e = max(static_cast<int>(m >> 7) - 127, -110);
    if (m == 0u) e = 7;
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 7 - e) << 23);
    if (kPad || n < it.rows) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t p = k == 0 ? u[i].x : u[i].z, q = k == 0 ? u[i].y : u[i].w;
          const float x0 = __uint_as_float(p << 16) * up, x1 = __uint_as_float(p & 0xFFFF0000u) * up;
          const float x2 = __uint_as_float(q << 16) * up, x3 = __uint_as_float(q & 0xFFFF0000u) * up;
          const uint16_t c0 = e4m3x2_from_f32(x0, x1), c1 = e4m3x2_from_f32(x2, x3);
          const float2 r0 = f32x2_from_e4m3x2(c0), r1 = f32x2_from_e4m3x2(c1);
          hi[k] = c0 | static_cast<uint32_t>(c1) << 16;
          lo[k] = e4m3x2_from_f32(x0 - r0.x, x1 - r0.y) | static_cast<uint32_t>(e4m3x2_from_f32(x2 - r1.x, x3 - r1.y)) << 16;
        }
        const int c = part * U + i, at = n * 128 + (((c >> 1) ^ (n & 7)) << 4) + (c & 1) * 8;
        *reinterpret_cast<uint2*>(qh + at) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(ql + at) = make_uint2(lo[0], lo[1]);
      }
    }
    if (part == 0) {
      rows.unscale[n] = finite ? a.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e - 7) << 23) : NAN;
      rows.out[n] = (it.tok0 + t) * a.hq + h;
      rows.lim[n] = n < it.rows ? min(it.key1, paged_key_limit(it.len, it.start + t, a.causal_block)) : it.key1;
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// The columns of paged_join: rows n0, n0 + step, .. (RB of them) of a warp, SU partials in flight.
template <int PR, int RB, int SU>
__device__ __forceinline__ void paged_join_rows(const PagedAttnArgs& a, const PagedItem& it, const float* first,
                                                const float* weight, const int* out_row, int n0, int step) {
  constexpr int kPart = PR * 132;  // floats
  const int lane = threadIdx.x & 31;
  float4 acc[RB];
#pragma unroll
  for (int j = 0; j < RB; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* from = reinterpret_cast<const float4*>(first + n0 * 128) + lane;
  const float* w = weight + n0;
#pragma unroll SU
  for (int s = 0; s < it.splits; ++s, from += kPart / 4, w += PR) {
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const float4 x = __ldcg(from + j * step * 32);
      const float f = w[j * step];
      acc[j].x += f * x.x, acc[j].y += f * x.y, acc[j].z += f * x.z, acc[j].w += f * x.w;
    }
  }
#pragma unroll
  for (int j = 0; j < RB; ++j)
    *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + static_cast<size_t>(out_row[n0 + j * step]) * 128 + 4 * lane) =
        make_uint2(pack_bf16x2(acc[j].x, acc[j].y), pack_bf16x2(acc[j].z, acc[j].w));
}

// The last item of a split tile to arrive (a.arrived) adds the tile's partials in item order, all THREADS threads:
// out = sum_s w_s O_s / sum_s w_s l_s, w_s = 2^(base_s - max base).  An item leaves [PR][128] columns of O, then PR
// pairs (base, sum).  Bound by what one SM reads from L2, about 42 bytes a clock: 12000 clocks for 64 rows x 15
// partials, 3000 for 128 x 2.  `scratch`: 16 bytes and 8 PR a split of shared memory that nothing else uses any more.
// Every thread calls it; the counter is zero again afterwards.
template <int PR, int THREADS>
__device__ __forceinline__ void paged_join(const PagedAttnArgs& a, const PagedItem& it, const int* out_row, uint8_t* scratch) {
  constexpr int kPart = PR * 132, kWarpsJ = THREADS / 32;
  int* last = reinterpret_cast<int*>(scratch);
  float* weight = reinterpret_cast<float*>(last + 4);  // [splits][PR]
  __syncthreads();
  if (threadIdx.x == 0) {  // the barriers carry its fences to the other threads
    __threadfence();
    *last = atomicAdd(&a.arrived[it.tile], 1u) == static_cast<unsigned>(it.splits - 1);
    __threadfence();
  }
  __syncthreads();
  if (!*last) return;
  const float* first = reinterpret_cast<const float*>(a.part + it.part) - static_cast<size_t>(it.split) * kPart;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // The weights.  Many rows: every thread loads pairs, then a thread a row; no more rows than warps: a warp a row, a
  // lane a partial.
  if (it.rows > kWarpsJ) {
    float* sum = weight + it.splits * PR;
    const int n_pairs = it.splits * PR;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < n_pairs; i0 += 4 * THREADS) {
      float2 p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * THREADS, s = i / PR, n = i - s * PR;
        p[j] = make_float2(0.f, 0.f);
        if (i < n_pairs && n < it.rows) p[j] = __ldcg(reinterpret_cast<const float2*>(first + s * kPart + PR * 128) + n);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j * THREADS < n_pairs)
          weight[i0 + j * THREADS] = p[j].y != 0.f ? p[j].x : -INFINITY, sum[i0 + j * THREADS] = p[j].y;
    }
    __syncthreads();
    if (threadIdx.x < it.rows) {
      const int n = threadIdx.x;
      float m = -INFINITY, l = 0.f;
#pragma unroll 4
      for (int s = 0; s < it.splits; ++s) m = fmaxf(m, weight[s * PR + n]);
#pragma unroll 4
      for (int s = 0; s < it.splits; ++s) {
        const float f = m != -INFINITY ? exp2f(weight[s * PR + n] - m) : 0.f;
        weight[s * PR + n] = f;
        l += f * sum[s * PR + n];
      }
      const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll 4
      for (int s = 0; s < it.splits; ++s) weight[s * PR + n] *= inv;
    }
    __syncthreads();
    int n = warp;
#pragma unroll 1
    for (; n + 3 * kWarpsJ < it.rows; n += 4 * kWarpsJ)
      paged_join_rows<PR, 4, 2>(a, it, first, weight, out_row, n, kWarpsJ);
#pragma unroll 1
    for (; n < it.rows; n += kWarpsJ) paged_join_rows<PR, 1, 8>(a, it, first, weight, out_row, n, kWarpsJ);
  } else if (warp < it.rows) {
    float2 bs = make_float2(0.f, 0.f);
    if (lane < it.splits) bs = __ldcg(reinterpret_cast<const float2*>(first + lane * kPart + PR * 128) + warp);
    float m = bs.y != 0.f ? bs.x : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float f = bs.y != 0.f ? exp2f(bs.x - m) : 0.f;
    float l = f * bs.y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (lane < it.splits) weight[lane * PR + warp] = l != 0.f ? f / l : 0.f;
    __syncwarp();
    paged_join_rows<PR, 1, 8>(a, it, first, weight, out_row, warp, kWarpsJ);
  }
  if (threadIdx.x == 0) a.arrived[it.tile] = 0;  // ready for the next call
}
#endif

}  // namespace fdllm
