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

// Item classes, a launch each: tiles of 16, 32 and 48 query rows (keys on the MMA's M side) and of up to 128 (rows
// on it) at head_dim 128, of 8, 16 and 24 at the others (mma.sync).
constexpr int kPagedClasses = 4;
constexpr int kPagedWide = 3;

// fdllm_paged_plan::priv
enum PagedPriv : int {
  kPagedPageUnits = 0,  // number of page units
  kPagedPageOff = 1,    // word offset of the page units
  kPagedTiles = 2,      // arrival counters needed
  kPagedParts = 3,      // workspace for partials, in 16-byte units
  kPagedItems = 4,      // [kPagedClasses] numbers of items
  kPagedItemOff = kPagedItems + kPagedClasses,  // [kPagedClasses] word offsets of the items
  kPagedQUnits = kPagedItemOff + kPagedClasses,  // number of query units
  kPagedQOff,           // word offset of the query units
  kPagedPrivEnd,
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
int launch_paged_attention_narrow(const PagedAttnArgs& a, int nt, int n_items, const CUtensorMap& k, const CUtensorMap& v,
                                  cudaStream_t s);
int launch_paged_attention_tc(const PagedAttnArgs& a, int cols, int n_items, const CUtensorMap& k, const CUtensorMap& v,
                              cudaStream_t s);
int launch_paged_attention_wide(const PagedAttnArgs& a, int n_items, const CUtensorMap& k, const CUtensorMap& v,
                                cudaStream_t s);
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
#endif

}  // namespace fdllm
