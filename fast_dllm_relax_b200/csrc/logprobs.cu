// Log probabilities of given tokens, with entropy and top alternatives, from logits (fdllm_logprobs);
// the reference reduces logits on the host (runners.py:877-881).  Per row of x, in fp32, with L = log2 e:
//   M = max x,  S0 = sum 2^((x - M) L),  S1 = sum 2^((x - M) L) (x - M) L
//   logprob = (x[target] - M) - ln S0,  entropy = ln S0 - ln 2 S1 / S0
// and the `top` largest by (value descending, id ascending).  S0 >= 1 and S1 <= 0, so a log probability is never
// positive and an entropy never negative.
//
// Bound: HBM, every logit read once.  A row is split into parts of whole chunks (256 threads x four
// 16-byte granules), a CTA a part.  A thread keeps its own running (B, S0, S1) relative to a base B, its maximum and
// the next chunk's granules in flight, so the main loop has no barrier:
//   - moving (B, S0, S1) to another base N: d = (B - N) L, f = 2^d, S1' = f (S1 + S0 d), S0' = f S0.  B starts at
//     the maximum of the part's first chunk and follows the thread's only when that is kLag above it, which few
//     chunks see; at the end all move to the row's maximum.  S1 + S0 d cancels what the lag put into S1, to 2^-24 of
//     lag S0; but a base lags only where another logit is within kLag of the maximum, so where the entropy is a good
//     part of a nat.  A peak that stands alone is its thread's base: its terms are exactly 1 and 0, and the chunks
//     after it are summed apart, as their terms may be below half a unit of that 1 (a base up to 40 behind and one
//     sum took 107.5 us where this takes 108.9, and gave a peaked row's entropy 4e-6 to 2e-5 off);
//   - the alternatives without sorting: in the part's first chunk the `top`-th largest of the 64 maxima
//     of 4-thread groups is a lower bound of its `top`-th largest logit.  Later logits matter only when
//     they exceed that bound (at equality the earlier ids win), so a chunk costs one compare a thread, and
//     the few that pass are ranked against each other by counting: after 2, 4, 8, .. chunks, when the bound
//     moves to the `top`-th largest so far, and at the end.  A part with more candidates than the buffer holds (many
//     equal logits, ascending logits) is read again and extracted in order, `top` rounds a chunk at most.
// The last CTA of a row (an arrival counter) joins the parts' statistics in part order and merges their
// sorted lists, so one launch serves any split and the result does not depend on the arrival order.
//
// Measured, fp32, 151936 logits a row, five alternatives: 1024 rows 106 to 109 us, 5.8 TB/s; 256 rows 36.8 us, 4.2 TB/s (512
// CTAs, one wave); one row 9.6 us (38 CTAs: latency of a chunk, its ranking and the join).
#include <algorithm>

#include "paged.h"

namespace fdllm {

namespace {

constexpr int kThreads = 256;
constexpr int kNV = 4;             // granules a thread per chunk
constexpr int kGroups = 64;        // 4-thread groups whose maxima bound the alternatives
constexpr int kMaxCand = 512;      // candidates of a part that are ranked by counting
constexpr int kMaxParts = 64;      // of a row: the last CTA holds their lists in shared memory
constexpr float kLag = 2.f;        // nats that a thread's maximum may be above its base
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
static_assert(kMaxTopLogprobs <= kGroups, "the bound needs `top` groups");
static_assert(kMaxTopLogprobs == 32, "a lane of one warp holds an alternative");

using Key = unsigned long long;

// Order of floats as unsigned ints (NaN as -inf, -0 as 0); 0 is below every float's rank.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x == x ? x + 0.f : -INFINITY);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t r) {
  return __uint_as_float((r & 0x80000000u) ? (r & 0x7FFFFFFFu) : ~r);
}
// The next float above x (after +inf comes NaN, which no comparison excludes).
__device__ __forceinline__ float above(float x) { return value_of(rank_of(x) + 1); }
// Order of the alternatives as one key: the value's rank, then the complemented id (lowest id first).
__device__ __forceinline__ Key make_key(float x, int id) {
  return (static_cast<Key>(rank_of(x)) << 32) | static_cast<uint32_t>(~id);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ Key warp_max_key(Key k) {
  // the high words' maximum, then the low words' among the lanes that have it
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<Key>(hi) << 32) | lo;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float* x) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float largest(const uint4& u) {  // NaN only if all are
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ float pick(const uint4& u, int i) {  // element i
    return __uint_as_float(i & 2 ? (i & 1 ? u.w : u.z) : (i & 1 ? u.y : u.x));
  }
};
template <> struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    auto pair = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float pick(const uint4& u, int i) {
    const uint32_t w = i & 4 ? (i & 2 ? u.w : u.z) : (i & 2 ? u.y : u.x);
    return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  }
};

// A thread's share of chunk c: granules (c * kNV + j) * kThreads + tid of the row, counted from the
// 16-byte granule that holds the row's first logit (`off` elements of it belong to another row).
// Granules that straddle an end of the row are read element by element, -inf outside it.
template <typename T>
struct Row {
  const T* x;
  int off, vocab;
  __device__ __forceinline__ long long id_of(int c, int j) const {  // id of granule j's first element
    return static_cast<long long>((c * kNV + j) * kThreads + static_cast<int>(threadIdx.x)) * Vec<T>::N - off;
  }
  __device__ __forceinline__ uint4 granule(int c, int j) const {
    constexpr int V = Vec<T>::N;
    const long long id = id_of(c, j);
    if (id >= 0 && id + V <= vocab) return __ldcs(reinterpret_cast<const uint4*>(x + id));
    union {
      uint4 u;
      T e[V];
    } g;
#pragma unroll
    for (int i = 0; i < V; ++i) g.e[i] = id + i >= 0 && id + i < vocab ? x[id + i] : from_f<T>(-INFINITY);
    return g.u;
  }
  __device__ __forceinline__ void load(int c, uint4 (&g)[kNV]) const {
    constexpr int V = Vec<T>::N;
    constexpr long long kChunk = static_cast<long long>(kThreads) * kNV * V;
    const long long first = c * kChunk - off;
    if (first >= 0 && first + kChunk <= vocab) {  // a whole chunk (uniform): no checks per granule
      const uint4* p = reinterpret_cast<const uint4*>(x + first) + threadIdx.x;
#pragma unroll
      for (int j = 0; j < kNV; ++j) g[j] = __ldcs(p + j * kThreads);
    } else {
#pragma unroll
      for (int j = 0; j < kNV; ++j) g[j] = granule(c, j);
    }
  }
};

__device__ __forceinline__ void join(float& M, float& s0, float& s1, float N) {  // to the larger base N
  if (N == M || M == -INFINITY) {
    M = N;
    return;
  }
  const float d = (M - N) * kLog2e, f = exp2f(d);
  s1 = f * (s1 + s0 * fmaxf(d, -1e30f));
  s0 *= f;
  M = N;
}

// The target's logit (NaN with the error recorded for an id outside the vocabulary).
template <typename T>
__device__ __forceinline__ float target_logit(const LogprobArgs& a, int row) {
  if (a.targets == nullptr) return 0.f;
  const int t = a.targets[row];
  if (t >= 0 && t < a.vocab) return to_f<T>(static_cast<const T*>(a.logits)[static_cast<size_t>(row) * a.ld + t]);
  report_error(a.err, kErrTokenRange);
  return NAN;
}

// The results of a row from its statistics, joined at its maximum M, and merged alternatives (lane < top holds one);
// xt: the target's logit, in lane 0.
__device__ __forceinline__ void write_row(const LogprobArgs& a, int row, float M, float s0, float s1, float xt, Key key,
                                          int lane) {
  // no distribution: only -inf logits (S0 = 0), or a NaN or +inf one (S0 = NaN)
  // the maximum's own term is 1, and no term of S1 is positive: what is below or above is rounding
  const float ls = s0 > 0.f ? logf(fmaxf(s0, 1.f)) : NAN;
  if (lane == 0) {
    if (a.targets != nullptr) a.logprob[row] = (xt - M) - ls;
    if (a.entropy != nullptr) a.entropy[row] = ls - kLn2 * (fminf(s1, 0.f) / s0);
  }
  if (lane < a.top) {
    a.top_ids[static_cast<size_t>(row) * a.top + lane] = static_cast<int>(~static_cast<uint32_t>(key));
    a.top_logprobs[static_cast<size_t>(row) * a.top + lane] = (value_of(static_cast<uint32_t>(key >> 32)) - M) - ls;
  }
}

// s_top[0 .. min(n, top)) = the largest of n distinct keys (0: none) in order, each placed by counting
// those above it; eight threads count for a key, an eighth of the keys each.
__device__ __forceinline__ void rank_candidates(const Key* keys, int n, int top, Key* s_top) {
  for (int c0 = 0; c0 < n; c0 += kThreads / 8) {  // uniform: the shuffles need whole warps
    const int c = c0 + (static_cast<int>(threadIdx.x) >> 3);
    const Key mine = c < n ? keys[c] : 0;
    int above = 0;
    for (int o = threadIdx.x & 7; o < n; o += 8) above += keys[o] > mine;
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    above += __shfl_xor_sync(0xffffffffu, above, 2);
    above += __shfl_xor_sync(0xffffffffu, above, 4);
    if (mine != 0 && above < top && (threadIdx.x & 7) == 0) s_top[above] = mine;
  }
}

// The sorted alternatives of chunks [c0, c1) by extraction, for a part whose candidates overflowed: per
// chunk the largest key below the last one taken, until `top` are taken or none beats the list's end.
template <typename T>
__device__ __noinline__ void extract_part(const Row<T>& row, int c0, int c1, int top, Key* s_top, Key* s_best) {
  constexpr int V = Vec<T>::N;
  __shared__ Key s_list[kMaxTopLogprobs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kMaxTopLogprobs) s_top[threadIdx.x] = 0;
  __syncthreads();
  for (int c = c0; c < c1; ++c) {
    uint4 g[kNV];
    row.load(c, g);
    const Key end = s_top[top - 1];
    Key last = ~Key(0);
    int taken = 0;
    for (; taken < top; ++taken) {
      Key b = 0;
#pragma unroll
      for (int j = 0; j < kNV; ++j) {
        float v[V];
        Vec<T>::unpack(g[j], v);
        const long long id = row.id_of(c, j);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const Key k = id + i >= 0 && id + i < row.vocab ? make_key(v[i], static_cast<int>(id + i)) : 0;
          if (k < last && k > b) b = k;
        }
      }
      b = warp_max_key(b);
      if (lane == 0) s_best[warp] = b;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) b = s_best[w] > b ? s_best[w] : b;
      __syncthreads();
      if (b <= end) break;  // uniform
      last = b;
      if (threadIdx.x == 0) s_list[taken] = b;
    }
    __syncthreads();
    // merge s_list[0, taken) into s_top: each key's place is its rank in both (keys are distinct)
    Key mine = 0;
    int place = kMaxTopLogprobs;
    if (warp < 2) {
      mine = warp == 0 ? (lane < top ? s_top[lane] : 0) : (lane < taken ? s_list[lane] : 0);
      if (mine != 0) {
        place = 0;
        for (int o = 0; o < top; ++o) place += s_top[o] > mine;
        for (int o = 0; o < taken; ++o) place += s_list[o] > mine;
      }
    }
    __syncthreads();
    if (place < top) s_top[place] = mine;
    __syncthreads();
  }
}

// parts: CTAs a row; part_chunks: chunks a part.  a.part[i] = (M, S0, S1, -) of part i of the row,
// a.keys[i * top ..] its sorted alternatives (0: none).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const LogprobArgs a, int parts, int part_chunks) {
  constexpr int V = Vec<T>::N, E = kNV * V;
  __shared__ uint32_t s_group[kGroups];
  __shared__ float s_M[8], s_s0[8], s_s1[8];
  __shared__ Key s_cand[kMaxCand], s_top[kMaxTopLogprobs], s_best[8];
  extern __shared__ Key s_lists[];  // [parts * top], the last CTA's merge
  __shared__ float s_tau, s_base;
  __shared__ int s_count, s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x / parts, part = blockIdx.x % parts;
  if (threadIdx.x == 0) s_count = 0;
  pdl_trigger();
  pdl_wait();

  Row<T> row;
  row.x = static_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld;
  row.off = static_cast<int>((reinterpret_cast<uintptr_t>(row.x) & 15) / sizeof(T));
  row.vocab = a.vocab;
  const int chunks = static_cast<int>((static_cast<long long>(a.vocab) + row.off + kThreads * E - 1) / (kThreads * E));
  const int c0 = part * part_chunks, c1 = min(c0 + part_chunks, chunks);

  float M = -INFINITY, top_x = -INFINITY, s0 = 0.f, s1 = 0.f, bound = -INFINITY;  // M: the base, top_x: the maximum
  float rest = 0.f;  // of S0, the chunks since the one that set the base
  uint4 next[kNV];
  row.load(c0, next);
  for (int c = c0; c < c1; ++c) {
    uint4 cur[kNV];
#pragma unroll
    for (int j = 0; j < kNV; ++j) cur[j] = next[j];
    if (c + 1 < c1) row.load(c + 1, next);
    float gmax[kNV], cm = -INFINITY;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      gmax[j] = Vec<T>::largest(cur[j]);
      cm = fmaxf(cm, gmax[j]);
    }
    top_x = fmaxf(top_x, cm);
    if (c == c0) {
      float gm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 1));
      gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
      if ((lane & 3) == 0) s_group[threadIdx.x >> 2] = rank_of(gm);
      __syncthreads();
      {  // the largest and the `top`-th largest group maximum: four threads count a group's rank, a quarter each
        const int g = threadIdx.x >> 2, o0 = (lane & 3) * (kGroups / 4);
        const uint32_t mine = s_group[g];
        int rank = 0;
#pragma unroll
        for (int o = 0; o < kGroups / 4; ++o) {
          const uint32_t other = s_group[o0 + o];
          rank += other > mine || (other == mine && o0 + o < g);
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (rank == 0) s_base = value_of(mine);
        if (rank == a.top - 1) s_tau = value_of(mine);
      }
      __syncthreads();
      M = s_base;
      if (a.top > 0) bound = s_tau;
    }
    if (a.top > 0) {
      // logits that reach the bound; a NaN passes (the comparison is negated) and ranks as -inf
#pragma unroll
      for (int j = 0; j < kNV; ++j) {
        if (!(gmax[j] < bound)) {
          uint32_t pass = 0;  // a bit per logit of the granule
          float v[V];
          Vec<T>::unpack(cur[j], v);
#pragma unroll
          for (int i = 0; i < V; ++i) pass |= static_cast<uint32_t>(!(v[i] < bound)) << i;
          const long long id0 = row.id_of(c, j);
          while (pass != 0) {
            const int i = __ffs(pass) - 1;
            pass &= pass - 1;
            const long long id = id0 + i;
            if (id < 0 || id >= a.vocab) continue;  // the -inf outside the row
            const int at = atomicAdd(&s_count, 1);
            if (at < kMaxCand) s_cand[at] = make_key(Vec<T>::pick(cur[j], i), static_cast<int>(id));
          }
        }
      }
      if (c == c0) bound = above(bound);
      // after 2, 4, 8, .. chunks the bound moves to the `top`-th largest so far
      const int done = c - c0 + 1;
      if (done >= 2 && (done & (done - 1)) == 0 && c + 1 < c1) {
        __syncthreads();
        const int n = s_count;
        if (n > a.top && n <= kMaxCand) {  // uniform
          rank_candidates(s_cand, n, a.top, s_top);
          __syncthreads();
          if (static_cast<int>(threadIdx.x) < a.top) s_cand[threadIdx.x] = s_top[threadIdx.x];
          if (threadIdx.x == 0) s_count = a.top;
          bound = above(value_of(static_cast<uint32_t>(s_top[a.top - 1] >> 32)));
        }
        __syncthreads();
      }
    }
    const bool peak = cm > M + kLag;
    if (peak) {
      s0 += rest, rest = 0.f;
      join(M, s0, s1, cm);
    }
    const float base = M == -INFINITY ? 0.f : M;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      float v[V];
      Vec<T>::unpack(cur[j], v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = (v[i] - base) * kLog2e, e = exp2_approx(d);
        sum += e;
        s1 = fmaf(e, fmaxf(d, -1e30f), s1);  // a logit of -inf adds 0, not 0 * inf
      }
    }
    if (peak || c == c0) s0 += sum;
    else rest += sum;
  }
  s0 += rest;

  // the part's statistics: the block's maximum, then the threads' sums relative to it
  float W = warp_max(top_x);
  if (lane == 0) s_M[warp] = W;
  __syncthreads();  // also: every candidate is in the buffer
  W = s_M[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) W = fmaxf(W, s_M[w]);
  join(M, s0, s1, W);
  s0 = warp_sum(s0);
  s1 = warp_sum(s1);
  if (lane == 0) s_s0[warp] = s0, s_s1[warp] = s1;
  if (a.top > 0) {
    const int n = s_count;
    if (n > kMaxCand) {
      extract_part<T>(row, c0, c1, a.top, s_top, s_best);
    } else {
      if (static_cast<int>(threadIdx.x) >= n && threadIdx.x < kMaxTopLogprobs) s_top[threadIdx.x] = 0;
      rank_candidates(s_cand, n, a.top, s_top);
    }
  }
  __syncthreads();
  if (warp == 0) {
    s0 = s_s0[0], s1 = s_s1[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) s0 += s_s0[w], s1 += s_s1[w];
    if (parts == 1) {
      write_row(a, r, W, s0, s1, lane == 0 ? target_logit<T>(a, r) : 0.f, lane < a.top ? s_top[lane] : 0, lane);
    } else {
      const size_t at = static_cast<size_t>(r) * parts + part;
      if (lane == 0) a.part[at] = make_float4(W, s0, s1, 0.f);
      if (lane < a.top) a.keys[at * a.top + lane] = s_top[lane];
      __threadfence();
      __syncwarp();
      if (lane == 0) s_last = atomicAdd(&a.arrived[r], 1u) == static_cast<unsigned>(parts - 1);
    }
  }
  if (parts == 1) return;
  __syncthreads();
  if (!s_last) return;

  // the row's last CTA: every part is published
  __threadfence();
  const size_t base = static_cast<size_t>(r) * parts;
  for (int i = threadIdx.x; i < parts * a.top; i += kThreads) s_lists[i] = __ldcg(&a.keys[base * a.top + i]);
  if (warp == 0) {
    const float4 none = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    float4 p = lane < parts ? __ldcg(&a.part[base + lane]) : none;
    const float4 q = lane + 32 < parts ? __ldcg(&a.part[base + lane + 32]) : none;
    W = warp_max(fmaxf(p.x, q.x));
    join(p.x, p.y, p.z, W);
    M = q.x, s0 = q.y, s1 = q.z;
    join(M, s0, s1, W);
    s0 = warp_sum(p.y + s0);
    s1 = warp_sum(p.z + s1);
  }
  const float xt = threadIdx.x == 0 ? target_logit<T>(a, r) : 0.f;
  __syncthreads();
  Key mine = 0;
  if (parts * a.top <= kThreads) {  // few keys: placed by counting
    rank_candidates(s_lists, parts * a.top, a.top, s_top);
    __syncthreads();
    if (warp != 0) return;
    if (lane < a.top) mine = s_top[lane];
  } else {  // a lane owns the lists of parts lane and lane + 32 and offers the better of their heads
    if (warp != 0) return;
    int h0 = 0, h1 = 0;
    auto head = [&](int p, int h) { return p < parts && h < a.top ? s_lists[p * a.top + h] : 0; };
    Key k0 = head(lane, 0), k1 = head(lane + 32, 0);
    for (int t = 0; t < a.top; ++t) {
      const Key best = warp_max_key(k0 > k1 ? k0 : k1);
      if (lane == t) mine = best;
      if (k0 == best) k0 = head(lane, ++h0);
      else if (k1 == best) k1 = head(lane + 32, ++h1);
    }
  }
  write_row(a, r, W, s0, s1, xt, mine, lane);
  if (lane == 0) a.arrived[r] = 0;  // ready for the next call
}

}  // namespace

// Parts of a row (at most kMaxParts) and chunks a part: what takes the fewest chunk times, waves of four CTAs an SM by
// the chunks of a part and about four more for its bound, its ranking and the join.  (256 x 151936 fp32, top 5: 3 parts
// in two waves 40.0 us, 2 in one 36.4; 32 rows: 19 parts 14.3, 18 in one wave 13.8.)
int logprobs_parts(int rows, int vocab, int dtype, int num_sms, int* part_chunks) {
  const int v = dtype == 1 ? Vec<bf16>::N : Vec<float>::N;
  const long long chunk = static_cast<long long>(kThreads) * kNV * v, slots = 4LL * num_sms;
  const int chunks = static_cast<int>((vocab + (v - 1) + chunk - 1) / chunk);  // v - 1: a row that starts inside a granule
  int best = 1;
  long long least = -1;
  for (int p = 1; p <= std::min(chunks, kMaxParts); ++p) {
    const int each = (chunks + p - 1) / p;
    if ((chunks + each - 1) / each != p) continue;
    const long long cost = (static_cast<long long>(rows) * p + slots - 1) / slots * (each + 4);
    if (least < 0 || cost < least) least = cost, best = p;
  }
  *part_chunks = (chunks + best - 1) / best;
  return best;
}

int launch_logprobs(const LogprobArgs& a, int dtype, int parts, int part_chunks, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.rows) * parts);
  const size_t lists = parts > 1 ? sizeof(Key) * parts * a.top : 0;  // at most 16 KB
  return dtype == 1 ? launch_k(logprobs_kernel<bf16>, grid, dim3(kThreads), lists, s, a, parts, part_chunks)
                    : launch_k(logprobs_kernel<float>, grid, dim3(kThreads), lists, s, a, parts, part_chunks);
}

}  // namespace fdllm
