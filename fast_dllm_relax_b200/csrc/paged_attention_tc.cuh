// Attention over a paged 8-bit KV cache on the 5th-generation tensor cores for up to 48 query rows
// (fdllm_paged_attention, bf16, head_dim 128).  Semantics as in paged_attention.cu; the cached codes are never
// widened.
//
// The query rows of one request and KV head are its (token, query head) pairs.  A CTA takes one item of the
// plan, a tile of at most N rows and a range of keys, in tiles of 128 keys with the keys on the MMA's M side:
//   S^T [128 keys, 2 N]    = K (Qh | Ql)^T          A: the K tile (e4m3, K-major), B: the queries (e4m3, K-major)
//   P^T [128 keys, N]      = 2^(a S + log2 vs - B)
//   O^T [128 columns, 3 N] += V^T (Pa | Pb | Pc)^T  A: the V tile (e4m3, MN-major), B: P (e5m2, MN-major)
// so a page goes from memory by TMA straight into both operands, N follows the number of query rows (a lone
// token needs 16 columns, not 128 rows of padding), and a thread of the softmax holds one key: the page's scales
// are one pair a thread.  What an SM pays a tile is shared-memory traffic (the tensor core reads A at 64 bytes a
// clock), so the terms of an operand sit side by side in N and each tile is read once.
//
// Precision.  A bf16 query has 8 significant bits: Q = Qh + Ql under one power of two per row (largest element
// in [2^7, 2^8)), exact for elements above 2^-10 of the row's largest and to 2^-18 of it below.  A probability
// is rounded to f16, as for many rows, and split into P = Pa + 2^-3 Pb + 2^-8 Pc, each term the e5m2 rounding of what
// the ones before leave.  e5m2 has f16's exponents and 3 of its 11 bits, and a signed remainder brings 4 with each
// term, so the three hold every f16 from 2^-13 on and are 2^-24 off at most below: 11 bits for weights down to 2^-21 of
// the largest (seated at 2^8 or more), then a bit less a power of two, the last lost at 2^-32.  (Three e4m3 terms hold
// 12 bits at the top, but end at 2^-22 of a maximum at 2^3: beside a sink whose own value is small the weights left
// over are the result.)  Each column's base B moves only when a weight passes 2^kTrip (then its maximum sits at
// 2^kSeat): one block-wide vote a tile instead of a maximum over 128 lanes.  log2 vs in the exponent keeps P in range
// whatever the page scales are; the row sums take it back out.
//
// Roles (384 threads, registers moved to the softmax): warp 0 the TMA producer (a lane a page; page ids and
// scales 32 pages at a time), warp 1 the MMA issuer and TMEM owner, warps 4-11 the softmax, a key and half the
// columns a thread.  S_{j+1} is computed while tile j is in the softmax, once its scores have been loaded.  Two
// CTAs share an SM.
//
// A tile whose keys are split over several items joins them through the workspace: the last item to arrive adds the
// partials in item order (paged_join).
//
// Measured, 12/2 heads of 128: one token over 397 keys 8.3 us (a chain of latencies: item, page ids, scales, copies,
// two products, the join), over 32000 keys 16.7; 64 tokens over 700 to 8191 keys 24.9 us, 4.1 TB/s (102 MB: each of
// the 284 items waits through its prologue once, and they end unevenly); 8 rows of 8 requests over 4096 keys 19.6 us.
#pragma once
#include "paged_mma.cuh"

namespace fdllm {
namespace paged_tc {

constexpr int kKeys = 128;
constexpr int kHd = 128;
constexpr int kTile = kKeys * kHd;  // bytes of a K or V tile
constexpr float kTrip = 15.f, kSeat = 8.f;

// Instruction descriptor, kind::f8f6f4: fp32 accumulator, M 128; S = K Q^T has both operands e4m3 and K-major,
// O^T = V^T P^T both MN-major and B e5m2.
constexpr uint32_t idesc_s(int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24); }
constexpr uint32_t idesc_o(int n) { return idesc_s(n) | (1u << 10) | (1u << 15) | (1u << 16); }

// Shared-memory descriptor of an unswizzled MN-major operand: core matrices of 8 K rows by 16 MN bytes
// (128 B, row after row), `mn` bytes between core matrices along MN and `k` along K.
__device__ __forceinline__ uint64_t umma_desc_mn(const void* p, uint32_t mn, uint32_t k) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr(p) >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((k >> 4) & 0x3FFFu) << 16;   // leading byte offset: along K
  d |= static_cast<uint64_t>((mn >> 4) & 0x3FFFu) << 32;  // stride byte offset: along MN
  d |= static_cast<uint64_t>(1u) << 46;                   // descriptor version (sm100)
  return d;
}

// 32 TMEM lanes (this warp's quarter) x 8 consecutive 32-bit columns -> 8 registers per thread, and back.
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// The registers of a load may be read only after its wait.
__device__ __forceinline__ void after_wait(uint32_t (&r)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) asm volatile("" : "+r"(r[i]));
}

// float8 e5m2 (1 sign, 5 exponent, 2 mantissa bits): nearest even, and back (exact).
__device__ __forceinline__ uint16_t e5m2x2_from_f16x2(__half2 h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&h)));
  return r;
}
__device__ __forceinline__ __half2 half2_from_e5m2x2(uint16_t c) {
  uint32_t u;
  asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(u) : "h"(c));
  return *reinterpret_cast<const __half2*>(&u);
}

// Whether any of the 256 softmax threads has `p` (named barrier 2).
__device__ __forceinline__ bool any_of_256(bool p) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 2, 256, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<int>(p))
      : "memory");
  __syncwarp();
  return r != 0;
}

// Eight values a lane, combined over the warp's 32 lanes (f: max or plus): lane l ends with value l & 7.  Halves
// of the values change hands at each of three steps, so it takes 9 shuffles, not 40.
template <typename F>
__device__ __forceinline__ float reduce_columns(const float* x, int lane, F f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = x[i];
#pragma unroll
  for (int h = 4; h >= 1; h >>= 1) {
    const bool up = (lane & h) != 0;
#pragma unroll
    for (int i = 0; i < h; ++i) {
      const float keep = up ? v[i + h] : v[i], give = up ? v[i] : v[i + h];
      v[i] = f(keep, __shfl_xor_sync(0xffffffffu, give, h));
    }
  }
  v[0] = f(v[0], __shfl_xor_sync(0xffffffffu, v[0], 8));
  return f(v[0], __shfl_xor_sync(0xffffffffu, v[0], 16));
}

constexpr int kRegsMisc = 48, kRegsSoftmax = 96;
static_assert(kRegsMisc + 2 * kRegsSoftmax == 3 * kRegsLaunch, "the split is the launch's registers");

template <int N>
struct Cfg {
  static constexpr int kStages = N <= 16 ? 3 : 2;  // K and V rings
  static constexpr int kPBufs = N == 32 ? 2 : 1;
  static constexpr int kQ = 2 * N * kHd;           // bytes of Qh | Ql
  static constexpr int kUnit = kKeys * 16;         // 16 columns of a term of P
  static constexpr int kP = 3 * N / 16 * kUnit;    // bytes of Pa | Pb | Pc
  static constexpr int kOffV = kStages * kTile, kOffQ = 2 * kStages * kTile, kOffP = kOffQ + kQ;
  static constexpr int kBytes = 1024 + kOffP + kPBufs * kP;
  static constexpr uint32_t kS = 0, kO = 2 * N;    // TMEM columns: S, then the three accumulators
  static constexpr uint32_t kCols = 5 * N <= 128 ? 128 : 256;
};

template <int N>
struct Bars {
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3];
  uint64_t q_ready, s_full, s_free, p_full[2], pv_done[2], o_final;
  uint32_t tmem;
  // of a stage's pages: log2 vs, 1 / vs, and ks over that of the first page of the 32 keys
  float4 scale[3][kKeys / 16];
  // x = S map + log2 vs - base: unscale ks of a column, for the first page of each 32 keys
  alignas(16) float map[3][4][N];
  alignas(16) float base[N], delta[N], factor[N];
  PagedRows<N> rows;
  float part[4][N];  // a warp's column maxima, at the end its column sums
};
template <int N>
constexpr bool two_ctas() { return Cfg<N>::kBytes + static_cast<int>(sizeof(Bars<N>)) + 1024 <= 228 * 1024 / 2; }
static_assert(two_ctas<16>() && two_ctas<32>() && two_ctas<48>(), "two CTAs per SM, with the system's 1 KB each");

// One item: `smem` 1024-byte aligned, `b` in static shared memory.
template <int N>
__device__ __forceinline__ void run(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint8_t* smem,
                                    Bars<N>& b) {
  using C = Cfg<N>;
  constexpr int kStages = C::kStages;
  uint8_t* sq = smem + C::kOffQ;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&b.k_full[i], 32);
      mbar_init(&b.k_empty[i], 1);
      mbar_init(&b.v_full[i], 32);
      mbar_init(&b.v_empty[i], 1);
    }
    mbar_init(&b.q_ready, 8);
    mbar_init(&b.s_full, 1);
    mbar_init(&b.s_free, 8);
    mbar_init(&b.p_full[0], 8);
    mbar_init(&b.p_full[1], 8);
    mbar_init(&b.pv_done[0], 1);
    mbar_init(&b.pv_done[1], 1);
    mbar_init(&b.o_final, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&b.tmem, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = b.tmem;
  pdl_trigger();
  pdl_wait();
  const PagedItem it = a.items[blockIdx.x];
  const int n_tiles = (it.key1 - it.key0 + kKeys - 1) / kKeys;

  if (warp < 4) set_registers<kRegsMisc, false>();
  if (warp == 0) {
    // ---------------- TMA producer: a lane a page ----------------
    const int ps = a.page_size, per_tile = kKeys >> a.page_shift, box = min(ps, 64);
    const int* table = a.table + static_cast<size_t>(it.req) * a.table_ld;
    const uint64_t policy = l2_policy_evict_first();
    int batch = -32, row = 0;  // first page of the 32 whose rows and scales the lanes hold
    float ks = 1.f;
    float4 sc = make_float4(0.f, 1.f, 1.f, 0.f);
    int issued = 0;
    for (int j = 0; j < n_tiles; ++j, ++issued) {
      const int page0 = (it.key0 + j * kKeys) >> a.page_shift, st = j % kStages;
      if (page0 + per_tile > batch + 32) {  // uniform
        batch = page0;
        const int p = page0 + lane;
        if (static_cast<long long>(p) * ps < it.key1) {
          const int id = max(paged_page_id(table[p], a.pages, a.err), 0);
          const size_t unit = static_cast<size_t>(id) * a.hkv + it.head;
          row = static_cast<int>(unit << a.page_shift);
          ks = __ldg(a.k_scale + unit);
          sc.x = __ldg(a.v_scale + unit);
        }
      }
      const int from = page0 - batch + (lane < per_tile ? lane : 0);
      const int src = a.layer_row + __shfl_sync(0xffffffffu, row, from);
      const bool live = lane < per_tile && static_cast<long long>(page0 + lane) * ps < it.key1;
      const uint32_t free_parity = ((j / kStages) & 1u) ^ 1u;
      auto load = [&](const CUtensorMap* map, uint64_t* bar, uint8_t* dst) {
        asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(ps * kHd)
                     : "memory");
        for (int r0 = 0; r0 < ps; r0 += box) tma_load_2d(dst + (lane * ps + r0) * kHd, map, bar, 0, src + r0, policy);
      };
      if (!__all_sync(0xffffffffu, mbar_wait(&b.k_empty[st], free_parity))) {
        report_wait(a.err, kErrTimeoutProducer, 41, a.total_rows, it.splits);
        break;
      }
      if (live) load(&tm_k, &b.k_full[st], smem + st * kTile);
      mbar_arrive(&b.k_full[st]);
      if (!__all_sync(0xffffffffu, mbar_wait(&b.v_empty[st], free_parity))) {
        report_wait(a.err, kErrTimeoutProducer, 47, a.total_rows, it.splits);
        (void)mbar_wait(&b.k_full[st], (j / kStages) & 1u);  // its K copies land first
        break;
      }
      if (live) load(&tm_v, &b.v_full[st], smem + C::kOffV + st * kTile);
      // the tile's scales (V's stage is free: its softmax is long past)
      const float ks_j = __shfl_sync(0xffffffffu, ks, from), vs_j = __shfl_sync(0xffffffffu, sc.x, from);
      const float ks_0 = __shfl_sync(0xffffffffu, ks_j, lane & ~1);  // (pages of 16: two to 32 keys)
      if (lane < per_tile) {  // a dead page's slot too: its keys' weights are 0, what multiplies them must be a number
        const float lv = __log2f(live ? vs_j : 1.f);
        b.scale[st][lane] = make_float4(lv, exp2_approx(-lv), a.page_shift == 4 && live ? ks_j / ks_0 : 1.f, 0.f);
      }
      if (j == 0 && !mbar_wait(&b.q_ready, 0))  // the queries' scales (the others' waits then expire too)
        report_wait(a.err, kErrTimeoutProducer, 50, a.total_rows, it.splits);
      __syncwarp();
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float kg = __shfl_sync(0xffffffffu, ks_j, (32 * g) >> a.page_shift);
        for (int n = lane; n < N; n += 32) b.map[st][g][n] = b.rows.unscale[n] * kg;
      }
      mbar_arrive(&b.v_full[st]);
      __syncwarp();
    }
    for (int j = max(0, issued - kStages); j < issued; ++j)  // every copy landed before leaving
      if (!mbar_wait(&b.k_full[j % kStages], (j / kStages) & 1u) || !mbar_wait(&b.v_full[j % kStages], (j / kStages) & 1u))
        break;
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t id_s = idesc_s(2 * N), id_o = idesc_o(3 * N);
      int site = 0;
      if (!mbar_wait(&b.q_ready, 0)) site = 42;
      for (int j = 0; j <= n_tiles && site == 0; ++j) {
        if (j < n_tiles) {  // S_j^T = K_j (Qh | Ql)^T
          const int st = j % kStages;
          if (!mbar_wait(&b.k_full[st], (j / kStages) & 1u)) {
            site = 43;
            break;
          }
          if (!mbar_wait(&b.s_free, (j & 1u) ^ 1u)) {
            site = 44;
            break;
          }
          tc_fence_after_sync();
          const uint64_t ad = umma_desc_sw128(smem + st * kTile), qd = umma_desc_sw128(sq);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_f8(tmem + C::kS, ad + 2 * k, qd + 2 * k, id_s, k > 0 ? 1u : 0u);
          tc_commit(&b.s_full);
          tc_commit(&b.k_empty[st]);
        }
        if (j >= 1) {  // O^T += V_i^T (Pa | Pb | Pc)_i^T, i = j - 1
          const int i = j - 1, st = i % kStages;
          if (!mbar_wait(&b.p_full[i & 1], (i >> 1) & 1u)) {
            site = 45;
            break;
          }
          tc_fence_after_sync();
          const uint8_t* p = smem + C::kOffP + (i % C::kPBufs) * C::kP;
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 keys a step: four 8-row groups of V and of P
            mma_f8(tmem + C::kO, umma_desc_sw128_mn(smem + C::kOffV + st * kTile + k * 4096, 0, 1024),
                   umma_desc_mn(p + k * 512, C::kUnit, 128), id_o, (i > 0 || k > 0) ? 1u : 0u);
          tc_commit(&b.pv_done[i & 1]);
          tc_commit(&b.v_empty[st]);
          if (i == n_tiles - 1) tc_commit(&b.o_final);
        }
      }
      if (site != 0) report_wait(a.err, kErrTimeoutMma, site, a.total_rows, it.splits);
    }
  } else if (warp >= 4) {
    set_registers<kRegsSoftmax, true>();
    if (threadIdx.x - 128 < N) b.base[threadIdx.x - 128] = 0.f;
    paged_stage_queries<N, true>(a, it, sq, sq + N * kHd, b.rows, threadIdx.x - 128);
    if (lane == 0) mbar_arrive(&b.q_ready);
    named_sync(2, 256);
    // ---------------- softmax: a key a thread, half the columns a warpgroup ----------------
    constexpr int H = N / 2;
    const int q4 = warp & 3, key_lane = q4 * 32 + lane;  // TMEM lane
    const int col0 = warp < 8 ? 0 : H;
    const uint32_t lane_base = (static_cast<uint32_t>(q4 * 32) << 16) + col0;
    // keys from which some row's mask ends (rows are in token order, so the first has the least)
    const int lim_min = b.rows.lim[0];
    const bool mine = it.rows > col0;  // rows among this warpgroup's columns
    float sum[H];
#pragma unroll
    for (int n = 0; n < H; ++n) sum[n] = 0.f;
    bool ok = true;

    for (int j = 0; j < n_tiles; ++j) {
      const int st = j % kStages;
      const int key = it.key0 + j * kKeys + key_lane;
      ok = ok && mbar_wait(&b.v_full[st], (j / kStages) & 1u);
      const float4 sc = b.scale[st][key_lane >> a.page_shift];
      ok = ok && mbar_wait(&b.s_full, j & 1u);
      __syncwarp();
      tc_fence_after_sync();
      // (no branch on the number of rows between here and the store of P: straight-line code hides the latencies)
      float s[H], top0 = -INFINITY, top1 = -INFINITY;
      if (mine) {
        uint32_t hi[H / 8][8], lo[H / 8][8];
#pragma unroll
        for (int c = 0; c < H / 8; ++c) {
          tmem_ld_32x32b_x8(tmem + lane_base + C::kS + c * 8, hi[c]);
          tmem_ld_32x32b_x8(tmem + lane_base + C::kS + N + c * 8, lo[c]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < H / 8; ++c) {
          after_wait(hi[c]);
          after_wait(lo[c]);
        }
#pragma unroll
        for (int n = 0; n < H; ++n) s[n] = __uint_as_float(hi[n / 8][n % 8]) + __uint_as_float(lo[n / 8][n % 8]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.s_free);
      if (mine) {
        const float4* map = reinterpret_cast<const float4*>(&b.map[st][q4][col0]);
        const float4* base = reinterpret_cast<const float4*>(&b.base[col0]);
        if (a.page_shift == 4) {
#pragma unroll
          for (int n = 0; n < H; ++n) s[n] *= sc.z;
        }
#pragma unroll
        for (int i = 0; i < H / 4; ++i) {
          const float4 m = map[i], bs = base[i];
          float* x = &s[4 * i];
          x[0] = fmaf(x[0], m.x, sc.x - bs.x);
          x[1] = fmaf(x[1], m.y, sc.x - bs.y);
          x[2] = fmaf(x[2], m.z, sc.x - bs.z);
          x[3] = fmaf(x[3], m.w, sc.x - bs.w);
        }
        if (it.key0 + (j + 1) * kKeys > lim_min) {
#pragma unroll
          for (int n = 0; n < H; ++n)
            if (key >= b.rows.lim[col0 + n]) s[n] = -INFINITY;  // (also what a dead key's garbage gave)
        }
#pragma unroll
        for (int n = 0; n < H; n += 2) {
          top0 = fmaxf(top0, s[n]);
          top1 = fmaxf(top1, s[n + 1]);
        }
      }
      if (any_of_256(fmaxf(top0, top1) > kTrip || j == 0 || !ok)) {
        if (any_of_256(!ok)) {  // a wait expired: all eight warps leave together
          ok = false;
          break;
        }
        // move the bases of the columns that need it to their maximum over these 128 keys
        if (mine) {
#pragma unroll
          for (int c = 0; c < H / 8; ++c) {
            const float m = reduce_columns(&s[c * 8], lane, [](float x, float y) { return fmaxf(x, y); });
            if (lane < 8) b.part[q4][col0 + c * 8 + lane] = m;
          }
        }
        named_sync(2, 256);
        const int t = threadIdx.x - 128;
        if (t < N) {
          const float m = fmaxf(fmaxf(b.part[0][t], b.part[1][t]), fmaxf(b.part[2][t], b.part[3][t]));
          const bool move = t < it.rows && m > -INFINITY && m < INFINITY && (j == 0 || m > kTrip);
          const float d = move ? kSeat - m : 0.f;  // new weights are 2^d times the old
          b.delta[t] = d;
          b.factor[t] = exp2f(d);
          b.base[t] -= d;
        }
        named_sync(2, 256);
        if (j > 0) {  // O of the earlier tiles: their last product has to land first
          ok = mbar_wait(&b.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1u);
          __syncwarp();
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < (mine ? H / 8 : 0); ++c) {
#pragma unroll 1
            for (int term = 0; term < 3; ++term) {
              uint32_t v[8];
              const uint32_t at = tmem + lane_base + C::kO + term * N + c * 8;
              tmem_ld_32x32b_x8(at, v);
              tmem_ld_wait();
              after_wait(v);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * b.factor[col0 + c * 8 + i]);
              tmem_st_32x32b_x8(at, v);
            }
          }
          tmem_st_wait();
          tc_fence_before_sync();
        }
        if (mine) {
#pragma unroll
          for (int n = 0; n < H; ++n) {
            s[n] += b.delta[col0 + n];
            if (j > 0) sum[n] *= b.factor[col0 + n];
          }
        }
      }
      // P_j: with two buffers P_{j-2} has left this one (S_j's commit covered every product issued before it)
      if (C::kPBufs == 1 && j > 0) ok = ok && mbar_wait(&b.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1u);
      uint8_t* p = smem + C::kOffP + (j % C::kPBufs) * C::kP + key_lane * 16;
      if (mine) {
#pragma unroll
      for (int c = 0; c < H / 8; ++c) {
        uint32_t w[3][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = c * 8 + 2 * i;
          const float p0 = exp2_approx(s[n]), p1 = exp2_approx(s[n + 1]);
          sum[n] = fmaf(p0, sc.y, sum[n]);
          sum[n + 1] = fmaf(p1, sc.y, sum[n + 1]);
          const __half2 h = __floats2half2_rn(p0, p1);
          const uint16_t ta = e5m2x2_from_f16x2(h);
          // remainders: exact, at most 2^-3 and 2^-4 of the power of two below their term, so scaled they stay in range
          const __half2 r1 = __hmul2(__hsub2(h, half2_from_e5m2x2(ta)), __float2half2_rn(8.f));
          const uint16_t tb = e5m2x2_from_f16x2(r1);
          const uint16_t tc = e5m2x2_from_f16x2(__hmul2(__hsub2(r1, half2_from_e5m2x2(tb)), __float2half2_rn(32.f)));
          const int k = i >> 1;
          if ((i & 1) == 0) w[0][k] = ta, w[1][k] = tb, w[2][k] = tc;
          else w[0][k] |= static_cast<uint32_t>(ta) << 16, w[1][k] |= static_cast<uint32_t>(tb) << 16, w[2][k] |= static_cast<uint32_t>(tc) << 16;
        }
        const int col = col0 + c * 8;  // 8 of the 16 columns of a core matrix
#pragma unroll
        for (int term = 0; term < 3; ++term)
          *reinterpret_cast<uint2*>(p + (term * (N / 16) + (col >> 4)) * C::kUnit + (col & 8)) = make_uint2(w[term][0], w[term][1]);
      }
      }
      if (key >= it.key1) {  // rows past the range hold anything: their weight is 0, their values must be
        uint4* v = reinterpret_cast<uint4*>(smem + C::kOffV + st * kTile + key_lane * kHd) + (col0 == 0 ? 0 : 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.p_full[j & 1]);
    }

    // row sums over the 128 keys
    if (mine) {
#pragma unroll
      for (int c = 0; c < H / 8; ++c) {
        const float l = reduce_columns(&sum[c * 8], lane, [](float x, float y) { return x + y; });
        if (lane < 8) b.part[q4][col0 + c * 8 + lane] = l;
      }
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&b.o_final, 0));
    if (!ok && lane == 0) report_wait(a.err, kErrTimeoutEpilogue, 46, a.total_rows, it.splits);
    named_sync(2, 256);
    const int t = threadIdx.x - 128;
    if (t < N) {
      float l = b.part[0][t] + b.part[1][t] + b.part[2][t] + b.part[3][t];
      if (l == INFINITY) l = NAN;  // a score past fp32: P's terms saturate, the quotient must not pass for a result
      b.factor[t] = it.splits == 1 ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
      b.delta[t] = l;
    }
    named_sync(2, 256);
    tc_fence_after_sync();
    // O^T: lane = head column, a row a TMEM column.  A split tile leaves its partial: [N][128], then [N] (base, sum)
    bf16* out = static_cast<bf16*>(a.out) + key_lane;
    float* part = reinterpret_cast<float*>(a.part + it.part) + key_lane;
    if (mine) {
#pragma unroll
      for (int c = 0; c < H / 8; ++c) {
        uint32_t v[3][8];
#pragma unroll
        for (int term = 0; term < 3; ++term) tmem_ld_32x32b_x8(tmem + lane_base + C::kO + term * N + c * 8, v[term]);
        tmem_ld_wait();
#pragma unroll
        for (int term = 0; term < 3; ++term) after_wait(v[term]);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = (__uint_as_float(v[0][i]) + (__uint_as_float(v[1][i]) + __uint_as_float(v[2][i]) * 0.03125f) * 0.125f) *
                 b.factor[col0 + c * 8 + i];
        const int n0 = col0 + c * 8;
        if (it.splits == 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n0 + i < it.rows) out[static_cast<size_t>(b.rows.out[n0 + i]) * kHd] = __float2bfloat16_rn(x[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n0 + i < it.rows) part[(n0 + i) * kHd] = x[i];
        }
      }
    }
    if (it.splits > 1) {
      if (t < it.rows)
        reinterpret_cast<float2*>(reinterpret_cast<float*>(a.part + it.part) + N * kHd)[t] = make_float2(b.base[t], b.delta[t]);
    }
    tc_fence_before_sync();
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  // Back to the launch's split.  Only here, past the barrier: a warp without a role that took its registers
  // back any earlier would leave the softmax waiting for them.
  if (warp >= 4) set_registers<kRegsLaunch, false>();
  else set_registers<kRegsLaunch, true>();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::kCols);
  }
  if (it.splits > 1) paged_join<N, kThreads>(a, it, b.rows.out, smem);
}

}  // namespace paged_tc
}  // namespace fdllm
