// Attention over a paged 8-bit KV cache on the 5th-generation tensor cores for many query rows
// (fdllm_paged_attention, bf16, head_dim 128): block steps and prompts.  Semantics as in paged_attention.cu.
//
// The query rows of one request and KV head are its (token, query head) pairs.  A CTA takes one item of the
// plan, a tile of at most 128 rows and a range of keys, in tiles of 64 keys with the rows on the MMA's M side:
//   S [128, 64]   = (Qh + Ql) K^T     A: the queries (e4m3 in shared memory), B: the K tile as cached (e4m3)
//   P [128, 64]   = 2^(a S + log2 vs - B)
//   O [128, 128] += P V               A: P (f16 in TMEM, over its S), B: V widened to f16 (exact)
// Precision: a bf16 query has 8 significant bits, so Q = Qh + Ql under one power of two per row (largest element
// in [2^7, 2^8)) is exact for elements above 2^-10 of the row's largest and to 2^-18 of it below; two 8-bit
// products cost one 16-bit product's time and K needs no widening.  P keeps 11 bits and weights down to 2^-32 of
// the largest.  A row's base B moves only when a weight passes 2^kTrip (then its maximum sits at 2^kSeat); then
// its row of O in TMEM is scaled.  log2 vs in the exponent keeps P in range whatever the page scales are; the row
// sum takes it back out.
//
// Roles (384 threads, registers moved to the softmax): warp 0 the TMA producer (a lane a page; page ids and
// scales 32 pages at a time), warp 1 issues S and owns TMEM, warp 2 issues P V (one thread for both took 128 us for
// 123 below: an issue blocks while the tensor core is busy), warps 4-7 the softmax, a row a thread, warps 8-11 widen
// V.  S, P and the widened V are double-buffered: S_{j+1} and V_{j+1} are made while tile j is in the softmax.  Two
// CTAs share an SM (256 TMEM columns and 110 KB each), so one's softmax covers the other's products.
//
// Measured, 12/2 heads of 128: 2 prompts of 4096 tokens, block-causal, 123 us, 845 TFLOP/s of the formula's two
// products; 32 block steps of 32 rows over 512 to 1024 keys 22.1 us, 8 over 4096 keys 27.9.
//
// What bounds it: no one pipe.  A tile of 8192 scores takes 1260 clocks of an SM (296 items, 1.28 us a key tile); over
// the prompts the tensor core with its operand reads is busy 62 % (Q is read twice for S, at 64 bytes a clock), the
// exponentials 42 % and issue 57 %.  The chain S, softmax, P, O of two CTAs does not keep any of them full, each wait on
// a barrier in it costs 100 clocks, and launch, prologues and epilogues of 768 items, 27 us, are a fifth of the prompts'
// time.  What did not shorten it, of 134 us then: S of two tiles in one product (159), half a row a thread on eight
// softmax warps (134.5), one S and two P buffers (140), that with Qh in TMEM (147).
//
// A tile whose keys are split over several items joins them through the workspace: the last item to arrive adds the
// partials in item order (paged_join).
#pragma once
#include "paged_mma.cuh"

namespace fdllm {
namespace paged_wide {

constexpr int kRows = 128, kKeys = 64, kHd = 128;
constexpr int kTile = kKeys * kHd;      // bytes of a K or V tile as cached
constexpr int kQ = kRows * kHd;         // bytes of Qh or Ql
constexpr int kV16 = kKeys * kHd * 2;   // bytes of a widened V tile: two sub-tiles of 64 columns
constexpr int kOffQ = 0, kOffK = 2 * kQ, kOffV = kOffK + 2 * kTile, kOffV16 = kOffV + 2 * kTile;
constexpr int kBytes = 1024 + kOffV16 + 2 * kV16;
constexpr uint32_t kTmemS = 0, kTmemO = 128, kTmemCols = 256;  // S: two buffers of 64 columns
constexpr float kTrip = 15.f, kSeat = 8.f;
constexpr int kRegsMisc = 48, kRegsSoftmax = 144, kRegsWiden = 48;
static_assert(kRegsMisc + kRegsSoftmax + kRegsWiden == 3 * kRegsLaunch, "the split is the launch's registers");
static_assert(2 * (kBytes + 2048) <= 228 * 1024, "two CTAs per SM");
static_assert(kRows * kHd * 4 <= kOffV16, "O over the queries and the rings");

// Instruction descriptors, fp32 accumulator, M 128: S (kind::f8f6f4, e4m3, K-major) and O (kind::f16, f16, A in
// TMEM, B MN-major).
constexpr uint32_t kIdescS = (1u << 4) | ((kKeys >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((kHd >> 3) << 17) | ((128u >> 4) << 24);

// D[tmem] (+)= A[tmem] * B[smem]^T, f16 operands (two to a TMEM column of A).
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {  // a load's registers are read only after its wait
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct Bars {
  uint64_t k_full[2], v_full[2], v_empty[2];
  uint64_t q_ready, s_full[2], pv_ready[2], pv_done[2], o_final;  // pv_ready: P and the widened V
  uint32_t tmem;
  PagedRows<kRows> rows;
  float4 scale[4][kKeys / 16];  // of tile j & 3, its 16-key groups: ks, log2 vs, 1 / vs
};

// One item: `smem` 1024-byte aligned, `b` in static shared memory.
__device__ __forceinline__ void run(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint8_t* smem,
                                    Bars& b) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b.k_full[i], 32);
      mbar_init(&b.v_full[i], 32);
      mbar_init(&b.v_empty[i], 4);
      mbar_init(&b.s_full[i], 2);
      mbar_init(&b.pv_ready[i], 8);
      mbar_init(&b.pv_done[i], 1);
    }
    mbar_init(&b.q_ready, 8);
    mbar_init(&b.o_final, 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&b.tmem, kTmemCols);
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

  if (warp >= 4) {
    paged_stage_queries<kRows, false>(a, it, smem + kOffQ, smem + kOffQ + kQ, b.rows, threadIdx.x - 128);
    if (lane == 0) mbar_arrive(&b.q_ready);
    named_sync(2, 256);
  }

  if (warp < 4) set_registers<kRegsMisc, false>();
  if (warp == 0) {
    // ---------------- TMA producer: a lane a page ----------------
    const int ps = a.page_size, per_tile = max(kKeys >> a.page_shift, 1), box = min(ps, kKeys);
    const int* table = a.table + static_cast<size_t>(it.req) * a.table_ld;
    const uint64_t policy = l2_policy_evict_last();  // the other tiles of this request read them too
    int batch = -32, row = 0;  // first page of the 32 whose rows and scales the lanes hold
    float ks = 1.f, vs = 1.f;
    int issued = 0;
    for (int j = 0; j < n_tiles; ++j, ++issued) {
      const int key = it.key0 + j * kKeys, page0 = key >> a.page_shift, st = j & 1;
      if (page0 + per_tile > batch + 32) {  // uniform
        batch = page0;
        const int p = page0 + lane;
        if (static_cast<long long>(p) * ps < it.key1) {
          const int id = max(paged_page_id(table[p], a.pages, a.err), 0);
          const size_t unit = static_cast<size_t>(id) * a.hkv + it.head;
          row = static_cast<int>(unit << a.page_shift);
          ks = __ldg(a.k_scale + unit);
          vs = __ldg(a.v_scale + unit);
        }
      }
      const int from = page0 - batch + (lane < per_tile ? lane : 0);
      const int src = a.layer_row + __shfl_sync(0xffffffffu, row, from) + (key & (ps - 1));  // (half of a page of 128)
      const bool live = lane < per_tile && static_cast<long long>(page0 + lane) * ps < it.key1;
      const uint32_t free_parity = ((j >> 1) & 1u) ^ 1u;
      auto load = [&](const CUtensorMap* map, uint64_t* bar, uint8_t* dst) {
        asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(box * kHd)
                     : "memory");
        tma_load_2d(dst + lane * box * kHd, map, bar, 0, src, policy);
      };
      // K_{j-2} has been used once S_{j-2} is there
      if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(&b.s_full[st], free_parity))) {
        report_wait(a.err, kErrTimeoutProducer, 51, a.total_rows, it.splits);
        break;
      }
      if (live) load(&tm_k, &b.k_full[st], smem + kOffK + st * kTile);
      // the scales of the tile's 16-key groups.  Slot j & 3: S_{j-2} is done, so P_{j-4} is used and its softmax past.
      // They reach the softmax through the MMA issuer, which waits for K and arrives for S (a wait costs 100 clocks).
      const int group_page = page0 - batch + ((16 * (lane & 3)) >> a.page_shift);
      const float kg = __shfl_sync(0xffffffffu, ks, group_page), vg = __shfl_sync(0xffffffffu, vs, group_page);
      if (lane < 4) {
        const float lv = __log2f(vg);
        b.scale[j & 3][lane] = make_float4(kg, lv, exp2_approx(-lv), 0.f);
      }
      __syncwarp();
      mbar_arrive(&b.k_full[st]);
      if (!__all_sync(0xffffffffu, mbar_wait(&b.v_empty[st], free_parity))) {
        report_wait(a.err, kErrTimeoutProducer, 52, a.total_rows, it.splits);
        (void)mbar_wait(&b.k_full[st], (j >> 1) & 1u);  // its K copies land first
        break;
      }
      if (live) load(&tm_v, &b.v_full[st], smem + kOffV + st * kTile);
      mbar_arrive(&b.v_full[st]);
      __syncwarp();
    }
    for (int j = max(0, issued - 2); j < issued; ++j)  // every copy landed before leaving
      if (!mbar_wait(&b.k_full[j & 1], (j >> 1) & 1u) || !mbar_wait(&b.v_full[j & 1], (j >> 1) & 1u)) break;
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- issuer of S_j = (Qh + Ql) K_j^T, into the buffer that P_{j-2} has left ----------------
      int site = 0;
      if (!mbar_wait(&b.q_ready, 0)) site = 53;
      const uint64_t qh = umma_desc_sw128(smem + kOffQ), ql = umma_desc_sw128(smem + kOffQ + kQ);
      for (int j = 0; j < n_tiles && site == 0; ++j) {
        const int st = j & 1;
        if (!mbar_wait(&b.k_full[st], (j >> 1) & 1u)) {
          site = 54;
          break;
        }
        if (j >= 2 && !mbar_wait(&b.pv_done[st], ((j - 2) >> 1) & 1u)) {
          site = 55;
          break;
        }
        tc_fence_after_sync();
        const uint64_t kd = umma_desc_sw128(smem + kOffK + st * kTile);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mma_f8(tmem + kTmemS + st * kKeys, qh + 2 * k, kd + 2 * k, kIdescS, k > 0 ? 1u : 0u);
          mma_f8(tmem + kTmemS + st * kKeys, ql + 2 * k, kd + 2 * k, kIdescS, 1u);
        }
        tc_commit(&b.s_full[st]);
        mbar_arrive(&b.s_full[st]);  // releases the scales
      }
      if (site != 0) report_wait(a.err, kErrTimeoutMma, site, a.total_rows, it.splits);
    }
  } else if (warp == 2) {
    if (lane == 0) {
      // ---------------- issuer of O += P_j V_j ----------------
      bool ok = true;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int buf = j & 1;
        ok = mbar_wait(&b.pv_ready[buf], (j >> 1) & 1u);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 16 keys a step: 8 columns of P, two 8-row groups of V
          mma_f16_ta(tmem + kTmemO, tmem + kTmemS + buf * kKeys + 8 * k,
                     umma_desc_sw128_mn(smem + kOffV16 + buf * kV16 + k * 2048, kV16 / 2, 1024), kIdescO,
                     (j > 0 || k > 0) ? 1u : 0u);
        tc_commit(&b.pv_done[buf]);
        if (j == n_tiles - 1) tc_commit(&b.o_final);
      }
      if (!ok) report_wait(a.err, kErrTimeoutMma, 56, a.total_rows, it.splits);
    }
  } else if (warp >= 8) {
    set_registers<kRegsWiden, false>();
    // ---------------- V in f16: a key a lane, half a row a thread ----------------
    const int half = warp & 1, k = 32 * ((warp - 8) >> 1) + lane;  // key of the tile
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int st = j & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&b.v_full[st], (j >> 1) & 1u));
      if (!ok) break;
      const uint8_t* src = smem + kOffV + st * kTile + k * kHd;
      // rows past the range hold anything: their weight is 0, their values must be
      const bool dead = it.key0 + j * kKeys + k >= it.key1;
      uint4 u[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        u[c] = *reinterpret_cast<const uint4*>(src + (((4 * half + c) ^ (k & 7)) << 4));
        if (dead) u[c] = make_uint4(0u, 0u, 0u, 0u);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.v_empty[st]);
      if (j >= 2) {  // P_{j-2} V_{j-2} has left the buffer
        ok = __all_sync(0xffffffffu, mbar_wait(&b.pv_done[st], ((j - 2) >> 1) & 1u));
        if (!ok) break;
      }
      uint8_t* dst = smem + kOffV16 + st * kV16 + half * (kV16 / 2) + k * 128;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t e[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
        uint32_t f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = f16x2_from_e4m3x2(static_cast<uint16_t>(e[i]));
          f[2 * i + 1] = f16x2_from_e4m3x2(static_cast<uint16_t>(e[i] >> 16));
        }
        *reinterpret_cast<uint4*>(dst + (((2 * c) ^ (k & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<uint4*>(dst + (((2 * c + 1) ^ (k & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.pv_ready[st]);
    }
    if (!ok && lane == 0) report_wait(a.err, kErrTimeoutEpilogue, 58, a.total_rows, it.splits);
  } else if (warp >= 4) {
    set_registers<kRegsSoftmax, true>();
    // ---------------- softmax and output: a row a thread ----------------
    const int q4 = warp & 3, tid = q4 * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(q4 * 32) << 16;
    const bool valid = tid < it.rows;
    const int lim = valid ? b.rows.lim[tid] : it.key0;
    const float unscale = b.rows.unscale[tid];
    float base = 0.f, l = 0.f;
    bool ok = true, seated = false;  // seated: the base has been set (the row has attended a key)
    for (int j = 0; j < n_tiles; ++j) {
      const int sb = j & 1, key0 = it.key0 + j * kKeys;
      ok = __all_sync(0xffffffffu, mbar_wait(&b.s_full[sb], (j >> 1) & 1u));
      if (!ok) break;
      if (q4 * 32 >= it.rows) {  // only padding rows: whatever P holds there stays in their rows of O
        if (lane == 0) mbar_arrive(&b.pv_ready[sb]);
        continue;
      }
      tc_fence_after_sync();
      const uint32_t s_at = tmem + lane_base + kTmemS + sb * kKeys;
      float x[kKeys];
      {
        uint32_t v0[32], v1[32];
        tmem_ld_32x32b_x32(s_at, v0);
        tmem_ld_32x32b_x32(s_at + 32, v1);
        tmem_ld_wait();
        after_wait(v0);
        after_wait(v1);
#pragma unroll
        for (int c = 0; c < 32; ++c) x[c] = __uint_as_float(v0[c]), x[32 + c] = __uint_as_float(v1[c]);
      }
      float inv_vs[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 sc = b.scale[j & 3][g];
        const float m = unscale * sc.x, c = sc.y - base;
        inv_vs[g] = sc.z;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[16 * g + i] = fmaf(x[16 * g + i], m, c);
      }
      if (__any_sync(0xffffffffu, key0 + kKeys > lim)) {  // (also what keys past the range gave)
#pragma unroll
        for (int c = 0; c < kKeys; ++c)
          if (key0 + c >= lim) x[c] = -INFINITY;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < kKeys; ++c) top[c & 3] = fmaxf(top[c & 3], x[c]);
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      const bool move = mx < INFINITY && (mx > kTrip || (!seated && mx > -INFINITY));
      if (__any_sync(0xffffffffu, move)) {
        const float d = move ? kSeat - mx : 0.f, f = exp2_approx(d);  // new weights are 2^d times the old
        if (__any_sync(0xffffffffu, move && seated)) {  // O holds earlier tiles: their last product has to land first
          ok = __all_sync(0xffffffffu, mbar_wait(&b.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1u));
          if (!ok) break;
          tc_fence_after_sync();
#pragma unroll 1
          for (int c0 = 0; c0 < kHd; c0 += 32) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(tmem + lane_base + kTmemO + c0, v);
            tmem_ld_wait();
            after_wait(v);
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * (seated ? f : 1.f));
            tmem_st_32x32b_x32(tmem + lane_base + kTmemO + c0, v);
          }
          tmem_st_wait();
        }
        base -= d;
        l *= seated ? f : 1.f;
        seated |= move;
#pragma unroll
        for (int c = 0; c < kKeys; ++c) x[c] += d;
      }
      uint32_t w[32];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float p0 = 0.f, p1 = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float e0 = exp2_approx(x[16 * g + i]), e1 = exp2_approx(x[16 * g + i + 1]);
          p0 += e0;
          p1 += e1;
          w[8 * g + i / 2] = pack_f16x2(e0, e1);
        }
        l = fmaf(p0 + p1, inv_vs[g], l);
      }
      tmem_st_32x32b_x32(s_at, w);  // P_j over S_j
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.pv_ready[sb]);
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&b.o_final, 0));
    if (!ok && lane == 0) report_wait(a.err, kErrTimeoutEpilogue, 59, a.total_rows, it.splits);
    tc_fence_after_sync();
    // O into shared memory, 16-byte units xor row mod 8 (the queries and the rings are done with): bf16, or fp32 for a
    // partial; every warp then writes whole rows.
    const float inv = it.splits > 1 ? 1.f : l != 0.f ? 1.f / l : 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < kHd; c0 += 32) {
      uint32_t v[32];
      tmem_ld_32x32b_x32(tmem + lane_base + kTmemO + c0, v);
      tmem_ld_wait();
      after_wait(v);
      auto at = [&](int c) { return __uint_as_float(v[c]) * inv; };
      if (it.splits == 1) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(smem + tid * 256 + (((c0 / 8 + c) ^ (tid & 7)) << 4)) =
              make_uint4(pack_bf16x2(at(8 * c), at(8 * c + 1)), pack_bf16x2(at(8 * c + 2), at(8 * c + 3)),
                         pack_bf16x2(at(8 * c + 4), at(8 * c + 5)), pack_bf16x2(at(8 * c + 6), at(8 * c + 7)));
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<float4*>(smem + tid * 512 + (((c0 / 4 + c) ^ (tid & 7)) << 4)) =
              make_float4(at(4 * c), at(4 * c + 1), at(4 * c + 2), at(4 * c + 3));
      }
    }
    if (it.splits > 1 && valid) reinterpret_cast<float2*>(a.part + it.part + kRows * (kHd / 4))[tid] = make_float2(base, l);
    tc_fence_before_sync();
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  // Back to the launch's split.  Only here, past the barrier: a warp without a role that took its registers
  // back any earlier would leave the softmax waiting for them.
  if (warp >= 4 && warp < 8) set_registers<kRegsLaunch, false>();
  else set_registers<kRegsLaunch, true>();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (it.splits == 1) {
    for (int i = threadIdx.x; i < it.rows * 16; i += kThreads) {
      const int row = i >> 4, c = i & 15;
      reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) + static_cast<size_t>(b.rows.out[row]) * kHd)[c] =
          *reinterpret_cast<const uint4*>(smem + row * 256 + ((c ^ (row & 7)) << 4));
    }
    return;
  }
  // a split tile leaves its partial: [128][128], then [128] (base, sum)
  for (int i = threadIdx.x; i < it.rows * 32; i += kThreads) {
    const int row = i >> 5, c = i & 31;
    a.part[it.part + i] = *reinterpret_cast<const float4*>(smem + row * 512 + ((c ^ (row & 7)) << 4));
  }
  paged_join<kRows, kThreads>(a, it, b.rows.out, smem);
}

}  // namespace paged_wide
}  // namespace fdllm
