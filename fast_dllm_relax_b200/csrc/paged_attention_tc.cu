// Attention over a paged 8-bit KV cache on the 5th-generation tensor cores (fdllm_paged_attention, bf16,
// head_dim 128).  Semantics as in paged_attention.cu; the codes are never widened.
//
// The query rows of one request and KV head are its (token, query head) pairs.  A CTA takes one item of the
// plan, a tile of at most N rows and a range of keys, in tiles of 128 keys with the keys on the MMA's M side:
//   S^T [128 keys, N]   = K Q^T        A: the K tile (e4m3, K-major), B: Q (e4m3, K-major)
//   P^T [128 keys, N]   = 2^(a S + log2 vs - B)
//   O^T [128 columns, N] += V^T P^T    A: the V tile (f16, MN-major), B: P (f16, MN-major)
// so N follows the number of query rows (a lone token needs 16 columns, not 128 rows of padding), and a thread
// of the softmax holds one key and all rows: the page's scales are one pair a thread.
//
// Precision.  K is used as it is cached.  A bf16 query has 8 significant bits: Q = Qh + Ql, both e4m3 under one
// power of two per row (largest element in [2^7, 2^8)), exact for elements above 2^-10 of the row's largest and
// to 2^-18 of it below; two 8-bit products cost one 16-bit product's time, and K needs no widening.  P would
// need three e4m3 terms to keep small weights, so the second product is in f16 (11 bits, weights down to 2^-32
// of the largest), and V is widened on the way (exact).  Each column's base B moves only when a weight passes
// 2^kTrip (then its maximum sits at 2^kSeat): one block-wide vote a tile instead of a maximum over 128 lanes.
// log2 vs in the exponent keeps P in range whatever the page scales are; the row sums take it back out.
//
// Roles (384 threads, registers moved to the softmax): warp 0 the TMA producer (a lane a page; page ids and
// scales 32 pages at a time), warp 1 the MMA issuer and TMEM owner, warps 4-7 the softmax, a key a thread, warps
// 8-11 widen V, 64 keys at a time so that a half tile's product overlaps the other half's widening.  S^T is
// double-buffered: S_{j+1} is computed while tile j is in the softmax.  K and V have rings of their own: a V
// stage is free once widened, a K stage once its scores are computed (16 rows) or, where P replaces K in it to
// leave room for two CTAs on an SM, once P is used.
//
// A tile whose keys are split over several items joins them through the workspace as in
// paged_attention_narrow.cu: the last item to arrive adds the partials in item order.
#include "paged.h"

namespace fdllm {

namespace {

constexpr int kKeys = 128;
constexpr int kHd = 128;
constexpr int kTile = kKeys * kHd;  // bytes of a K or V tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTrip = 15.f, kSeat = 8.f;

// Instruction descriptors, fp32 accumulator, M 128: S = K Q^T (kind::f8f6f4, both e4m3 and K-major) and
// O^T = V^T P^T (kind::f16, both f16 and MN-major).
constexpr uint32_t idesc_s(int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24); }
constexpr uint32_t idesc_o(int n) { return idesc_s(n) | (1u << 15) | (1u << 16); }

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 operands, fp32 accumulate, one CTA.
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

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

// 16 registers per thread -> 32 TMEM lanes x 16 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Whether any of the 128 softmax threads has `p` (named barrier 2).
__device__ __forceinline__ bool any_of_128(bool p) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 2, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<int>(p))
      : "memory");
  __syncwarp();
  return r != 0;
}

// Order-preserving map of floats to unsigned ints (for the integer warp reductions).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t r) {
  return __uint_as_float((r & 0x80000000u) ? (r & 0x7FFFFFFFu) : ~r);
}

constexpr int kStages = 2;

template <int N>
struct Cfg {
  static constexpr bool kOwnP = N <= 16;   // P has its own buffers (two); else it replaces K in its stage
  static constexpr int kQ = N * kHd;       // bytes of Qh or Ql
  static constexpr int kP = kKeys * N * 2; // bytes of P
  static constexpr int kOffK = 0, kOffV = kStages * kTile;      // rings
  static constexpr int kOffV16 = kOffV + kStages * kTile;       // two sub-tiles of 64 columns
  static constexpr int kOffQ = kOffV16 + 2 * kTile;
  static constexpr int kOffP = kOffQ + 2 * kQ;
  static constexpr int kBytes = 1024 + kOffP + (kOwnP ? 2 * kP : 0);
  static constexpr uint32_t kS = 0, kO = 2 * N;  // TMEM columns: S (two buffers), O
  static constexpr uint32_t kCols = 3 * N <= 64 ? 64 : 3 * N <= 128 ? 128 : 256;
  static_assert(kP <= kTile, "P replaces K in its stage");
};

constexpr int kThreads = 384;
constexpr int kRegsLaunch = 80, kRegsMisc = 48, kRegsSoftmax = 144, kRegsWiden = 48;
static_assert(kRegsMisc + kRegsSoftmax + kRegsWiden == 3 * kRegsLaunch, "the split is the launch's registers");

template <int N>
struct Bars {
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t q_ready, s_full[2], s_free[2], p_full, w_full[2], pv_done[2], o_final;
  uint32_t tmem;
  int last;
  float2 scale[kStages][kKeys / 16];  // (K, V) scales of a stage's pages
  alignas(16) float2 map[4][N];       // x = S a + c for a softmax warp's first page: (a, c) a column
  float unscale[N], base[N], delta[N], factor[N];
  float part[4][N];  // a warp's column maxima, at the end its column sums
  int lim[N];
  int out[N];        // (token, head) row of the output
};
template <int N>
constexpr bool two_ctas() { return Cfg<N>::kBytes + static_cast<int>(sizeof(Bars<N>)) + 1024 <= 228 * 1024 / 2; }
static_assert(two_ctas<16>() && two_ctas<32>() && two_ctas<48>(), "two CTAs per SM, with the system's 1 KB each");

}  // namespace

template <int kRegs, bool kGrow>
__device__ __forceinline__ void set_registers() {
  if constexpr (kGrow) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <int N>
__global__ void __launch_bounds__(kThreads, 2)
    paged_attn_tc_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v) {
  using C = Cfg<N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem + C::kOffQ;
  uint8_t* sv16 = smem + C::kOffV16;
  __shared__ Bars<N> b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&b.k_full[i], 32);
      mbar_init(&b.k_empty[i], 1);
      mbar_init(&b.v_full[i], 32);
      mbar_init(&b.v_empty[i], 8);
    }
    mbar_init(&b.q_ready, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b.s_full[i], 1);
      mbar_init(&b.s_free[i], 4);
      mbar_init(&b.w_full[i], 4);
      mbar_init(&b.pv_done[i], 1);
    }
    mbar_init(&b.p_full, 4);
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
  const int G = a.hq / a.hkv;
  const int n_tiles = (it.key1 - it.key0 + kKeys - 1) / kKeys;

  if (warp >= 4) {
    // queries, by the softmax and widening warps: a warp a row, four head columns a lane, all loads in flight
    constexpr int kQr = N / 8;
    const int w8 = warp - 4;
    uint2 raw[kQr];
#pragma unroll
    for (int i = 0; i < kQr; ++i) {
      const int n = w8 + 8 * i, row = it.row0 + n;
      raw[i] = make_uint2(0u, 0u);
      if (n < it.rows)
        raw[i] = *reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.q) + static_cast<size_t>(it.tok0 + row / G) * a.ldq +
                                                 static_cast<size_t>(it.head * G + row % G) * kHd + 4 * lane);
    }
#pragma unroll
    for (int i = 0; i < kQr; ++i) {
      const int n = w8 + 8 * i;
      const uint2 u = raw[i];
      const float x[4] = {__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                          __uint_as_float(u.y & 0xFFFF0000u)};
      float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
      m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
      // exponent of m, kept where both the scale and its inverse are normal floats
      const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -110), 110);
      const float up = m > 0.f ? __uint_as_float(static_cast<uint32_t>(127 + 7 - e) << 23) : 1.f;
      uint32_t hi = 0, lo = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x0 = x[2 * h] * up, x1 = x[2 * h + 1] * up;
        const uint16_t c = e4m3x2_from_f32(x0, x1);
        const float2 r = f32x2_from_e4m3x2(c);
        hi |= static_cast<uint32_t>(c) << (16 * h);
        lo |= static_cast<uint32_t>(e4m3x2_from_f32(x0 - r.x, x1 - r.y)) << (16 * h);
      }
      const int at = n * kHd + (((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4;  // 128-byte swizzle
      *reinterpret_cast<uint32_t*>(sq + at) = hi;
      *reinterpret_cast<uint32_t*>(sq + C::kQ + at) = lo;
      if (lane == 0) {
        const int row = it.row0 + n;
        b.unscale[n] = a.scale * kLog2e / up;
        b.base[n] = 0.f;
        b.lim[n] = n < it.rows ? min(it.key1, paged_key_limit(it.len, it.start + row / G, a.causal_block)) : it.key1;
        b.out[n] = (it.tok0 + row / G) * a.hq + it.head * G + row % G;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&b.q_ready);
    named_sync(3, 256);
  }

  if (warp < 4) set_registers<kRegsMisc, false>();
  if (warp == 0) {
    // ---------------- TMA producer: a lane a page ----------------
    const int ps = a.page_size, per_tile = kKeys >> a.page_shift, box = min(ps, 64);
    const int* table = a.table + static_cast<size_t>(it.req) * a.table_ld;
    const uint64_t policy = l2_policy_evict_first();
    int batch = -32, row = 0;  // first page of the 32 whose rows and scales the lanes hold
    float2 sc = make_float2(1.f, 1.f);
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
          sc = make_float2(__ldg(a.k_scale + unit), __ldg(a.v_scale + unit));
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
      if (live) load(&tm_k, &b.k_full[st], smem + C::kOffK + st * kTile);
      mbar_arrive(&b.k_full[st]);
      if (!__all_sync(0xffffffffu, mbar_wait(&b.v_empty[st], free_parity))) {
        report_wait(a.err, kErrTimeoutProducer, 47, a.total_rows, it.splits);
        (void)mbar_wait(&b.k_full[st], (j / kStages) & 1u);  // its K copies land first
        break;
      }
      if (live) load(&tm_v, &b.v_full[st], smem + C::kOffV + st * kTile);
      const float2 s2 = make_float2(__shfl_sync(0xffffffffu, sc.x, from), __shfl_sync(0xffffffffu, sc.y, from));
      if (live) b.scale[st][lane] = s2;
      mbar_arrive(&b.v_full[st]);
      __syncwarp();
    }
    for (int j = max(0, issued - kStages); j < issued; ++j)  // every copy landed before leaving
      if (!mbar_wait(&b.k_full[j % kStages], (j / kStages) & 1u) || !mbar_wait(&b.v_full[j % kStages], (j / kStages) & 1u))
        break;
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t id_s = idesc_s(N), id_o = idesc_o(N);
      int site = 0;
      if (!mbar_wait(&b.q_ready, 0)) site = 42;
      for (int j = 0; j <= n_tiles && site == 0; ++j) {
        if (j < n_tiles) {  // S_j^T = K_j (Qh + Ql)^T
          const int st = j % kStages, sb = j & 1;
          if (!mbar_wait(&b.k_full[st], (j / kStages) & 1u)) {
            site = 43;
            break;
          }
          if (!mbar_wait(&b.s_free[sb], ((j >> 1) & 1u) ^ 1u)) {
            site = 44;
            break;
          }
          tc_fence_after_sync();
          const uint64_t ad = umma_desc_sw128(smem + C::kOffK + st * kTile);
          const uint64_t qh = umma_desc_sw128(sq), ql = umma_desc_sw128(sq + C::kQ);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma_f8(tmem + C::kS + sb * N, ad + 2 * k, qh + 2 * k, id_s, k > 0 ? 1u : 0u);
            mma_f8(tmem + C::kS + sb * N, ad + 2 * k, ql + 2 * k, id_s, 1u);
          }
          tc_commit(&b.s_full[sb]);
          if (C::kOwnP) tc_commit(&b.k_empty[st]);
        }
        if (j >= 1) {  // O^T += V_i^T P_i^T, i = j - 1
          const int i = j - 1;
          if (!mbar_wait(&b.p_full, i & 1u)) {
            site = 45;
            break;
          }
          const uint8_t* p = C::kOwnP ? smem + C::kOffP + (i & 1) * C::kP : smem + C::kOffK + (i % kStages) * kTile;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!mbar_wait(&b.w_full[h], i & 1u)) {
              site = 48;
              break;
            }
            tc_fence_after_sync();
#pragma unroll
            for (int k = 4 * h; k < 4 * h + 4; ++k)  // 16 keys a step: two 8-row groups of V and of P
              tc_mma_bf16(tmem + C::kO, umma_desc_sw128_mn(sv16 + k * 2048, kTile, 1024),
                          umma_desc_mn(p + k * 256, kKeys * 16, 128), id_o, (i > 0 || k > 0) ? 1u : 0u);
            tc_commit(&b.pv_done[h]);
          }
          if (site != 0) break;
          if (!C::kOwnP) tc_commit(&b.k_empty[i % kStages]);
          if (i == n_tiles - 1) tc_commit(&b.o_final);
        }
      }
      if (site != 0) report_wait(a.err, kErrTimeoutMma, site, a.total_rows, it.splits);
    }
  } else if (warp >= 8) {
    set_registers<kRegsWiden, false>();
    // ---------------- V in f16: a key a lane, half a row a thread, 64 keys at a time ----------------
    const int half = warp & 1;
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int st = j % kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&b.v_full[st], (j / kStages) & 1u));
      if (!ok) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 64 * h + 32 * ((warp - 8) >> 1) + lane;  // key of the tile
        const uint8_t* src = smem + C::kOffV + st * kTile + k * kHd;
        // rows past the range hold anything: their weight is 0, their values must be
        const bool dead = it.key0 + j * kKeys + k >= it.key1;
        uint4 u[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u[c] = *reinterpret_cast<const uint4*>(src + (((4 * half + c) ^ (k & 7)) << 4));
          if (dead) u[c] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (h == 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&b.v_empty[st]);
        }
        if (j > 0) {  // the previous tile's product of this half has left the buffer
          ok = __all_sync(0xffffffffu, mbar_wait(&b.pv_done[h], (j - 1) & 1u));
          if (!ok) break;
        }
        uint8_t* dst = sv16 + half * kTile + k * 128;
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
        if (lane == 0) mbar_arrive(&b.w_full[h]);
      }
    }
    if (!ok && lane == 0) report_wait(a.err, kErrTimeoutEpilogue, 49, a.total_rows, it.splits);
  } else if (warp >= 4) {
    set_registers<kRegsSoftmax, true>();
    // ---------------- softmax: a key a thread ----------------
    const int q4 = warp & 3, tid = q4 * 32 + lane;  // TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>(q4 * 32) << 16;
    // keys from which some row's mask ends (rows are in token order, so the first has the least)
    const int lim_min = b.lim[0];
    const int nc = (it.rows + 15) >> 4;  // 16-column chunks with rows
    float sum[N];
#pragma unroll
    for (int n = 0; n < N; ++n) sum[n] = 0.f;
    bool ok = true;

    for (int j = 0; j < n_tiles; ++j) {
      const int sb = j & 1, st = j % kStages;
      const int key = it.key0 + j * kKeys + tid;
      ok = ok && mbar_wait(&b.v_full[st], (j / kStages) & 1u);
      // x = S (unscale ks) + (log2 vs - base): the pair of every column, once a warp.  Its 32 keys are in one
      // page, or at page size 16 in two: then the second half's scores and offsets move by the scales' ratios.
      float inv_vs, ratio = 1.f, shift = 0.f;
      {
        __syncwarp();
        const float2 sc = b.scale[st][tid >> a.page_shift];
        const bool dead = key >= it.key1;  // (its page may not exist)
        const float lv = dead ? 0.f : __log2f(sc.y), ks = dead ? 0.f : sc.x;
        inv_vs = exp2_approx(-lv);
        const float ks0 = __shfl_sync(0xffffffffu, ks, 0), lv0 = __shfl_sync(0xffffffffu, lv, 0);
        for (int n = lane; n < nc * 16; n += 32) b.map[q4][n] = make_float2(b.unscale[n] * ks0, lv0 - b.base[n]);
        if (a.page_shift == 4 && !dead) ratio = ks / ks0, shift = lv - lv0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.v_empty[st]);  // (the scales')
      }
      ok = ok && mbar_wait(&b.s_full[sb], (j >> 1) & 1u);
      __syncwarp();
      tc_fence_after_sync();
      float s[N];
#pragma unroll
      for (int c = 0; c < N / 16; ++c) {
        if (c < nc) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(tmem + lane_base + C::kS + sb * N + c * 16, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) s[c * 16 + i] = __uint_as_float(v[i]);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.s_free[sb]);
      float top0 = -INFINITY, top1 = -INFINITY;
      const float4* map = reinterpret_cast<const float4*>(b.map[q4]);
      const bool edge = it.key0 + (j + 1) * kKeys > lim_min;
#pragma unroll
      for (int c = 0; c < N / 16; ++c) {
        if (c < nc) {
          float4 m[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) m[i] = map[c * 8 + i];
          if (a.page_shift == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[c * 16 + i] *= ratio;
#pragma unroll
            for (int i = 0; i < 8; ++i) m[i].y += shift, m[i].w += shift;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            s[c * 16 + 2 * i] = fmaf(s[c * 16 + 2 * i], m[i].x, m[i].y);
            s[c * 16 + 2 * i + 1] = fmaf(s[c * 16 + 2 * i + 1], m[i].z, m[i].w);
          }
          if (edge) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (key >= b.lim[c * 16 + i]) s[c * 16 + i] = -INFINITY;  // (also what a dead key's garbage gave)
          }
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            top0 = fmaxf(top0, s[c * 16 + i]);
            top1 = fmaxf(top1, s[c * 16 + i + 1]);
          }
        }
      }
      if (any_of_128(fmaxf(top0, top1) > kTrip || j == 0 || !ok)) {
        if (any_of_128(!ok)) {  // a wait expired: all four warps leave together
          ok = false;
          break;
        }
        // move the bases of the columns that need it to their maximum over these 128 keys
#pragma unroll
        for (int c = 0; c < N / 16; ++c)
          if (c < nc) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t m = __reduce_max_sync(0xffffffffu, ordered(s[c * 16 + i]));
              if (lane == 0) b.part[q4][c * 16 + i] = unordered(m);
            }
          }
        named_sync(2, 128);
        if (tid < N) {
          const float m = fmaxf(fmaxf(b.part[0][tid], b.part[1][tid]), fmaxf(b.part[2][tid], b.part[3][tid]));
          const bool move = tid < nc * 16 && m > -INFINITY && m < INFINITY && (j == 0 || m > kTrip);
          const float d = move ? kSeat - m : 0.f;  // new weights are 2^d times the old
          b.delta[tid] = d;
          b.factor[tid] = exp2f(d);
          b.base[tid] -= d;
        }
        named_sync(2, 128);
        if (j > 0) {  // O of the earlier tiles: their last product has to land first
          ok = mbar_wait(&b.pv_done[1], (j - 1) & 1u);
          __syncwarp();
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < nc; ++c) {
            uint32_t v[16];
            tmem_ld_32x32b_x16(tmem + lane_base + C::kO + c * 16, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * b.factor[c * 16 + i]);
            tmem_st_32x32b_x16(tmem + lane_base + C::kO + c * 16, v);
          }
          tmem_st_wait();
          tc_fence_before_sync();
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n < nc * 16) {
            s[n] += b.delta[n];
            if (j > 0) sum[n] *= b.factor[n];
          }
        }
      }
      // P_j over K_j (S_j is done with it), or into the buffer that P_{j-2} has left (S_j's commit covered
      // every product issued before it)
      uint8_t* p = (C::kOwnP ? smem + C::kOffP + sb * C::kP : smem + C::kOffK + st * kTile) + tid * 16;
#pragma unroll
      for (int c = 0; c < N / 8; ++c) {
        if (c >= 2 * nc) continue;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = c * 8 + 2 * i;
          const float p0 = exp2_approx(s[n]), p1 = exp2_approx(s[n + 1]);
          sum[n] = fmaf(p0, inv_vs, sum[n]);
          sum[n + 1] = fmaf(p1, inv_vs, sum[n + 1]);
          w[i] = pack_f16x2(p0, p1);
        }
        *reinterpret_cast<uint4*>(p + c * (kKeys * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.p_full);
    }

    // row sums over the 128 keys: lane l of a warp ends with column l & 15 of each 16-column chunk
#pragma unroll
    for (int c = 0; c < N / 16; ++c) {
      if (c >= nc) continue;
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = sum[c * 16 + i];
#pragma unroll
      for (int h = 8; h >= 1; h >>= 1) {
        const bool up = (lane & h) != 0;
#pragma unroll
        for (int i = 0; i < h; ++i) {
          const float keep = up ? v[i + h] : v[i], give = up ? v[i] : v[i + h];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, h);
        }
      }
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
      if (lane < 16) b.part[q4][c * 16 + lane] = v[0];
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&b.o_final, 0));
    if (!ok && lane == 0) report_wait(a.err, kErrTimeoutEpilogue, 46, a.total_rows, it.splits);
    named_sync(2, 128);
    if (tid < N) {
      const float l = b.part[0][tid] + b.part[1][tid] + b.part[2][tid] + b.part[3][tid];
      b.factor[tid] = it.splits == 1 ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
      b.delta[tid] = l;
    }
    named_sync(2, 128);
    tc_fence_after_sync();
    // O^T: lane = head column, a row a TMEM column.  A split tile leaves its partial: [N][128], then [N] (base, sum)
    bf16* out = static_cast<bf16*>(a.out) + tid;
    float* part = reinterpret_cast<float*>(a.part + it.part) + tid;
#pragma unroll 1
    for (int c = 0; c < nc; ++c) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + lane_base + C::kO + c * 16, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int n = c * 16 + i;
        if (n >= it.rows) continue;
        const float x = __uint_as_float(v[i]) * b.factor[n];
        if (it.splits == 1) out[static_cast<size_t>(b.out[n]) * kHd] = __float2bfloat16_rn(x);
        else part[n * kHd] = x;
      }
    }
    if (it.splits > 1) {
      if (tid < it.rows)
        reinterpret_cast<float2*>(reinterpret_cast<float*>(a.part + it.part) + N * kHd)[tid] = make_float2(b.base[tid], b.delta[tid]);
      __threadfence();
    }
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
    tmem_dealloc(tmem, C::kCols);
  }
  if (it.splits == 1) return;

  // the tile's last item adds the partials, all threads: a row's weights 2^(base - max) / sum, then its columns
  if (threadIdx.x == 0) b.last = atomicAdd(&a.arrived[it.tile], 1u) == static_cast<unsigned>(it.splits - 1);
  __syncthreads();
  if (!b.last) return;
  __threadfence();
  constexpr int kPart = N * kHd + 4 * N;  // floats
  const float* first = reinterpret_cast<const float*>(a.part + it.part) - static_cast<size_t>(it.split) * kPart;
  float* weight = reinterpret_cast<float*>(smem);  // [kMaxPagedSplits][N], over the K ring
  for (int n = warp; n < it.rows; n += kThreads / 32) {  // a lane a split
    float2 bs = make_float2(0.f, 0.f);
    if (lane < it.splits) bs = __ldcg(reinterpret_cast<const float2*>(first + lane * kPart + N * kHd) + n);
    float m = bs.y != 0.f ? bs.x : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float f = bs.y != 0.f ? exp2f(bs.x - m) : 0.f;
    float l = f * bs.y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    weight[lane * N + n] = l != 0.f ? f / l : 0.f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < it.rows * (kHd / 4); i += kThreads) {
    const int n = i >> 5, c4 = i & 31;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < it.splits; ++s) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(first + s * kPart + n * kHd) + c4);
      const float f = weight[s * N + n];
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
    }
    *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + static_cast<size_t>(b.out[n]) * kHd + 4 * c4) =
        make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
  }
  if (threadIdx.x == 0) a.arrived[it.tile] = 0;  // ready for the next call
}

template <int N>
static int launch_n(const PagedAttnArgs& a, int n_items, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  return launch_k(paged_attn_tc_kernel<N>, dim3(n_items), dim3(kThreads), Cfg<N>::kBytes, s, a, k, v);
}
// The register split only ever asks for what the launch brought: checked here, not by waiting for more.
template <int N>
static cudaError_t opt_in() {
  cudaFuncAttributes f;
  cudaError_t e = cudaFuncGetAttributes(&f, paged_attn_tc_kernel<N>);
  if (e == cudaSuccess && f.numRegs < kRegsLaunch) e = cudaErrorInvalidKernelImage;
  return e != cudaSuccess ? e
                          : cudaFuncSetAttribute(paged_attn_tc_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 Cfg<N>::kBytes);
}

int init_paged_attention_tc_attributes() {
  for (cudaError_t e : {opt_in<16>(), opt_in<32>(), opt_in<48>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

int launch_paged_attention_tc(const PagedAttnArgs& a, int cols, int n_items, const CUtensorMap& k, const CUtensorMap& v,
                              cudaStream_t s) {
  switch (cols) {
    case 16: return launch_n<16>(a, n_items, k, v, s);
    case 32: return launch_n<32>(a, n_items, k, v, s);
    default: return launch_n<48>(a, n_items, k, v, s);
  }
}

}  // namespace fdllm
