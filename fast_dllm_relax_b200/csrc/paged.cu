// Host side of the paged 8-bit KV cache and of the log-probability reduction: batch plans, argument
// checks and the C ABI entries of include/fdllm_sm100.h.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <mutex>
#include <string>
#include <vector>

#include "handle.h"
#include "paged.h"

using namespace fdllm;

namespace {

// No C++ exception crosses the ABI: `body` returns a status, an exception becomes one.
template <typename F>
int guarded(F body) {
  try {
    return body();
  } catch (const std::exception& e) {
    return fail(FDLLM_ERR_INVALID, std::string("internal error: ") + e.what());
  } catch (...) {
    return fail(FDLLM_ERR_INVALID, "internal error");
  }
}

bool page_size_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// At least n arrival counters: zero when allocated (in the order of the call's stream), and again after
// every launch that uses them.
int ensure_counters(CallBuf<unsigned>* b, size_t n, cudaStream_t s) {
  if (b->n >= n) return FDLLM_OK;
  FDLLM_TRY(b->ensure(n));
  CUDA_TRY(cudaMemsetAsync(b->p, 0, b->bytes(), s));
  return FDLLM_OK;
}

// Rows of `cols` elements with a row stride of ld elements, every row 16-byte aligned.
int check_rows(const fdllm_handle* h, const char* name, const void* p, int ld, int cols) {
  if (p == nullptr) return fail(FDLLM_ERR_INVALID, std::string(name) + ": null pointer");
  if (ld < cols) return fail(FDLLM_ERR_INVALID, std::string(name) + ": row stride below " + std::to_string(cols));
  if (!aligned16(p) || (static_cast<size_t>(ld) * h->esz) % 16 != 0)
    return fail(FDLLM_ERR_INVALID, std::string(name) + ": rows must be 16-byte aligned");
  return FDLLM_OK;
}

// The checks that append and attention share; *layer_codes / *layer_scales: this layer's offsets.
int check_paged(const fdllm_handle* h, const fdllm_paged_cache* c, int layer, const fdllm_paged_plan* p,
                const int32_t* words, const int32_t* table, int table_ld, size_t* layer_codes, size_t* layer_scales) {
  if (c == nullptr || p == nullptr) return fail(FDLLM_ERR_INVALID, "null cache or plan");
  if (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr)
    return fail(FDLLM_ERR_INVALID, "null paged cache");
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(FDLLM_ERR_INVALID, "paged cache must be 16-byte aligned");
  if (c->layers <= 0 || c->pages <= 0 || !page_size_ok(c->page_size))
    return fail(FDLLM_ERR_INVALID, "paged cache needs layers, pages and a page size of 16, 32, 64 or 128");
  if (layer < 0 || layer >= c->layers)
    return fail(FDLLM_ERR_INVALID, "layer " + std::to_string(layer) + " outside [0, " + std::to_string(c->layers) + ")");
  if (p->page_size != c->page_size)
    return fail(FDLLM_ERR_INVALID, "the plan is for pages of " + std::to_string(p->page_size) + " rows, the cache has " +
                                       std::to_string(c->page_size));
  if (p->total_rows > 0 && (words == nullptr || table == nullptr)) return fail(FDLLM_ERR_INVALID, "null plan words or table");
  if (!aligned16(words)) return fail(FDLLM_ERR_INVALID, "plan words must be 16-byte aligned");
  if (table_ld < p->table_cols)
    return fail(FDLLM_ERR_INVALID, "page table has " + std::to_string(table_ld) + " columns; the longest request needs " +
                                       std::to_string(p->table_cols));
  const fdllm_config& cfg = h->cfg;
  if (const int32_t* s = p->priv + kPagedShape; s[0] != cfg.num_attention_heads || s[1] != cfg.num_key_value_heads ||
                                                s[2] != cfg.head_dim || s[3] != h->dtype)
    return fail(FDLLM_ERR_INVALID, "the plan was laid out for " + std::to_string(s[0]) + "/" + std::to_string(s[1]) +
                                       " heads of " + std::to_string(s[2]) + " in another handle");
  const size_t heads = static_cast<size_t>(c->pages) * h->cfg.num_key_value_heads;
  *layer_scales = static_cast<size_t>(layer) * heads;
  *layer_codes = static_cast<size_t>(layer) * heads * c->page_size * h->cfg.head_dim;
  return FDLLM_OK;
}

// A share costs its prologue and its part of the join, more with more rows: 256 keys at least for up to 16 rows
// (one token over 4000 keys: 8.9 us, 10.7 with 512), 512 above (8 requests of 8 rows over 4096 keys, 12/2 heads: 19.8
// us, 21.9 with 256 and 23.8 with 1024).
constexpr int kMinShareFew = 256, kMinShareMany = 512;
constexpr int kShareUnit = 128;

// The attention items of a bf16 batch.
struct ItemPlan {
  std::vector<PagedItem> items[kPagedClasses];
  int tiles = 0;
  long long parts = 0;
};

// Rows of a request and KV head are cut into equal tiles of a class's size.  Keys are cut into shares only
// as far as that fills the SMs (`slots` CTAs are resident at once): a share costs its prologue, its partial
// and a part of the join, so shares grow until the items fit one wave.
int plan_items(const fdllm_handle* h, const std::vector<PagedReq>& reqs, int causal_block, ItemPlan* out) {
  const fdllm_config& c = h->cfg;
  const int G = c.num_attention_heads / c.num_key_value_heads, heads = c.num_key_value_heads;
  const bool tc = c.head_dim == 128;
  const int unit = tc ? 16 : 8, narrow = tc ? 48 : 24;  // largest tile of the classes by rows
  auto is_wide = [&](long long rows) { return tc && rows > narrow; };
  const long long slots = static_cast<long long>(tc ? 2 : kPagedNarrowCtas) * h->num_sms;
  auto tile_rows = [&](long long rows) {
    const int largest = is_wide(rows) ? 128 : narrow;
    const long long tiles = (rows + largest - 1) / largest;
    return static_cast<int>(((rows + tiles - 1) / tiles + unit - 1) / unit * unit);
  };
  auto keys_of = [&](const PagedReq& r, long long row_end) {  // keys of a tile whose last row is row_end - 1
    const long long pos = r.start + (row_end - 1) / G;
    return causal_block > 0 ? static_cast<int>(std::min<long long>(r.len, (pos / causal_block + 1) * causal_block)) : r.len;
  };
  struct Tile { int keys, min_share; };
  auto splits_of = [&](const Tile& t, long long share) {
    const long long each = std::max<long long>(share, t.min_share);
    return static_cast<int>(std::min<long long>(kMaxPagedSplits, (t.keys + each - 1) / each));
  };
  auto min_share = [](int rows) { return rows <= 16 ? kMinShareFew : kMinShareMany; };
  std::vector<Tile> tiles;  // of one head
  long long work = 0, longest = 0;
  for (const PagedReq& r : reqs) {
    const long long rows = static_cast<long long>(r.rows) * G;
    const int step = rows > 0 ? tile_rows(rows) : 1;
    for (long long t = 0; t < rows; t += step) {
      tiles.push_back(Tile{keys_of(r, std::min(rows, t + step)), min_share(step)});
      work += tiles.back().keys;
      longest = std::max<long long>(longest, tiles.back().keys);
    }
  }
  // the least share, in units, whose items fit one wave; the longest tile's where none does
  long long low = work * heads / slots / kShareUnit, high = (longest + kShareUnit - 1) / kShareUnit;
  while (low + 1 < high) {
    const long long mid = (low + high) / 2;
    long long items = 0;
    for (const Tile& t : tiles) items += splits_of(t, mid * kShareUnit);
    (items * heads <= slots ? high : low) = mid;
  }
  const long long share = high * kShareUnit;
  for (size_t i = 0; i < reqs.size(); ++i) {
    const PagedReq& r = reqs[i];
    const long long rows = static_cast<long long>(r.rows) * G;
    if (rows == 0) continue;
    const int step = tile_rows(rows), cls = is_wide(rows) ? kPagedWide : step / unit - 1;
    const int part_rows = is_wide(rows) ? 128 : step;
    for (long long t = 0; t < rows; t += step) {
      const int keys = keys_of(r, std::min(rows, t + step));
      const int want = splits_of(Tile{keys, min_share(step)}, share);
      const int each = ((keys + want - 1) / want + kShareUnit - 1) / kShareUnit * kShareUnit;
      const int splits = (keys + each - 1) / each;
      const int part = part_rows * (c.head_dim / 4) + part_rows;  // 16-byte units
      for (int head = 0; head < heads; ++head) {
        for (int s = 0; s < splits; ++s) {
          PagedItem it{};
          it.req = static_cast<int>(i);
          it.head = head;
          it.row0 = static_cast<int>(t);
          it.rows = static_cast<int>(std::min<long long>(step, rows - t));
          it.tok0 = r.tok0;
          it.start = r.start;
          it.len = r.len;
          it.key0 = s * each;
          it.key1 = std::min(keys, (s + 1) * each);
          it.split = s;
          it.splits = splits;
          it.tile = out->tiles;
          it.part = splits > 1 ? static_cast<int>(out->parts + static_cast<long long>(s) * part) : 0;
          out->items[cls].push_back(it);
        }
        if (splits > 1) {
          out->parts += static_cast<long long>(splits) * part;
          ++out->tiles;
        }
        if (out->parts > 0x7FFFFFFFLL) return fail(FDLLM_ERR_INVALID, "batch too large for one plan");
      }
    }
  }
  // longest items first: the last CTAs to start are the short ones
  for (auto& v : out->items)
    std::stable_sort(v.begin(), v.end(), [](const PagedItem& a, const PagedItem& b) { return a.key1 - a.key0 > b.key1 - b.key0; });
  return FDLLM_OK;
}

}  // namespace

int fdllm::paged_append(fdllm_handle* h, const fdllm_paged_cache* cache, int layer, const fdllm_paged_plan* plan,
                        const int32_t* plan_words, const int32_t* table, int table_ld, const void* q, int ldq,
                        const void* k, int ldk, const void* v, int ldv, const float* rope_cos, const float* rope_sin,
                        int rope_rows, void* q_out, cudaStream_t s) {
  size_t codes, scales;
  FDLLM_TRY(check_paged(h, cache, layer, plan, plan_words, table, table_ld, &codes, &scales));
  if ((rope_cos == nullptr) != (rope_sin == nullptr)) return fail(FDLLM_ERR_INVALID, "rope_cos and rope_sin go together");
  const int have = rope_cos != nullptr ? rope_rows : h->cfg.max_positions;
  if (plan->max_position > have)
    return fail(FDLLM_ERR_INVALID, "RoPE positions reach " + std::to_string(plan->max_position) + "; the tables have " +
                                       std::to_string(have) + " rows");
  if (rope_cos != nullptr && (!aligned16(rope_cos) || !aligned16(rope_sin)))
    return fail(FDLLM_ERR_INVALID, "RoPE tables must be 16-byte aligned");
  if (plan->total_rows == 0) return FDLLM_OK;
  const fdllm_config& c = h->cfg;
  if ((q == nullptr) != (q_out == nullptr)) return fail(FDLLM_ERR_INVALID, "q and q_out go together");
  if (q != nullptr) {
    FDLLM_TRY(check_rows(h, "q", q, ldq, c.num_attention_heads * c.head_dim));
    FDLLM_TRY(check_rows(h, "q_out", q_out, c.num_attention_heads * c.head_dim, c.num_attention_heads * c.head_dim));
  }
  FDLLM_TRY(check_rows(h, "k", k, ldk, c.num_key_value_heads * c.head_dim));
  FDLLM_TRY(check_rows(h, "v", v, ldv, c.num_key_value_heads * c.head_dim));
  PagedAppendArgs a{};
  a.reqs = reinterpret_cast<const PagedReq*>(plan_words);
  a.units = reinterpret_cast<const PagedPageUnit*>(plan_words + plan->priv[kPagedPageOff]);
  a.n_units = plan->priv[kPagedPageUnits];
  a.q_units = reinterpret_cast<const PagedPageUnit*>(plan_words + plan->priv[kPagedQOff]);
  a.n_q_units = plan->priv[kPagedQUnits];
  a.n = plan->n;
  a.total_rows = plan->total_rows;
  a.table = table;
  a.table_ld = table_ld;
  a.k = static_cast<uint8_t*>(cache->k) + codes;
  a.v = static_cast<uint8_t*>(cache->v) + codes;
  a.k_scale = cache->k_scale + scales;
  a.v_scale = cache->v_scale + scales;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.hq = c.num_attention_heads;
  a.hkv = c.num_key_value_heads;
  a.hd = c.head_dim;
  a.q_in = q;
  a.k_in = k;
  a.v_in = v;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.table_f32 = rope_cos != nullptr || h->dtype == FDLLM_FLOAT32;
  a.cos = rope_cos != nullptr ? static_cast<const void*>(rope_cos) : h->rope_cos.p;
  a.sin = rope_sin != nullptr ? static_cast<const void*>(rope_sin) : h->rope_sin.p;
  a.q_out = q_out;
  a.err = h->err.p;
  CUDA_TRY(launch_paged_append(a, h->dtype, s));
  return FDLLM_OK;
}

int fdllm::paged_attention(fdllm_handle* h, const fdllm_paged_cache* cache, int layer, const fdllm_paged_plan* plan,
                           const int32_t* plan_words, const int32_t* table, int table_ld, const void* q, int ldq,
                           float scale, void* out, cudaStream_t s) {
  size_t codes, scales;
  FDLLM_TRY(check_paged(h, cache, layer, plan, plan_words, table, table_ld, &codes, &scales));
  if (!std::isfinite(scale)) return fail(FDLLM_ERR_INVALID, "scale must be finite");
  if (plan->total_rows == 0) return FDLLM_OK;
  const fdllm_config& c = h->cfg;
  const int cols = c.num_attention_heads * c.head_dim;
  FDLLM_TRY(check_rows(h, "q", q, ldq, cols));
  FDLLM_TRY(check_rows(h, "out", out, cols, cols));
  PagedAttnArgs a{};
  a.reqs = reinterpret_cast<const PagedReq*>(plan_words);
  a.n = plan->n;
  a.total_rows = plan->total_rows;
  a.table = table;
  a.table_ld = table_ld;
  a.k = static_cast<const uint8_t*>(cache->k) + codes;
  a.v = static_cast<const uint8_t*>(cache->v) + codes;
  a.k_scale = cache->k_scale + scales;
  a.v_scale = cache->v_scale + scales;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  while ((1 << a.page_shift) < a.page_size) ++a.page_shift;
  a.hq = c.num_attention_heads;
  a.hkv = c.num_key_value_heads;
  a.hd = c.head_dim;
  a.causal_block = plan->causal_block;
  a.q = q;
  a.ldq = ldq;
  a.scale = scale;
  a.out = out;
  a.err = h->err.p;
  if (h->dtype != FDLLM_BFLOAT16) {
    CUDA_TRY(launch_paged_attention_simt(a, s));
    return FDLLM_OK;
  }
  FDLLM_TRY(h->paged_part.ensure(plan->priv[kPagedParts]));
  FDLLM_TRY(ensure_counters(&h->paged_ctr, plan->priv[kPagedTiles], s));
  CUtensorMap tm_k, tm_v;
  FDLLM_TRY(make_page_map(&tm_k, cache->k, cache, c.num_key_value_heads, c.head_dim));
  FDLLM_TRY(make_page_map(&tm_v, cache->v, cache, c.num_key_value_heads, c.head_dim));
  a.layer_row = static_cast<int>(codes / c.head_dim);
  a.part = h->paged_part.p;
  a.arrived = h->paged_ctr.p;
  a.items = reinterpret_cast<const PagedItem*>(plan_words + plan->priv[kPagedItemOff]);
  for (int k = kPagedClasses - 1, end = 0; k >= 0; --k) a.class_end[k] = end += plan->priv[kPagedItems + k];
  CUDA_TRY(c.head_dim == 128 ? launch_paged_attention_mma(a, tm_k, tm_v, s)
                             : launch_paged_attention_narrow(a, tm_k, tm_v, s));
  return FDLLM_OK;
}

extern "C" {

int fdllm_paged_plan_batch(fdllm_handle* h, const int32_t* rows, const int32_t* start, const int32_t* live, int n,
                           int page_size, int causal_block, int32_t* words, int cap, fdllm_paged_plan* plan) {
  return guarded([&]() -> int {
    if (h == nullptr) return fail(FDLLM_ERR_INVALID, "null handle");
    if (plan == nullptr || n < 0 || (n > 0 && (rows == nullptr || start == nullptr)) || cap < 0 ||
        (cap > 0 && words == nullptr))
      return fail(FDLLM_ERR_INVALID, "bad plan arguments");
    if (!page_size_ok(page_size)) return fail(FDLLM_ERR_INVALID, "page size must be 16, 32, 64 or 128");
    if (causal_block < 0) return fail(FDLLM_ERR_INVALID, "causal_block must not be negative");
    std::vector<PagedReq> reqs(n);
    std::vector<PagedPageUnit> units, q_units;
    long long total = 0, max_len = 0, max_pos = 0;
    for (int i = 0; i < n; ++i) {
      const long long r = rows[i], s = start[i], lv = live != nullptr ? live[i] : start[i];
      if (r < 0 || s < 0 || lv < s)
        return fail(FDLLM_ERR_INVALID, "request " + std::to_string(i) + ": rows and start must not be negative, and live (" +
                                           std::to_string(lv) + ") not below start (" + std::to_string(s) + ")");
      const long long len = std::max(lv, s + r);
      if (len > (1LL << 30) || total + r > (1LL << 30)) return fail(FDLLM_ERR_INVALID, "batch too long");
      reqs[i] = PagedReq{static_cast<int>(total), static_cast<int>(r), static_cast<int>(s), static_cast<int>(lv),
                         static_cast<int>(len), {0, 0, 0}};
      total += r;
      max_len = std::max(max_len, len);
      if (r > 0) max_pos = std::max(max_pos, s + r);
      for (long long p = s / page_size; r > 0 && p <= (s + r - 1) / page_size; ++p)
        units.push_back(PagedPageUnit{i, static_cast<int>(p)});
      for (long long t = 0; t < r; t += kPagedQTokens) q_units.push_back(PagedPageUnit{i, static_cast<int>(t)});
    }
    fdllm_paged_plan out{};
    out.n = n;
    out.total_rows = static_cast<int>(total);
    out.page_size = page_size;
    out.causal_block = causal_block;
    out.table_cols = static_cast<int>((max_len + page_size - 1) / page_size);
    out.max_position = static_cast<int>(max_pos);
    const int32_t shape[4] = {h->cfg.num_attention_heads, h->cfg.num_key_value_heads, h->cfg.head_dim, h->dtype};
    std::copy(shape, shape + 4, out.priv + kPagedShape);
    int at = n * kPagedReqWords;
    out.priv[kPagedPageUnits] = static_cast<int>(units.size());
    out.priv[kPagedPageOff] = at;
    at += 2 * static_cast<int>(units.size());
    out.priv[kPagedQUnits] = static_cast<int>(q_units.size());
    out.priv[kPagedQOff] = at;
    at += 2 * static_cast<int>(q_units.size());
    at = (at + 3) & ~3;  // items are read in 16-byte words
    ItemPlan ip;
    if (h->dtype == FDLLM_BFLOAT16) FDLLM_TRY(plan_items(h, reqs, causal_block, &ip));
    out.priv[kPagedTiles] = ip.tiles;
    out.priv[kPagedParts] = static_cast<int>(ip.parts);
    out.priv[kPagedItemOff] = at;
    for (int c = kPagedClasses - 1; c >= 0; --c) {
      out.priv[kPagedItems + c] = static_cast<int>(ip.items[c].size());
      at += kPagedItemWords * static_cast<int>(ip.items[c].size());
    }
    out.words = at;
    *plan = out;
    if (cap < at) {
      if (cap == 0 && words == nullptr) return FDLLM_OK;  // size query
      return fail(FDLLM_ERR_INVALID, "plan needs " + std::to_string(at) + " words, given " + std::to_string(cap));
    }
    std::memset(words, 0, sizeof(int32_t) * at);
    if (n > 0) std::memcpy(words, reqs.data(), reqs.size() * sizeof(PagedReq));
    if (!units.empty())
      std::memcpy(words + out.priv[kPagedPageOff], units.data(), units.size() * sizeof(PagedPageUnit));
    if (!q_units.empty())
      std::memcpy(words + out.priv[kPagedQOff], q_units.data(), q_units.size() * sizeof(PagedPageUnit));
    int32_t* to = words + out.priv[kPagedItemOff];
    for (int c = kPagedClasses - 1; c >= 0; --c) {
      if (!ip.items[c].empty()) std::memcpy(to, ip.items[c].data(), ip.items[c].size() * sizeof(PagedItem));
      to += kPagedItemWords * ip.items[c].size();
    }
    return FDLLM_OK;
  });
}

int fdllm_paged_append(fdllm_handle* h, const fdllm_paged_cache* cache, int layer, const fdllm_paged_plan* plan,
                       const int32_t* plan_words, const int32_t* table, int table_ld, const void* q, int ldq,
                       const void* k, int ldk, const void* v, int ldv, const float* rope_cos, const float* rope_sin,
                       int rope_rows, void* q_out, void* stream) {
  return guarded([&]() -> int {
    FDLLM_TRY(check_handle(h));
    std::lock_guard<std::mutex> lock(h->mu);
    return paged_append(h, cache, layer, plan, plan_words, table, table_ld, q, ldq, k, ldk, v, ldv, rope_cos, rope_sin,
                        rope_rows, q_out, static_cast<cudaStream_t>(stream));
  });
}

int fdllm_paged_attention(fdllm_handle* h, const fdllm_paged_cache* cache, int layer, const fdllm_paged_plan* plan,
                          const int32_t* plan_words, const int32_t* table, int table_ld, const void* q, int ldq,
                          float scale, void* out, void* stream) {
  return guarded([&]() -> int {
    FDLLM_TRY(check_handle(h));
    std::lock_guard<std::mutex> lock(h->mu);
    return paged_attention(h, cache, layer, plan, plan_words, table, table_ld, q, ldq, scale, out,
                           static_cast<cudaStream_t>(stream));
  });
}

int fdllm_forward_paged(fdllm_handle* h, const fdllm_paged_cache* cache, const fdllm_paged_plan* plan,
                        const int32_t* plan_words, const int32_t* table, int table_ld, const void* x, void* out,
                        void* stream) {
  return guarded([&]() -> int {
    FDLLM_TRY(check_handle(h));
    size_t codes, scales;
    FDLLM_TRY(check_paged(h, cache, 0, plan, plan_words, table, table_ld, &codes, &scales));
    if (cache->layers != h->cfg.num_hidden_layers)
      return fail(FDLLM_ERR_INVALID, "the paged cache has " + std::to_string(cache->layers) + " layers, the model " +
                                         std::to_string(h->cfg.num_hidden_layers));
    if (plan->max_position > h->cfg.max_positions)
      return fail(FDLLM_ERR_INVALID, "RoPE positions exceed max_positions");
    if (plan->total_rows == 0) return FDLLM_OK;
    if (x == nullptr) return fail(FDLLM_ERR_INVALID, "null x");
    std::lock_guard<std::mutex> lock(h->mu);
    return forward_paged(h, cache, plan, plan_words, table, table_ld, x, out, static_cast<cudaStream_t>(stream));
  });
}

int fdllm_logprobs(fdllm_handle* h, const void* logits, int logits_dtype, int rows, int vocab, long long ld,
                   const int32_t* targets, int top, float* logprob, float* entropy, int32_t* top_ids,
                   float* top_logprobs, void* stream) {
  return guarded([&]() -> int {
    FDLLM_TRY(check_handle(h));
    if (logits_dtype != FDLLM_FLOAT32 && logits_dtype != FDLLM_BFLOAT16)
      return fail(FDLLM_ERR_UNSUPPORTED, "logits must be fp32 or bf16");
    if (rows < 0 || vocab <= 0) return fail(FDLLM_ERR_INVALID, "bad logits shape");
    if (ld < vocab) return fail(FDLLM_ERR_INVALID, "logits row stride below the vocabulary");
    if (top < 0 || top > kMaxTopLogprobs || top > vocab)
      return fail(FDLLM_ERR_INVALID, "top must be in [0, " + std::to_string(std::min(kMaxTopLogprobs, vocab)) + "]");
    if (rows == 0) return FDLLM_OK;
    if ((targets == nullptr) != (logprob == nullptr)) return fail(FDLLM_ERR_INVALID, "targets and logprob go together");
    if (top > 0 && (top_ids == nullptr || top_logprobs == nullptr)) return fail(FDLLM_ERR_INVALID, "null top outputs");
    if (logits == nullptr) return fail(FDLLM_ERR_INVALID, "null logits");
    LogprobArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.vocab = vocab;
    a.ld = ld;
    a.targets = targets;
    a.top = top;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    int part_chunks = 0;
    const int parts = logprobs_parts(rows, vocab, logits_dtype, h->num_sms, &part_chunks);
    if (static_cast<long long>(rows) * parts > 0x7FFFFFFFLL) return fail(FDLLM_ERR_INVALID, "too many logits");
    std::lock_guard<std::mutex> lock(h->mu);
    if (parts > 1) {
      const size_t n = static_cast<size_t>(rows) * parts;
      FDLLM_TRY(h->logprob_part.ensure(n));
      FDLLM_TRY(h->logprob_keys.ensure(n * std::max(top, 1)));
      FDLLM_TRY(ensure_counters(&h->logprob_ctr, rows, static_cast<cudaStream_t>(stream)));
      a.part = h->logprob_part.p;
      a.keys = h->logprob_keys.p;
      a.arrived = h->logprob_ctr.p;
    }
    a.err = h->err.p;
    CUDA_TRY(launch_logprobs(a, logits_dtype, parts, part_chunks, static_cast<cudaStream_t>(stream)));
    return FDLLM_OK;
  });
}

}  // extern "C"
