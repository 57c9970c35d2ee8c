"""64-bit CPU restatement of the paged 8-bit cache operators (test infrastructure)."""

from __future__ import annotations

import math

import torch

from fast_dllm_relax_b200.config import ModelConfig, make_synthetic_params
from oracle.model import OracleModel

HEADS = [(12, 2, 128), (4, 2, 64), (8, 8, 64), (8, 1, 128), (16, 1, 128), (4, 4, 32)]


def paged_engine(heads, dtype, max_positions=16384):
    from fast_dllm_relax_b200.engine import Engine
    hq, hkv, hd = heads
    cfg = ModelConfig(vocab_size=256, hidden_size=256, intermediate_size=256, num_hidden_layers=1,
                      num_attention_heads=hq, num_key_value_heads=hkv, head_dim=hd, context_window_size=max_positions)
    return Engine(cfg, [p.cuda() for p in make_synthetic_params(cfg, 0, dtype)], dtype=dtype)


def make_table(lens, page, gen, spare=2, width_extra=1):
    """Page tables of shuffled pages: (int32 [n, width] with unused columns -1, pages of the pool)."""
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lens), max(used, default=0) + width_extra), -1, dtype=torch.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u].to(torch.int32)
        at += u
    return table, pages


def values(codes):
    """float8 e4m3 codes as float64 (exact)."""
    return codes.float().double()


def round_e4m3(x):
    """float64 to the nearest e4m3 value (ties to even, saturating; NaN stays)."""
    y = x.clamp(-448.0, 448.0)
    step = torch.exp2((torch.frexp(y)[1].clamp(min=-5) - 4).double())
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def e4m3_half_step(x):
    """Half the spacing of the e4m3 values around |x| (float64)."""
    return torch.exp2((torch.frexp(x.clamp(-448.0, 448.0))[1].clamp(min=-5) - 5).double())


def scale_of(amax):
    """The least power of two >= 2^-64 with amax <= 448 * scale."""
    if amax == 0:
        return 2.0 ** -64
    e = max(math.ceil(math.log2(amax / 448.0)) - 1, -64)
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rope_tables(rows, hd, theta=1e6):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return angle.cos().float(), angle.sin().float()


def rotate(x, cos, sin):
    a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def attend(q, k, v, ks, vs, table, rows, start, live, page, causal, hq, scale):
    """(out, sum of weight * |v|, largest scale * sum |q k| of a row) in float64.  q [tokens, hq, hd],
    k / v codes float64 [pages, hkv, page, hd], ks / vs [pages, hkv]."""
    hkv, hd = k.shape[1], k.shape[3]
    outs, mags, dots, at = [], [], [], 0
    for i, (n, s, lv) in enumerate(zip(rows, start, live)):
        length = max(lv, s + n)
        ids = table[i, :-(-length // page)].long()
        K = (k[ids] * ks[ids][:, :, None, None]).transpose(0, 1).reshape(hkv, -1, hd)[:, :length]
        V = (v[ids] * vs[ids][:, :, None, None]).transpose(0, 1).reshape(hkv, -1, hd)[:, :length]
        for j in range(n):
            lim = min(length, ((s + j) // causal + 1) * causal) if causal else length
            Q = q[at + j].view(hkv, hq // hkv, hd)
            w = torch.softmax(torch.einsum("hgd,hkd->hgk", Q, K[:, :lim]) * scale, -1)
            outs.append(torch.einsum("hgk,hkd->hgd", w, V[:, :lim]).reshape(hq, hd))
            mags.append(torch.einsum("hgk,hkd->hgd", w, V[:, :lim].abs()).reshape(hq, hd))
            dots.append((torch.einsum("hgd,hkd->hgk", Q.abs(), K[:, :lim].abs()) * scale).amax(-1).reshape(hq, 1))
        at += n
    empty = torch.zeros(0, hq, hd, dtype=torch.float64)
    return (torch.stack(outs), torch.stack(mags), torch.stack(dots)) if outs else (empty, empty, empty[..., :1])


class PagedOracle(OracleModel):
    """The oracle over a cache of e4m3 codes with a power-of-two scale per page and head.  The k_cache /
    v_cache tensors hold the cached values (code * scale); scales are kept per cache tensor."""

    page = 32

    def _write(self, cache, layer, start, live, x):
        """Rows [start, start + n) of one layer, live rows held before (as fdllm_paged_append defines it)."""
        scales = self.__dict__.setdefault("_scales", {}).setdefault((cache.data_ptr(), layer), {})
        n, page = x.shape[0], self.page
        for slot in range(start // page, -(-(start + n) // page)):
            lo, hi = max(start - slot * page, 0), min(start + n - slot * page, page)
            new = x[slot * page + lo - start:slot * page + hi - start].double()
            kept = [r for r in range(min(max(live - slot * page, 0), page)) if not lo <= r < hi]
            for h in range(x.shape[1]):
                old = scales.get((slot, h), 0.0)
                scale = max(scale_of(float(new[:, h].abs().max())), old if kept else 0.0)
                rows = cache[layer, 0, slot * page:(slot + 1) * page, h]
                if kept and scale != old:
                    rows[kept] = (round_e4m3(rows[kept].double() / scale) * scale).to(rows.dtype)
                rows[lo:hi] = (round_e4m3(new[:, h] / scale) * scale).to(rows.dtype)
                scales[slot, h] = scale

    def _qkv_exact(self, layer, xn, offset):
        """q in the model dtype; k rotated in fp32 and not rounded before it is coded."""
        cfg, n = self.cfg, xn.shape[0]
        qkv = self.linear(xn, layer["qkv_w"], layer["qkv_b"])
        qd, kd = cfg.num_attention_heads * cfg.head_dim, cfg.num_key_value_heads * cfg.head_dim
        half = cfg.head_dim // 2
        c, s = (t[:, None, :half].float() for t in self.rope_tables(n, offset))
        q, k = (rotate(t.reshape(n, -1, cfg.head_dim).float(), c, s) for t in (qkv[:, :qd], qkv[:, qd:qd + kd]))
        return self._r(q), k, qkv[:, qd + kd:].reshape(n, -1, cfg.head_dim).float()

    def _paged_forward(self, x, k_cache, v_cache, start, live, causal):
        h = x[0].to(self.dtype)
        rows = h.shape[0]
        length = max(live, start + rows)
        bias = None
        if causal:
            limit = (torch.arange(start, start + rows) // causal + 1) * causal
            bias = torch.where(torch.arange(length)[None, :] < limit[:, None], 0.0, -math.inf)
        for i, layer in enumerate(self.layers):
            q, k, v = self._qkv_exact(layer, self.rms_norm(h, layer["ln1"]), start)
            self._write(k_cache, i, start, live, k)
            self._write(v_cache, i, start, live, v)
            attn = self._attend(q, k_cache[i, 0, :length], v_cache[i, 0, :length], bias)
            h = self._r(h.float() + self.linear(attn, layer["o_w"]).float())
            h = self._mlp(layer, h)
        return self.rms_norm(h, self.norm_w)[None]

    def build_prefix_cache(self, x, bias, k_cache, v_cache):
        self._paged_forward(x, k_cache, v_cache, 0, 0, self.cfg.bd_size)

    def forward_cached(self, x, k_cache, v_cache, cache_offset, prefix_len, write_rel=0, attend_rel=None):
        rows = x.shape[1]
        attend = prefix_len + (rows if attend_rel is None else attend_rel)
        partial = write_rel > 0 or rows < attend - prefix_len
        return self._paged_forward(x, k_cache, v_cache, prefix_len + write_rel, attend if partial else prefix_len, 0)
