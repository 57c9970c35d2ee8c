"""The paged 8-bit KV cache (append with RoPE, attention) against a 64-bit CPU restatement."""

import pytest
import torch

from _paged_util import (HEADS, attend, e4m3_half_step, make_table, paged_engine, rope_tables, rotate, round_e4m3,
                         scale_of, values)

pytestmark = pytest.mark.gpu

_ENGINES: dict = {}


def engine(heads, dtype):
    if (heads, dtype) not in _ENGINES:
        _ENGINES[heads, dtype] = paged_engine(heads, dtype)
    return _ENGINES[heads, dtype]


def random_cache(eng, pages, page, gen, layers=1, fill_nan=False):
    """A cache of unit-normal values; with fill_nan every code is NaN and every scale NaN."""
    cache = eng.new_paged_cache(pages, page_size=page, layers=layers)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if fill_nan:
            codes.view(torch.uint8).fill_(0x7F)
            scale.fill_(float("nan"))
            continue
        s = 2.0 ** torch.randint(-9, -5, scale.shape, generator=gen).float()
        x = torch.randn(codes.shape, generator=gen) / s[..., None, None]
        codes.copy_(x.clamp(-448, 448).to(torch.float8_e4m3fn))
        scale.copy_(s)
    return cache


# ---- append --------------------------------------------------------------------------------------

BATCHES = {
    "one": ([1], [0], None),
    "mid-page": ([1, 3], [37, 15], None),
    "empty-request": ([5, 0, 7], [16, 40, 0], None),
    "rewrite-inside": ([8, 8, 1], [64, 40, 3], [96, 128, 70]),
    "pages": ([32, 129, 64], [32, 5, 0], None),
}


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,page", [((12, 2, 128), 32), ((4, 2, 64), 16), ((8, 8, 64), 64), ((8, 1, 128), 128),
                                        ((4, 4, 32), 16)])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_append_matches_the_definition(batch, heads, page, dtype):
    rows, start, live = BATCHES[batch]
    hq, hkv, hd = heads
    eng = engine(heads, dtype)
    gen = torch.Generator().manual_seed(hash((batch, page)) % 1000 + 1)
    lens = [max(lv, s + n) for n, s, lv in zip(rows, start, live or start)]
    table, pages = make_table(lens, page, gen)
    cache = random_cache(eng, pages, page, gen, layers=2)
    before = {n: (getattr(cache, n).cpu().clone(), getattr(cache, n + "_scale").cpu().clone()) for n in "kv"}
    total = sum(rows)
    # magnitudes over many powers of two: pages whose scale grows, and pages whose scale stands
    mag = 2.0 ** torch.randint(-6, 7, (total, 1), generator=gen).float()
    wide = torch.randn(total, (hq + 2 * hkv) * hd + 16, generator=gen) * mag
    qkv = wide.to(eng.dtype).cuda()[:, 8:-8]  # strided rows
    q, k, v = qkv.split([hq * hd, hkv * hd, hkv * hd], dim=1)
    cos, sin = rope_tables(max(lens), hd)
    plan = eng.paged_plan(rows, start, live, page_size=page)
    got = eng.paged_append(cache, 1, plan, table.cuda(), q, k, v, rope=(cos.cuda(), sin.cuda()))
    assert eng.device_error() == 0

    pos = torch.cat([torch.arange(s, s + n) for n, s in zip(rows, start)])
    c, s_ = cos[pos].double()[:, None], sin[pos].double()[:, None]
    x = qkv.double().cpu()
    qr = rotate(x[:, :hq * hd].view(total, hq, hd), c, s_).reshape(total, -1)
    # one rounding to the dtype, and fp32 arithmetic of two products (3 roundings of 2^-24)
    unit = 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -24
    size = x[:, :hq * hd].abs().amax(1, keepdim=True)
    assert ((got.double().cpu() - qr).abs() <= unit * qr.abs() + 2.0 ** -22 * size).all()

    new = {"k": rotate(x[:, hq * hd:(hq + hkv) * hd].view(total, hkv, hd), c, s_), "v": x[:, (hq + hkv) * hd:].view(total, hkv, hd)}
    for name in "kv":
        codes, scales = getattr(cache, name).cpu(), getattr(cache, name + "_scale").cpu()
        old_codes, old_scales = before[name]
        assert torch.equal(codes[0].view(torch.uint8), old_codes[0].view(torch.uint8))  # the other layer
        want, want_scale = values(old_codes[1]), old_scales[1].double().clone()
        touched = torch.zeros(pages, page, dtype=torch.bool)
        slack = torch.zeros_like(want)
        at = 0
        for i, (n, s, lv) in enumerate(zip(rows, start, live or start)):
            for slot in range(s // page, -(-(s + n) // page) if n else 0):
                p, lo, hi = int(table[i, slot]), max(s - slot * page, 0), min(s + n - slot * page, page)
                part = new[name][at + slot * page + lo - s: at + slot * page + hi - s]
                kept = [r for r in range(page) if slot * page + r < lv and not lo <= r < hi]
                for h in range(hkv):
                    scale = scale_of(float(part[:, h].abs().max()))
                    if kept:
                        scale = max(scale, float(old_scales[1, p, h]))
                        ratio = float(old_scales[1, p, h]) / scale
                        if ratio != 1:
                            want[p, h, kept] = round_e4m3(want[p, h, kept] * ratio)
                    want_scale[p, h] = scale
                    want[p, h, lo:hi] = part[:, h] / scale
                    # half an e4m3 step plus the fp32 arithmetic of the rotation
                    slack[p, h, lo:hi] = e4m3_half_step(part[:, h] / scale) + 2.0 ** -22 * float(part[:, h].abs().max()) / scale
            at += n
        assert torch.equal(scales[1].double(), want_scale)
        err = (values(codes[1]) - want).abs()
        assert (err <= slack).all(), float((err - slack).max())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_append_with_the_engines_tables_and_no_queries(dtype):
    heads, page = (12, 2, 128), 32
    eng = engine(heads, dtype)
    gen = torch.Generator().manual_seed(3)
    table, pages = make_table([45], page, gen)
    k = torch.randn(40, 256, generator=gen).to(eng.dtype).cuda()
    caches = [random_cache(eng, pages, page, torch.Generator().manual_seed(1)) for _ in range(2)]
    plan = eng.paged_plan([40], [5], page_size=page)
    assert eng.paged_append(caches[0], 0, plan, table.cuda(), None, k, k) is None
    # the tables the library computes: cos / sin of fp32 angles, in the handle's dtype
    i = torch.arange(64, dtype=torch.float32)
    angle = torch.arange(64, dtype=torch.float32)[:, None] * torch.exp(-torch.log(torch.tensor(1e6)) * i / 64)
    cos, sin = (f(angle).to(eng.dtype).float().cuda() for f in (torch.cos, torch.sin))
    eng.paged_append(caches[1], 0, plan, table.cuda(), None, k, k, rope=(cos, sin))
    assert torch.equal(caches[0].v.view(torch.uint8), caches[1].v.view(torch.uint8))
    a, b = (values(c.k.cpu()) * c.k_scale.cpu().double()[..., None, None] for c in caches)
    # the two tables may differ by one rounding of the dtype (2^-8 in bf16), a code by one step (2^-3)
    assert float((a - b).norm() / b.norm()) < 2.0 ** -6


def test_append_special_values():
    heads, page = (4, 2, 64), 16
    eng = engine(heads, "float32")
    gen = torch.Generator().manual_seed(9)
    table, pages = make_table([6], page, gen)
    cache = random_cache(eng, pages, page, gen, fill_nan=True)
    p = int(table[0, 0])
    v = torch.zeros(6, 128)
    v[0, 0], v[1, 1], v[2, 2], v[3, 3] = float("inf"), float("-inf"), float("nan"), 448.0
    plan = eng.paged_plan([6], [0], page_size=page)
    eng.paged_append(cache, 0, plan, table.cuda(), None, torch.zeros(6, 128).cuda(), v.cuda())
    got = values(cache.v.cpu())[0, p]
    assert float(cache.v_scale[0, p, 0]) == 1.0 and float(cache.v_scale[0, p, 1]) == 2.0 ** -64
    assert got[0, 0, 0] == 448 and got[0, 1, 1] == -448 and got[0, 2, 2].isnan() and got[0, 3, 3] == 448
    assert (cache.k_scale[0, p] == 2.0 ** -64).all() and (values(cache.k.cpu())[0, p, :, :6] == 0).all()
    assert (cache.v[0, p, :, 6:].view(torch.uint8) == 0x7F).all()  # rows beyond the live ones are not touched
    # the scale's boundary: 448 * 2^e fits, the next float does not
    for x, want in ((448.0 * 2.0 ** -10, 2.0 ** -10), (448.0 * 2.0 ** -10 * (1 + 2.0 ** -23), 2.0 ** -9), (1e-38, 2.0 ** -64)):
        eng.paged_append(cache, 0, plan, table.cuda(), None, torch.zeros(6, 128).cuda(), torch.full((6, 128), x).cuda())
        assert float(cache.v_scale[0, p, 0]) == want


def test_append_outside_the_pool_writes_nothing():
    eng = engine((4, 2, 64), "float32")
    cache = random_cache(eng, 3, 16, torch.Generator().manual_seed(1))
    before = cache.k.clone()
    plan = eng.paged_plan([4], [0], page_size=16)
    for bad in (-1, 3):
        eng.paged_append(cache, 0, plan, torch.tensor([[bad]], dtype=torch.int32).cuda(), None,
                         torch.ones(4, 128).cuda(), torch.ones(4, 128).cuda())
        assert eng.device_error() == 6
    assert torch.equal(before.view(torch.uint8), cache.k.view(torch.uint8))


# ---- attention -----------------------------------------------------------------------------------

def run_attention(heads, dtype, page, rows, start, live, causal, seed=0, scale=None, layers=1, qstd=1.5):
    """The call and the bound: dead rows and unused pages hold NaN codes."""
    hq, hkv, hd = heads
    eng = engine(heads, dtype)
    gen = torch.Generator().manual_seed(seed)
    live = live or list(start)
    lens = [max(lv, s + n) for n, s, lv in zip(rows, start, live)]
    table, pages = make_table(lens, page, gen)
    cache = random_cache(eng, pages, page, gen, layers=layers)
    layer = layers - 1
    dead = torch.ones(pages, page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for slot in range(-(-n // page)):
            dead[int(table[i, slot]), :min(n - slot * page, page)] = False
    for c in (cache.k, cache.v):
        c.view(torch.uint8)[layer].masked_fill_(dead.cuda()[:, None, :, None], 0x7F)
    gone = dead.all(1).cuda()
    cache.k_scale[layer][gone] = float("nan")
    cache.v_scale[layer][gone] = float("nan")
    total = sum(rows)
    q = (torch.randn(total, hq * hd + 16, generator=gen) * qstd).to(eng.dtype).cuda()[:, 8:-8]
    plan = eng.paged_plan(rows, start, live, page_size=page, causal_block=causal)
    out = eng.paged_attention(cache, layer, plan, table.cuda(), q, scale)
    assert eng.device_error() == 0
    sc = hd ** -0.5 if scale is None else scale
    clean = [torch.nan_to_num(values(c.cpu()[layer])) for c in (cache.k, cache.v)]
    ks, vs = (torch.nan_to_num(s.cpu()[layer].double()) for s in (cache.k_scale, cache.v_scale))
    ref, mag, dot = attend(q.double().cpu().view(total, hq, hd), *clean, ks, vs, table, rows, start, live, page, causal, hq, sc)
    got = out.double().cpu().view(total, hq, hd)
    # scores: hd fp32 products and sums and the exponential, 2^-24 (hd + 16) of sum |q k|, entering
    # numerator and denominator; sums over the keys: 2^-24 per key and 2^-21 for exp2; in bf16 the
    # probabilities keep 8 bits and the result is rounded once
    ds = 2.0 ** -24 * (hd + 16) * dot
    rel = 2 * ds + 2.0 ** -24 * max(lens, default=0) + 2.0 ** -21
    bound = (rel + (2.0 ** -8 if dtype == "bfloat16" else 0)) * mag + (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -23) * ref.abs()
    err = (got - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), float((err / bound).max())
    return out


MASKS = {
    "one-key": ([1], [0], None, 0),
    "odd": ([1], [396], None, 0),
    "ragged-tokens": ([1, 1, 1, 1, 1], [0, 63, 64, 700, 1291], None, 0),
    "empty-request": ([1, 0, 5], [65, 10, 0], None, 0),
    "block-step": ([32, 32, 8], [512, 64, 130], [512, 64, 160], 0),
    "partial": ([8, 8], [1000, 24], [1024, 32], 0),
    "mixed": ([1, 33, 8, 1, 130], [800, 100, 31, 2, 0], None, 0),
    "causal-32": ([97, 300], [32, 0], None, 32),
    "causal-1": ([65, 3, 1], [0, 131, 77], None, 1),
    "causal-ahead": ([8, 16], [8, 128], [40, 256], 32),
}


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("mask", list(MASKS))
def test_attention_matches_the_definition(mask, heads, dtype):
    rows, start, live, causal = MASKS[mask]
    run_attention(heads, dtype, 32, rows, start, live, causal, seed=len(mask))


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 2, 64)], ids=str)
@pytest.mark.parametrize("mask", ["odd", "mixed", "causal-32", "partial"])
def test_attention_page_sizes(mask, heads, page):
    rows, start, live, causal = MASKS[mask]
    run_attention(heads, "bfloat16", page, rows, start, live, causal, seed=page, layers=2)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows", [1, 8, 40])
def test_attention_long_split_keys(rows, dtype):
    run_attention((12, 2, 128), dtype, 64, [rows], [6001], None, 0, seed=rows)


@pytest.mark.parametrize("heads", [(12, 2, 128), (8, 1, 128), (4, 2, 64), (8, 8, 64)], ids=str)
def test_attention_split_tiles_of_every_size_in_one_call(heads):
    # tiles of all sizes with their keys cut into 2 to 12 shares, beside a request that ends in its first page
    run_attention(heads, "bfloat16", 32, [1, 3, 5, 8, 11, 16, 21, 40, 2],
                  [3071, 2500, 1900, 3300, 1025, 2047, 2600, 1500, 9], None, 0, seed=heads[0])


@pytest.mark.parametrize("rows", [1, 32])
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scales(scale, rows):
    # scale 0: the mean of the values; 1.0: scores of some tens, one key dominates
    run_attention((12, 2, 128), "bfloat16", 32, [rows], [200], None, 0, seed=5, scale=scale, qstd=1.0)


@pytest.mark.parametrize("rows", [1, 32])
def test_attention_a_sink_and_many_small_weights(rows):
    """One key outweighs each of 4000 others by 2^20, whose sum still matters: no weight is lost."""
    heads, page, n = (12, 2, 128), 32, 4001
    eng = engine(heads, "bfloat16")
    gen = torch.Generator().manual_seed(2)
    start = n - rows
    table, pages = make_table([n], page, gen, spare=0, width_extra=0)
    cache = eng.new_paged_cache(pages, page_size=page, layers=1)
    one = torch.tensor(1.0).to(torch.float8_e4m3fn).view(torch.uint8)
    cache.v.view(torch.uint8).fill_(int(one))        # values 1 with scale 1 ...
    p0 = int(table[0, 0])
    cache.v.view(torch.uint8)[0, p0, :, 0] = 0       # ... but 0 at the sink
    cache.k.view(torch.uint8)[0, p0, :, 0, 0] = int(one)
    q = torch.zeros(rows, 12, 128)
    q[:, :, 0] = 20.0
    q = q.view(rows, -1).to(torch.bfloat16).cuda()
    out = eng.paged_attention(cache, 0, eng.paged_plan([rows], [start], page_size=page), table.cuda(), q,
                              scale=0.6931471805599453)  # the sink scores 2^20, the others 1
    want = (n - 1) / (2.0 ** 20 + n - 1)
    assert float((out.double() - want).abs().max()) <= want * (2.0 ** -8 + 2.0 ** -8)


def test_attention_scores_and_scales_of_extreme_range():
    """Page scales from 2^-30 to 2^20: the weights of a small-scaled page are not lost beside a large one."""
    heads, page = (12, 2, 128), 32
    eng = engine(heads, "bfloat16")
    for rows in (1, 32):
        gen = torch.Generator().manual_seed(rows)
        table, pages = make_table([256], page, gen, spare=0, width_extra=0)
        cache = random_cache(eng, pages, page, gen)
        cache.v_scale[0, :, 0] = 2.0 ** torch.tensor([-30, 20, -10, 0, 5, -3, 11, -25]).float().cuda()
        q = torch.randn(rows, 1536, generator=gen).to(torch.bfloat16).cuda()
        out = eng.paged_attention(cache, 0, eng.paged_plan([rows], [256 - rows], page_size=page), table.cuda(), q)
        ref, mag, _ = attend(q.double().cpu().view(rows, 12, 128), values(cache.k.cpu()[0]), values(cache.v.cpu()[0]),
                             cache.k_scale.cpu()[0].double(), cache.v_scale.cpu()[0].double(), table, [rows], [256 - rows],
                             [256 - rows], page, 0, 12, 128 ** -0.5)
        err = (out.double().cpu().view_as(ref) - ref).abs()
        assert (err <= 2.0 ** -7 * mag).all()


def test_attention_past_32_bit_offsets():
    """Pages beyond 4 GiB of codes."""
    heads, page = (12, 2, 128), 128
    eng = engine(heads, "bfloat16")
    pages = (1 << 32) // (2 * page * 128) + 7
    cache = eng.new_paged_cache(pages, page_size=page, layers=1)
    gen = torch.Generator().manual_seed(4)
    ids = torch.tensor([[pages - 1, 0, pages - 4]], dtype=torch.int32)
    kv = [torch.randn(300, 256, generator=gen).to(torch.bfloat16).cuda() for _ in range(2)]
    q = torch.randn(300, 1536, generator=gen).to(torch.bfloat16).cuda()
    plan = eng.paged_plan([300], [0], page_size=page)
    eng.paged_append(cache, 0, plan, ids.cuda(), None, *kv)
    small = eng.new_paged_cache(3, page_size=page, layers=1)
    low = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
    eng.paged_append(small, 0, plan, low, None, *kv)
    for a, b in zip(ids[0].tolist(), [2, 0, 1]):
        assert torch.equal(cache.k[0, a].view(torch.uint8), small.k[0, b].view(torch.uint8))
        assert torch.equal(cache.v_scale[0, a], small.v_scale[0, b])
    for rows in (300, 1):
        p = eng.paged_plan([rows], [300 - rows], page_size=page)
        assert torch.equal(eng.paged_attention(cache, 0, p, ids.cuda(), q[:rows]),
                           eng.paged_attention(small, 0, p, low, q[:rows]))
    del cache


@pytest.mark.parametrize("rows", [1, 8, 32])
def test_attention_repeats_bit_for_bit_and_on_another_stream(rows):
    heads = (12, 2, 128)
    eng = engine(heads, "bfloat16")
    gen = torch.Generator().manual_seed(rows)
    table, pages = make_table([3000, 700], 32, gen)
    cache = random_cache(eng, pages, 32, gen)
    q = torch.randn(2 * rows, 1536, generator=gen).to(torch.bfloat16).cuda()
    plan = eng.paged_plan([rows, rows], [3000 - rows, 700 - rows])
    t = table.cuda()
    first = eng.paged_attention(cache, 0, plan, t, q)
    for _ in range(3):
        assert torch.equal(first, eng.paged_attention(cache, 0, plan, t, q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eng.paged_attention(cache, 0, plan, t, q)
    side.synchronize()
    assert torch.equal(first, other)


def test_page_id_outside_the_pool_is_reported():
    eng = engine((12, 2, 128), "bfloat16")
    for rows in (1, 32):
        cache = eng.new_paged_cache(2, layers=1)
        q = torch.zeros(rows, 1536, dtype=torch.bfloat16, device="cuda")
        eng.paged_attention(cache, 0, eng.paged_plan([rows], [0]), torch.tensor([[2]], dtype=torch.int32).cuda(), q)
        assert eng.device_error() == 6


# ---- refusals ------------------------------------------------------------------------------------

def test_refusals():
    eng = engine((12, 2, 128), "bfloat16")
    cache = eng.new_paged_cache(4, page_size=32, layers=2)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    plan = eng.paged_plan([8], [40])
    q = torch.zeros(8, 1536, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(8, 256, dtype=torch.bfloat16, device="cuda")
    for args in (([-1], [0], None), ([1], [-1], None), ([1], [5], [4]), ([1], [0, 1], None), ([1 << 30], [1 << 29], None)):
        with pytest.raises(ValueError):
            eng.paged_plan(*args)
    for kw in (dict(page_size=24), dict(page_size=0), dict(causal_block=-1)):
        with pytest.raises(ValueError):
            eng.paged_plan([1], [0], **kw)
    with pytest.raises(ValueError):
        eng.new_paged_cache(4, page_size=8)
    with pytest.raises(ValueError):  # layer
        eng.paged_attention(cache, 2, plan, table, q)
    with pytest.raises(ValueError):  # table too narrow
        eng.paged_attention(cache, 0, plan, table[:, :1].contiguous(), q)
    with pytest.raises(ValueError):  # table rows
        eng.paged_attention(cache, 0, plan, table.expand(2, 2).contiguous(), q)
    with pytest.raises(ValueError):  # table type
        eng.paged_attention(cache, 0, plan, table.long(), q)
    with pytest.raises(ValueError):  # page size of the plan
        eng.paged_attention(cache, 0, eng.paged_plan([8], [40], page_size=16), torch.zeros(1, 3, dtype=torch.int32, device="cuda"), q)
    with pytest.raises(ValueError):  # rows, dtype, columns, device
        eng.paged_attention(cache, 0, plan, table, q[:7])
    with pytest.raises(ValueError):
        eng.paged_attention(cache, 0, plan, table, q.float())
    with pytest.raises(ValueError):
        eng.paged_attention(cache, 0, plan, table, q[:, :1024])
    with pytest.raises(ValueError):
        eng.paged_attention(cache, 0, plan, table, q.cpu())
    with pytest.raises(ValueError):
        eng.paged_attention(cache, 0, plan, table, q, scale=float("nan"))
    with pytest.raises(ValueError):  # another head layout's cache
        eng.paged_attention(engine((4, 2, 64), "bfloat16").new_paged_cache(4, layers=1), 0, plan, table, q)
    cos, sin = (t.cuda() for t in rope_tables(47, 128))
    with pytest.raises(ValueError):  # 48 positions needed
        eng.paged_append(cache, 0, plan, table, q, k, k, rope=(cos, sin))
    with pytest.raises(ValueError):
        eng.paged_append(cache, 0, plan, table, q, k, k, rope=(cos.double(), sin.double()))
    with pytest.raises(ValueError):
        eng.paged_append(cache, 0, eng.paged_plan([8], [16380]), torch.zeros(1, 600, dtype=torch.int32, device="cuda"), q, k, k)
    with pytest.raises(ValueError):
        eng.paged_append(cache, 0, plan, table, q, k[:, :128], k)
    empty = eng.paged_plan([], [])
    assert eng.paged_attention(cache, 0, empty, table[:0], q[:0]).shape == (0, 1536)
    assert eng.device_error() == 0


@pytest.mark.parametrize("other", [((8, 1, 128), "bfloat16"), ((16, 4, 128), "bfloat16"), ((4, 2, 64), "bfloat16"),
                                   ((12, 2, 128), "float32")], ids=str)
def test_a_plan_for_other_heads_or_another_type_is_refused(other):
    eng = engine((12, 2, 128), "bfloat16")
    plan = engine(*other).paged_plan([8], [40])
    cache = eng.new_paged_cache(4, layers=1)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    q = torch.zeros(8, 1536, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="laid out for"):
        eng.paged_attention(cache, 0, plan, table, q)
    with pytest.raises(ValueError, match="laid out for"):
        eng.paged_append(cache, 0, plan, table, q, q[:, :256], q[:, :256])


def test_unaligned_rows_are_copied():
    eng = engine((12, 2, 128), "bfloat16")
    gen = torch.Generator().manual_seed(8)
    table, pages = make_table([50], 32, gen)
    cache = random_cache(eng, pages, 32, gen)
    wide = torch.randn(3, 1537, generator=gen).to(torch.bfloat16).cuda()
    plan = eng.paged_plan([3], [47])
    a = eng.paged_attention(cache, 0, plan, table.cuda(), wide[:, 1:])
    b = eng.paged_attention(cache, 0, plan, table.cuda(), wide[:, 1:].contiguous())
    assert torch.equal(a, b)
