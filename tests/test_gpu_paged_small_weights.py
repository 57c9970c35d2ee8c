"""Paged attention past a sink: one key outweighs every other by 2^20 and more but has no value, so the result is
made of the small weights alone.  A weight of 2^-22 of the largest must keep 10 bits (as a half-precision number
does whose largest is 2^8 or more), whatever the number of query rows."""

import pytest
import torch

from _paged_util import attend, make_table, values
from test_gpu_paged_cache import engine

pytestmark = pytest.mark.gpu

LN2 = 0.6931471805599453
HEADS = (12, 2, 128)


def sink_cache(eng, n, page, gen, k_rest, v_rest):
    """One request of n keys: key 0 is 1 in column 0 with value 0, the others k_rest [n] there, v_rest [n, 128]."""
    table, pages = make_table([n], page, gen, spare=0, width_extra=0)
    cache = eng.new_paged_cache(pages, page_size=page, layers=1)
    k = torch.zeros(pages * page, 128)
    v = torch.zeros(pages * page, 128)
    k[1:n, 0], v[1:n] = k_rest[1:], v_rest[1:]
    k[0, 0] = 1.0
    ids = table[0].long()
    for to, x in ((cache.k, k), (cache.v, v)):
        codes = x.to(torch.float8_e4m3fn).view(torch.uint8).view(pages, 1, page, 128).expand(-1, 2, -1, -1)
        to.view(torch.uint8)[0, ids.cuda()] = codes.cuda()
    return cache, table


@pytest.mark.parametrize("rows", [1, 5, 8, 9, 32])
@pytest.mark.parametrize("weight", [20.25, 21.5, 22.375, 23.625])
def test_equal_weights_beside_a_sink(rows, weight):
    eng, n = engine(HEADS, "bfloat16"), 241  # the keys of one share
    gen = torch.Generator().manual_seed(rows)
    cache, table = sink_cache(eng, n, 32, gen, torch.zeros(n), torch.ones(n, 128))
    q = torch.zeros(rows, 12, 128)
    q[:, :, 0] = weight  # exact in bf16: the sink scores 2^weight, the others 1
    out = eng.paged_attention(cache, 0, eng.paged_plan([rows], [n - rows]), table.cuda(),
                              q.view(rows, -1).to(torch.bfloat16).cuda(), scale=LN2)
    want = (n - 1) / (2.0 ** weight + n - 1)
    # 2^-9 for the result's bf16; at 2^-23.6 of the largest, 2^-15.6 as seated, half a step of 2^-24 is 2^-9.4
    assert float((out.double() - want).abs().max()) <= want * 2.0 ** -8 * 1.5


@pytest.mark.parametrize("rows", [1, 5, 8, 9, 32])
@pytest.mark.parametrize("page", [16, 128])
def test_spread_weights_beside_a_sink(rows, page):
    eng, n = engine(HEADS, "bfloat16"), 12003
    gen = torch.Generator().manual_seed(rows)
    # scores of 0 to 22 / 16 of the sink's exponent in steps that e4m3 holds, values of one sign
    k_rest = torch.randint(0, 9, (n,), generator=gen).float() / 128
    v_rest = torch.rand(n, 128, generator=gen) + 0.5
    cache, table = sink_cache(eng, n, page, gen, k_rest, v_rest)
    q = torch.zeros(rows, 12, 128)
    q[:, :, 0] = torch.tensor([20.0, 21.0, 21.5, 22.0, 20.5, 22.25])[None, :].repeat(rows, 2)
    q = q.to(torch.bfloat16)
    out = eng.paged_attention(cache, 0, eng.paged_plan([rows], [n - rows], page_size=page), table.cuda(),
                              q.view(rows, -1).cuda(), scale=LN2)
    ref, _, _ = attend(q.double(), values(cache.k.cpu()[0]), values(cache.v.cpu()[0]), cache.k_scale.cpu()[0].double(),
                       cache.v_scale.cpu()[0].double(), table, [rows], [n - rows], [n - rows], page, 0, 12, LN2)
    err = (out.double().cpu().view_as(ref) - ref).abs()
    assert (err <= 2.0 ** -8 * ref).all(), float((err / ref).max())


def test_a_row_does_not_depend_on_the_tile_it_lands_in():
    """The same query alone, among few and among many rows: bf16 results within one rounding of each other."""
    eng, n = engine(HEADS, "bfloat16"), 251
    gen = torch.Generator().manual_seed(3)
    cache, table = sink_cache(eng, n, 32, gen, torch.randint(-8, 9, (n,), generator=gen).float() / 64,
                              torch.randn(n, 128, generator=gen) * 0.1 + 1)
    q = torch.zeros(40, 12, 128)
    q[:, :, 0] = 21.5
    q = q.view(40, -1).to(torch.bfloat16).cuda()
    outs = [eng.paged_attention(cache, 0, eng.paged_plan([r], [n - r]), table.cuda(), q[:r], scale=LN2)[:1].double()
            for r in (1, 4, 8, 9, 40)]
    for o in outs[1:]:
        assert ((o - outs[0]).abs() <= 2.0 ** -7 * outs[0].abs()).all()
