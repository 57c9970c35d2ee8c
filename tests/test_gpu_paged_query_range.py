"""Paged attention with queries at the ends of their type: infinities and NaN, and finite values up to the largest."""

import math

import pytest
import torch

from _paged_util import attend, make_table, values
from test_gpu_paged_cache import engine, random_cache

pytestmark = pytest.mark.gpu

LENGTHS = [40, 700]  # one share, and several where the rows are few


def call(eng, rows, length, q, cache, table):
    return eng.paged_attention(cache, 0, eng.paged_plan([rows], [length - rows]), table.cuda(), q)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 2, 64)], ids=str)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_query_that_is_not_finite_gives_nan_and_leaves_the_others(bad, heads, dtype):
    hq, hkv, hd = heads
    eng = engine(heads, dtype)
    for rows in (1, 5, 8, 32):
        for length in LENGTHS:
            gen = torch.Generator().manual_seed(rows)
            table, pages = make_table([length], 32, gen)
            cache = random_cache(eng, pages, 32, gen)
            q = torch.randn(rows, hq, hd, generator=gen)
            good = call(eng, rows, length, q.view(rows, -1).to(eng.dtype).cuda(), cache, table).view(rows, hq, hd)
            t, h = rows // 2, hq - 2
            q[t, h, hd // 3] = bad
            got = call(eng, rows, length, q.view(rows, -1).to(eng.dtype).cuda(), cache, table).view(rows, hq, hd)
            assert got[t, h].isnan().all(), (rows, length)
            other = torch.ones(rows, hq, dtype=torch.bool)
            other[t, h] = False
            assert torch.equal(got[other.cuda()], good[other.cuda()]), (rows, length)
    assert eng.device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 2, 64)], ids=str)
def test_an_infinite_query_whose_every_score_is_minus_infinity_gives_nan(heads, dtype):
    """-inf times a positive column of every key: no weight is defined, and zeros would read as an empty row."""
    hq, hkv, hd = heads
    eng = engine(heads, dtype)
    gen = torch.Generator().manual_seed(1)
    table, pages = make_table([300], 32, gen)
    cache = random_cache(eng, pages, 32, gen)
    cache.k.view(torch.uint8)[..., 3] = 0x38  # 1.0
    for rows in (1, 5, 8, 32):
        q = torch.zeros(rows, hq, hd)
        q[0, 0, 3] = -math.inf
        got = call(eng, rows, 300, q.view(rows, -1).to(eng.dtype).cuda(), cache, table).view(rows, hq, hd)
        assert got[0, 0].isnan().all(), rows
        assert got[0, 1:].isfinite().all() and got[1:].isfinite().all(), rows


@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 2, 64)], ids=str)
@pytest.mark.parametrize("exponent", [-100, 100, 116])
def test_finite_queries_of_any_size(heads, exponent):
    """Queries of 2^exponent over keys of 2^-exponent: the scores, and so the results, are ordinary."""
    hq, hkv, hd = heads
    eng = engine(heads, "bfloat16")
    for rows in (1, 5, 8, 32):
        for length in LENGTHS:
            gen = torch.Generator().manual_seed(rows)
            table, pages = make_table([length], 32, gen)
            cache = random_cache(eng, pages, 32, gen)
            cache.k_scale.copy_(torch.ldexp(cache.k_scale.cpu(), torch.tensor(-exponent)))
            q = torch.ldexp(torch.randn(rows, hq, hd, generator=gen), torch.tensor(exponent)).to(torch.bfloat16)
            got = call(eng, rows, length, q.view(rows, -1).cuda(), cache, table).double().cpu().view(rows, hq, hd)
            ref, mag, _ = attend(q.double(), values(cache.k.cpu()[0]), values(cache.v.cpu()[0]),
                                 cache.k_scale.cpu()[0].double(), cache.v_scale.cpu()[0].double(), table, [rows],
                                 [length - rows], [length - rows], 32, 0, hq, hd ** -0.5)
            assert ((got - ref).abs() <= 2.0 ** -7 * mag).all(), (rows, length)
