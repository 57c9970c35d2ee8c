"""Paged attention with finite queries and keys whose scores pass fp32's range: NaN, never a finite wrong result."""

import pytest
import torch

from _paged_util import make_table
from test_gpu_paged_cache import engine, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 2, 64)], ids=str)
@pytest.mark.parametrize("length", [40, 700])
def test_scores_beyond_fp32_give_nan(length, heads, dtype):
    hq, hkv, hd = heads
    eng = engine(heads, dtype)
    for rows in (1, 5, 8, 32):
        gen = torch.Generator().manual_seed(rows)
        table, pages = make_table([length], 32, gen)
        cache = random_cache(eng, pages, 32, gen)
        cache.k.view(torch.uint8)[..., 5] = 0x78  # 256, under the largest scale the append gives such a value
        cache.k_scale.fill_(2.0 ** 10)
        q = torch.randn(rows, hq, hd, generator=gen)
        q[0, 0], q[0, 0, 5] = 0.0, 2.0 ** 126  # every score of the row is 2^144 head_dim ** -0.5
        q[:, 1:] *= 2.0 ** -12
        plan = eng.paged_plan([rows], [length - rows])
        got = eng.paged_attention(cache, 0, plan, table.cuda(), q.view(rows, -1).to(eng.dtype).cuda()).view(rows, hq, hd)
        assert got[0, 0].isnan().all(), rows
        assert got[0, 1:].isfinite().all(), rows
    assert eng.device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads", [(12, 2, 128), (4, 2, 64)], ids=str)
def test_a_negative_scale_is_the_scale_of_negated_queries(heads, dtype):
    hq, hkv, hd = heads
    eng = engine(heads, dtype)
    for rows, length in ((1, 700), (5, 130), (8, 700), (32, 300)):
        gen = torch.Generator().manual_seed(rows)
        table, pages = make_table([length], 32, gen)
        cache, table = random_cache(eng, pages, 32, gen), table.cuda()
        q = torch.randn(rows, hq * hd, generator=gen).to(eng.dtype).cuda()
        plan = eng.paged_plan([rows], [length - rows])
        assert torch.equal(eng.paged_attention(cache, 0, plan, table, q, scale=-0.2),
                           eng.paged_attention(cache, 0, plan, table, -q, scale=0.2))
