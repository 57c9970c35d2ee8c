"""Appending to pages whose present scale is not a power of two (a cache that another program filled):
code = e4m3(value / scale), the quotient rounded once."""

import numpy as np
import pytest
import torch

from _paged_util import make_table, round_e4m3, rope_tables, rotate, values
from test_gpu_paged_cache import engine

pytestmark = pytest.mark.gpu


def ties(scale):
    """fp32 values whose quotient by `scale` is exactly half way between two codes."""
    t = np.concatenate([(16 + 2 * np.arange(8) + 1) / 16 * 2.0 ** e for e in range(-4, 4)])
    x = (t * np.float64(scale)).astype(np.float32)
    assert (x.astype(np.float64) == t * np.float64(scale)).all()  # the scale has few bits
    return x


@pytest.mark.parametrize("heads,page", [((4, 2, 64), 16), ((12, 2, 128), 32), ((4, 4, 32), 64)], ids=str)
def test_codes_are_the_rounded_quotients(heads, page):
    hq, hkv, hd = heads
    eng = engine(heads, "float32")
    rng = np.random.default_rng(page)
    kept, new = 3, page - 5
    table, pages = make_table([kept + new], page, torch.Generator().manual_seed(1))
    p = int(table[0, 0])
    plan = eng.paged_plan([new], [kept], page_size=page)
    cos, sin = rope_tables(page, hd)
    differing = 0
    for _ in range(24):
        scale = np.float32((513 + 2 * rng.integers(0, 255)) / 512)  # ten bits, odd
        inv = np.float32(1) / scale
        x = ties(scale)
        odd = x * inv != (x.astype(np.float64) / np.float64(scale)).astype(np.float32)
        differing += int(odd.sum())
        x = np.resize(np.concatenate([x[odd], x]), (new, hkv * hd))
        v = torch.from_numpy(x)
        cache = eng.new_paged_cache(pages, page_size=page, layers=1)
        cache.k_scale.fill_(float(scale))
        cache.v_scale.fill_(float(scale))
        cache.v.view(torch.uint8)[0, p, :, :kept] = 0x39
        eng.paged_append(cache, 0, plan, table.cuda(), None, v.cuda(), v.cuda(), rope=(cos.cuda(), sin.cuda()))
        assert (cache.v_scale[0, p] == float(scale)).all()
        want = round_e4m3(v.double() / float(scale)).view(new, hkv, hd).transpose(0, 1)
        assert torch.equal(values(cache.v.cpu())[0, p, :, kept:kept + new], want)
        assert (cache.v.view(torch.uint8)[0, p, :, :kept] == 0x39).all()
        # the keys are rotated first: within half a step and the rotation's fp32 arithmetic
        k = rotate(v.double().view(new, hkv, hd), *(t[kept:kept + new].double()[:, None] for t in (cos, sin)))
        got = values(cache.k.cpu())[0, p, :, kept:kept + new].transpose(0, 1)
        quotient = k / float(scale)
        step = torch.exp2((torch.frexp(quotient)[1].clamp(min=-5) - 5).double())
        assert ((got - quotient).abs() <= step + 2.0 ** -21 * quotient.abs().max()).all()
    assert differing > 0  # a product with the rounded inverse would give other codes
    assert eng.device_error() == 0
