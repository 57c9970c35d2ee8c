"""The model over a paged 8-bit cache (fdllm_forward_paged, generate_batch(pool=...), paged scoring) against
the CPU oracle with the same cache rounding."""

import pytest
import torch

from _paged_util import PagedOracle, make_table
from fast_dllm_relax_b200.config import TINY, TINY_MASK_ID, make_synthetic_params
from fast_dllm_relax_b200.paged import PagedPool
from oracle.decode import relax_greedy_generate
from oracle.model import confidence
from tests._oracle_util import oracle_config

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["float32", "bfloat16"])
def pair(request):
    from fast_dllm_relax_b200.engine import Engine
    params = make_synthetic_params(TINY, seed=0, dtype=request.param, mask_id=TINY_MASK_ID)
    return Engine(TINY, [p.cuda() for p in params], dtype=request.param), PagedOracle(oracle_config(TINY), params, request.param)


def oracle_cache(cap=512):
    shape = (TINY.num_hidden_layers, 1, cap, TINY.num_key_value_heads, TINY.head_dim)
    return torch.zeros(shape), torch.zeros(shape)


def bound(eng):
    """Relative L2 error of hidden states.  fp32: a code differs where two fp32 sums fall on either side of a
    rounding midpoint, about 2^-16 of them, by 2^-4 of the value: 2^-12 of the norm, times 4 layers' terms.
    bf16: every projection rounds to 2^-9 in another order, a code moves by 2^-4 for about 2^-4 of them and
    averages over the keys."""
    return 2.0 ** -10 if eng.dtype == torch.float32 else 2.0 ** -5


@pytest.mark.parametrize("page", [16, 32, 64])
def test_forward_paged_matches_the_oracle(pair, page):
    eng, orc = pair
    orc.page = page
    gen = torch.Generator().manual_seed(page)
    lens = [96, 45, 160]
    ids = [torch.randint(0, 1000, (n,), generator=gen, dtype=torch.int32) for n in lens]
    block = torch.randint(0, 1000, (3, 32), generator=gen, dtype=torch.int32)
    table, pages = make_table([n + 32 for n in lens], page, gen)
    cache, table = eng.new_paged_cache(pages, page_size=page), table.cuda()
    plan = eng.paged_plan(lens, [0, 0, 0], page_size=page, causal_block=32)
    h = eng.forward_paged(eng.embed(torch.cat(ids).cuda()), cache, plan, table)
    caches = [oracle_cache() for _ in lens]
    want = [orc._paged_forward(orc.embed(i)[None], k, v, 0, 0, 32)[0] for i, (k, v) in zip(ids, caches)]
    want = torch.cat(want)
    assert float((h.float().cpu() - want.float()).norm() / want.float().norm()) < bound(eng)
    # a full step over all three, then an 8-row partial step of the middle one beside a single token
    plan = eng.paged_plan([32] * 3, lens, page_size=page)
    h = eng.forward_paged(eng.embed(block.reshape(-1).cuda()), cache, plan, table)
    want = torch.cat([orc.forward_cached(orc.embed(b)[None], k, v, n, n)[0] for b, n, (k, v) in zip(block, lens, caches)])
    assert float((h.float().cpu() - want.float()).norm() / want.float().norm()) < bound(eng)
    new = torch.randint(0, 1000, (9,), generator=gen, dtype=torch.int32)
    plan = eng.paged_plan([0, 8, 1], [lens[0], lens[1] + 8, lens[2] + 31], [lens[0], lens[1] + 32, lens[2] + 32], page_size=page)
    h = eng.forward_paged(eng.embed(new.cuda()), cache, plan, table)
    want = torch.cat([orc.forward_cached(orc.embed(new[:8])[None], *caches[1], 0, lens[1], 8, 32)[0],
                      orc.forward_cached(orc.embed(new[8:])[None], *caches[2], 0, lens[2], 31, 32)[0]])
    assert float((h.float().cpu() - want.float()).norm() / want.float().norm()) < bound(eng)
    assert eng.device_error() == 0


def test_paged_generation_matches_the_oracle(pair):
    """fp32: the tokens of the reference's loop over the oracle with the same cache rounding."""
    from fast_dllm_relax_b200.batch_decode import generate_batch
    eng, orc = pair
    orc.page = 32
    gen = torch.Generator().manual_seed(11)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (64, 45, 96)]
    pool = PagedPool(eng.new_paged_cache(40))
    for use_block_cache in (False, True):
        kw = dict(max_new_tokens=40, block_size=32, small_block_size=8, threshold=0.9, use_block_cache=use_block_cache,
                  mask_id=TINY_MASK_ID)
        toks, stats = generate_batch(eng, prompts, pool=pool, **kw)
        assert pool.free_pages == 40
        assert all(s["block_recomputes"] > 0 for s in stats)
        if eng.dtype == torch.float32:
            for p, t in zip(prompts, toks):
                assert t == relax_greedy_generate(orc, p, **kw)[0]
    with pytest.raises(MemoryError):
        generate_batch(eng, prompts, pool=PagedPool(eng.new_paged_cache(2)), **kw)


def test_paged_scoring(pair):
    from fast_dllm_relax_b200.scorebench import score_batch_paged
    eng, orc = pair
    orc.page = 32
    gen = torch.Generator().manual_seed(12)
    b, C, N, top = 3, 64, 5, 4
    ctx = torch.randint(0, 1000, (b, C), generator=gen, dtype=torch.int32)
    blocks = torch.full((b, 32), TINY_MASK_ID, dtype=torch.int32)
    targets = torch.randint(0, 1000, (b, 32), generator=gen, dtype=torch.int32)
    pool = PagedPool(eng.new_paged_cache(b * 3))
    sums, ent, ids, tlp = score_batch_paged(eng, pool, ctx.cuda(), blocks.cuda(), targets.cuda(), N, top)
    assert pool.free_pages == b * 3 and ids.shape == (b, N, top)
    tol = 64 * bound(eng)  # logits of size sqrt(hidden) * 0.02 per unit of hidden error, a few units
    for i in range(b):
        k, v = oracle_cache()
        orc.build_prefix_cache(orc.embed(ctx[i])[None], None, k, v)
        h = orc.forward_cached(orc.embed(blocks[i])[None], k, v, C, C)
        logp = torch.log_softmax(orc.get_logits(h)[0, :N].double(), -1)
        assert abs(float(sums[i]) - float(logp.gather(1, targets[i, :N, None].long()).sum())) < tol * N
        assert float((ent[i].cpu() + (logp.exp() * logp).sum(-1)).abs().max()) < tol
        assert float((tlp[i].cpu() - logp.sort(-1, descending=True)[0][:, :top]).abs().max()) < tol


def test_forward_paged_refusals(pair):
    eng, _ = pair
    cache = eng.new_paged_cache(4)
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    plan = eng.paged_plan([32], [0])
    x = eng.embed(torch.zeros(32, dtype=torch.int32))
    with pytest.raises(ValueError):  # one layer's cache
        eng.forward_paged(x, eng.new_paged_cache(4, layers=1), plan, table)
    with pytest.raises(ValueError):
        eng.forward_paged(x[:31], cache, plan, table)
    with pytest.raises(ValueError):  # positions beyond the model's
        eng.forward_paged(x, cache, eng.paged_plan([32], [TINY.context_window_size]), torch.zeros(1, 200, dtype=torch.int32, device="cuda"))
