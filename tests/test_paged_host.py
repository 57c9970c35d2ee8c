"""Host side of the paged cache, without a GPU: the pool's pages, and that they come back whatever ends a call."""

import pytest
import torch

from fast_dllm_relax_b200.batch_decode import generate_batch
from fast_dllm_relax_b200.paged import PagedCache, PagedPool
from fast_dllm_relax_b200.scorebench import score_batch_paged

PAGE = 32


def cache(pages, page=PAGE, layers=1):
    codes = [torch.zeros(layers, pages, 2, page, 64, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    return PagedCache(*codes, torch.ones(layers, pages, 2), torch.ones(layers, pages, 2))


class Plan:
    def __init__(self, rows):
        self.total_rows = sum(rows)


class HostEngine:
    """The calls that generate_batch and score_batch_paged make, on the CPU: every step commits token 7, and
    `fail_at` raises in that forward over the pages."""

    device = torch.device("cpu")

    class cfg:
        bd_size = 32

    def __init__(self, pool, fail_at=None):
        self.pool, self.fail_at, self.forwards, self.most = pool, fail_at, 0, 0

    def embed(self, ids):
        return torch.zeros(ids.numel(), 4)

    def paged_plan(self, rows, start, live=None, *, page_size, causal_block=0):
        return Plan(rows)

    def forward_paged(self, x, cache, plan, table, hidden=True):
        assert x.shape[0] == plan.total_rows
        used = table.flatten().tolist()
        self.most = max(self.most, cache.pages - self.pool.free_pages)
        assert all(0 <= p < cache.pages for p in used)
        self.forwards += 1
        if self.forwards == self.fail_at:
            raise RuntimeError("device lost")
        return torch.zeros(plan.total_rows, 4) if hidden else None

    def forward_hidden(self, x, bias):
        return x

    def get_logits(self, hidden):
        return torch.zeros(*hidden.shape[:-1], 16)

    def logprobs(self, logits, targets, top):
        n = targets.numel()
        return torch.zeros(n), torch.zeros(n), torch.zeros(n, top, dtype=torch.int32), torch.zeros(n, top)

    def confidence(self, hidden):
        return torch.zeros(hidden.shape[0], dtype=torch.int32), torch.ones(hidden.shape[0])

    def unmask_batch(self, ids, conf, desc, threshold):
        out = torch.zeros(desc.shape[0], 2 + 32, dtype=torch.int32)
        for j, (_, _, _, win, bits) in enumerate(desc.tolist()):
            out[j, 0], out[j, 1] = bits & ((1 << win) - 1), 7
            out[j, 2:] = 7
        return out


KW = dict(max_new_tokens=64, block_size=32, small_block_size=8, threshold=0.9, mask_id=15)
PROMPTS = [[1] * 64, [2] * 45, [3] * 96, [4] * 200]


def run(pool, **kw):
    eng = HostEngine(pool, **kw)
    return eng, generate_batch(eng, PROMPTS, pool=pool, **KW)


def test_pages_come_back_when_all_requests_are_done():
    pool = PagedPool(cache(64))
    eng, (tokens, _) = run(pool)
    assert pool.free_pages == 64 and eng.most > 8 and all(set(t) == {7} for t in tokens)
    assert sorted(pool._free) == list(range(64))


@pytest.mark.parametrize("fail_at", [1, 2, 3, 7])
def test_pages_come_back_when_a_forward_fails(fail_at):
    pool = PagedPool(cache(64))
    with pytest.raises(RuntimeError, match="device lost"):
        run(pool, fail_at=fail_at)
    assert sorted(pool._free) == list(range(64))
    run(pool)  # the pool serves the next batch
    assert sorted(pool._free) == list(range(64))


@pytest.mark.parametrize("pages", [1, 2, 5, 9, 13, 16])
def test_pages_come_back_when_the_pool_is_too_small(pages):
    pool = PagedPool(cache(pages))
    with pytest.raises(MemoryError):
        run(pool)
    assert sorted(pool._free) == list(range(pages))


@pytest.mark.parametrize("pages,fail_at,error", [(2, None, MemoryError), (7, None, MemoryError), (64, 1, RuntimeError),
                                                 (64, 2, RuntimeError), (64, None, None)])
def test_scoring_gives_its_pages_back(pages, fail_at, error):
    pool = PagedPool(cache(pages))
    eng = HostEngine(pool, fail_at=fail_at)
    ctx, blocks = torch.zeros(3, 64, dtype=torch.int32), torch.zeros(3, 32, dtype=torch.int32)
    if error is None:
        score_batch_paged(eng, pool, ctx, blocks, blocks, 5, 2)
    else:
        with pytest.raises(error):
            score_batch_paged(eng, pool, ctx, blocks, blocks, 5, 2)
    assert sorted(pool._free) == list(range(pages))


def test_pool_grows_by_whole_pages_and_refuses_without_taking_any():
    pool = PagedPool(cache(4, page=16))
    a, b = [], []
    pool.grow(a, 0)
    assert a == [] and pool.free_pages == 4
    pool.grow(a, 16)
    pool.grow(a, 16)
    pool.grow(b, 17)
    assert len(a) == 1 and len(b) == 2 and pool.free_pages == 1
    assert len({*a, *b}) == 3
    with pytest.raises(MemoryError):
        pool.grow(a, 49)
    assert len(a) == 1 and pool.free_pages == 1
    assert pool.table([a, [], b]).tolist() == [[a[0], 0], [0, 0], b]
    assert pool.table([]).shape == (0, 1)
    pool.release(b)
    pool.release(b)  # an empty list now
    assert b == [] and pool.free_pages == 3


def test_a_cache_of_other_tensors_is_refused():
    good = cache(3)
    for change in (dict(k=good.k[0]), dict(v=good.v[:, :2]), dict(k=good.k.view(torch.uint8), v=good.v.view(torch.uint8)),
                   dict(k_scale=good.k_scale.double()), dict(v_scale=good.v_scale[:, :2]),
                   dict(k=good.k.transpose(3, 4), v=good.v.transpose(3, 4))):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(k=good.k, v=good.v, k_scale=good.k_scale, v_scale=good.v_scale), **change})
