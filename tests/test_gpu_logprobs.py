"""fdllm_logprobs (log probabilities, entropy, top alternatives) against a 64-bit restatement."""

import math

import pytest
import torch

from _paged_util import paged_engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    return paged_engine((4, 2, 64), "float32")


def check(eng, logits, targets, top, got=None):
    lp, ent, ids, tlp = eng.logprobs(logits, targets, top=top) if got is None else got
    assert eng.device_error() == 0
    x = logits.double().cpu().reshape(-1, logits.shape[-1])
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    want_ent = -torch.where(p > 0, p * logp, torch.zeros(())).sum(-1)
    # fp32 sums of `vocab` terms in chains of at most vocab / 64 + 64 roundings, the exponential 2^-21
    # relative, the logits and log-sum-exp themselves one rounding each of their size
    n = x.shape[-1]
    chain = 2.0 ** -24 * (n / 64 + 64) + 2.0 ** -21
    size = torch.where(x.isfinite(), x.abs(), torch.zeros(())).amax(-1) + math.log(n)
    tol = chain + 2.0 ** -22 * size
    if targets is not None:
        want = logp.gather(1, targets.long().cpu()[:, None])[:, 0]
        fin = want.isfinite()
        assert torch.equal(lp.cpu().double()[~fin], want[~fin])
        assert ((lp.cpu().double() - want).abs()[fin] <= tol[fin]).all()
    else:
        assert lp is None
    # S1 / S0: both sums' errors times the mean distance from the maximum, at most the logits' span
    span = (x.amax(-1, keepdim=True) - x)
    span = (p * torch.where(p > 0, span, torch.zeros(()))).sum(-1)
    assert ((ent.cpu().double() - want_ent).abs() <= tol + 2 * chain * (span + 1)).all()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(ids.cpu().long(), order)
    want = logp.gather(1, order)
    fin = want.isfinite()
    assert torch.equal(tlp.cpu().double()[~fin], want[~fin])
    err = torch.where(fin, (tlp.cpu().double() - want).abs(), torch.zeros(()))
    assert (err <= tol[:, None]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 31, 31), (5, 1024, 20), (2, 8191, 5), (2, 8192, 32),
                                            (3, 8193, 1), (4, 32003, 20), (33, 151936, 5), (1, 151936, 32), (7, 50001, 0),
                                            (300, 1000, 8)])
def test_matches_the_definition(eng, rows, vocab, top, dtype):
    gen = torch.Generator().manual_seed(vocab + top)
    x = (torch.randn(rows, vocab, generator=gen) * 2.5).to(dtype).cuda()
    check(eng, x, torch.randint(0, vocab, (rows,), generator=gen).cuda(), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_id(eng, dtype):
    for vocab in (1000, 40000):
        x = torch.zeros(4, vocab)
        x[1] = (torch.arange(vocab) % 3).float()
        x[2] = -0.0
        x[2, ::7] = 0.0
        x[3, vocab - 40:] = 1.0
        check(eng, x.to(dtype).cuda(), torch.tensor([0, 1, 2, vocab - 1]).cuda(), 32)


@pytest.mark.parametrize("order", ["ascending", "descending", "one-spike", "sorted-blocks"])
def test_orders_and_spikes(eng, order):
    vocab = 50000
    x = torch.linspace(-20, 20, vocab)[None].repeat(2, 1)
    if order == "descending":
        x = x.flip(1)
    elif order == "one-spike":
        x = torch.full((2, vocab), -3.0)
        x[0, 12345], x[1, vocab - 1] = 80.0, 2.0
    elif order == "sorted-blocks":
        x = x.view(2, 50, 1000).flip(2).reshape(2, vocab)
    check(eng, x.contiguous().cuda(), torch.tensor([12345, vocab - 1]).cuda(), 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_banned_ids_and_lowest_values(eng, dtype):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(5, 20011, generator=gen).to(dtype)
    x[0, 100:] = -math.inf
    x[1, 1:] = -math.inf          # one id left
    x[2, ::2] = torch.finfo(dtype).min
    x[3, :20000] = -math.inf      # fewer finite ids than alternatives
    x[4] = torch.finfo(dtype).min / 2
    x[4, 7] = torch.finfo(dtype).min / 4
    check(eng, x.cuda(), torch.tensor([5, 0, 1, 3, 7]).cuda(), 20)  # row 3: a banned target


def test_rows_without_a_distribution(eng):
    x = torch.randn(4, 9000, generator=torch.Generator().manual_seed(2))
    x[0] = -math.inf
    x[1, 4000] = math.nan
    x[2, 8999] = math.inf
    lp, ent, ids, tlp = eng.logprobs(x.cuda(), torch.tensor([1, 2, 3, 4]).cuda(), top=3)
    assert lp[:3].isnan().all() and ent[:3].isnan().all() and tlp[:3].isnan().all()
    assert lp[3].isfinite() and ent[3].isfinite()
    assert ids[0].tolist() == [0, 1, 2] and int(ids[2, 0]) == 8999
    y = x[1].clone()
    y[4000] = -math.inf
    assert torch.equal(ids[1].cpu().long(), torch.sort(y, descending=True, stable=True)[1][:3])


def test_strided_rows_and_layouts(eng):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 12001, generator=gen).cuda()
    t = torch.randint(0, 11999, (6,), generator=gen).cuda()
    for view in (x[:, 1:12000], x[:, 2:], x[::2, :-2], x.t().contiguous().t()[:, :11999]):
        check(eng, view, t[:view.shape[0]], 7)
    check(eng, x[None], t, 7)  # the [1, rows, vocab] shape of get_logits
    check(eng, x[1:2].expand(4, -1), t[:4], 7)
    check(eng, x.bfloat16()[:, 1:], t, 7)
    check(eng, x, None, 4)


def test_repeats_and_another_stream(eng):
    x = (torch.randn(40, 151936, generator=torch.Generator().manual_seed(4)) * 2).bfloat16().float().cuda()
    t = torch.arange(40).cuda()
    first = eng.logprobs(x, t, top=20)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, eng.logprobs(x, t, top=20)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eng.logprobs(x, t, top=20)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_refusals(eng):
    x = torch.zeros(2, 100, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for top in (-1, 33, 101):
        with pytest.raises(ValueError):
            eng.logprobs(x, t, top=top)
    with pytest.raises(ValueError):
        eng.logprobs(x[:, :5], t, top=6)
    with pytest.raises(ValueError):
        eng.logprobs(x, t[:1])
    with pytest.raises(ValueError):
        eng.logprobs(x.half(), t)
    with pytest.raises(ValueError):
        eng.logprobs(x.cpu(), t)
    assert eng.device_error() == 0
    lp, *_ = eng.logprobs(x, torch.tensor([100, -1]).cuda())
    assert lp.isnan().all() and eng.device_error() == 4
    assert [tuple(o.shape) for o in eng.logprobs(x[:0], t[:0], top=3)] == [(0,), (0,), (0, 3), (0, 3)]
