"""Log probabilities and entropies of confident rows: what is small has to be small, with its own sign."""

import math

import pytest
import torch

from _paged_util import paged_engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    return paged_engine((4, 2, 64), "float32")


def check(eng, x, targets, top):
    lp, ent, _, tlp = (t.double().cpu() if t is not None else t for t in eng.logprobs(x, targets, top=top))
    y = x.double().cpu()
    logp = torch.log_softmax(y, -1)
    p = logp.exp()
    want = -torch.where(p > 0, p * logp, torch.zeros((), dtype=torch.float64)).sum(-1)
    n = y.shape[-1]
    span = torch.where(p > 1e-12, y.amax(-1, keepdim=True) - y, torch.zeros((), dtype=torch.float64)).amax(-1)
    # Relative to the row's maximum S0 is 1 and the rest.  Joining threads and parts rounds it up to 18 times, by 2^-24;
    # the rest and S1 are sums of n / 256 terms a thread (their roundings independent: 4 sqrt), each term 2^-22 of the
    # exponential and its argument's rounding, 2^-23 of the distance.
    rest = 4 * math.sqrt(n / 256 + 20) * 2.0 ** -24 + 2.0 ** -22 + span * 2.0 ** -22
    tol = 20 * 2.0 ** -24 + 2 * rest * want
    assert ((ent - want).abs() <= tol).all(), ((ent - want).abs() / tol).max()
    assert (ent >= 0).all()
    for got, exact in ((lp, logp.gather(1, targets.cpu().long()[:, None])[:, 0]),
                       (tlp, torch.sort(logp, dim=-1, descending=True, stable=True)[0][:, :top])):
        # the distance from the maximum and ln S0: one rounding each
        t = tol if exact.dim() == 1 else tol[:, None]
        fin = exact.isfinite()
        assert ((got - exact).abs()[fin] <= (t + 2.0 ** -23 * exact.abs())[fin]).all()
        assert (got <= 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,rows", [(151936, 12), (151936, 600), (32003, 9), (5000, 9)])
def test_a_late_peak_over_many_small_logits(eng, vocab, rows, dtype):
    gen = torch.Generator().manual_seed(vocab + rows)
    x = torch.randn(rows, vocab, generator=gen) * 0.3
    at = torch.randint(vocab // 2, vocab, (rows,), generator=gen)
    height = 8 + 32 * torch.arange(rows) / rows  # 8 to 40 above the rest
    x[torch.arange(rows), at] = height
    x = x.to(dtype).cuda()
    check(eng, x, at.to(torch.int32).cuda(), 5)
    check(eng, x, torch.zeros(rows, dtype=torch.int32).cuda(), 5)


@pytest.mark.parametrize("gap", [0.25, 1.0, 3.0, 10.0, 39.0])
@pytest.mark.parametrize("order", ["up", "down"])
def test_two_peaks_and_a_floor(eng, gap, order):
    """A second peak `gap` below the first, before or after it in the same thread's share and elsewhere."""
    vocab, chunk = 151936, 4096
    x = torch.full((6, vocab), -30.0)
    for r, second in enumerate((7 + chunk, 7 + 5 * chunk, 8, 300, 20 * chunk, 7 + 30 * chunk)):
        first = 7
        a, b = (20.0 - gap, 20.0) if order == "up" else (20.0, 20.0 - gap)
        x[r, first], x[r, second] = a, b
    check(eng, x.cuda(), torch.full((6,), 7, dtype=torch.int32).cuda(), 3)


@pytest.mark.parametrize("order", ["ascending", "descending"])
def test_logits_in_order(eng, order):
    x = torch.linspace(-30, 30, 100000)[None].repeat(2, 1) ** 3 / 900
    if order == "descending":
        x = x.flip(1)
    check(eng, x.contiguous().cuda(), torch.tensor([0, 99999], dtype=torch.int32).cuda(), 8)


def test_one_id_left(eng):
    x = torch.full((2, 40000), -math.inf)
    x[0, 3], x[1, 39999] = 17.3, -1e30
    lp, ent, _, tlp = eng.logprobs(x.cuda(), torch.tensor([3, 39999], dtype=torch.int32).cuda(), top=1)
    assert (lp == 0).all() and (ent == 0).all() and (tlp == 0).all()
