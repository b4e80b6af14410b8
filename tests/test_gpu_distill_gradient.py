"""The gradient of a distillation where a row's largest logit lies far below zero and much of the row is masked, against its formula in
64 bits.  Bars are those of test_gpu_distill.py: they count distances from the row's largest value, wherever that lies."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import test_gpu_distill as D
from gpu_util import dev

INF = math.inf


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def members(c):
    """Which ids a row's list names."""
    m = torch.zeros(c.rows, c.vocab, dtype=torch.bool, device=dev())
    return m.scatter_(1, c.ids.long(), True)


def far_below(c, top):
    """The rows' largest logit at `top`, and of each row a part at -inf that its list does not name: a vocabulary padded by two thirds, all
    but two ids, every other run of 64, what lies behind the last whole eight."""
    z = c.logits.float()
    c.logits.copy_(z - z.amax(1, keepdim=True) + top)
    at = torch.arange(c.vocab, device=dev())
    masks = torch.stack([at >= c.vocab // 3, (at != 0) & (at != c.vocab // 2), at // 64 % 2 == 1, at >= c.vocab // 8 * 8])
    c.logits.masked_fill_(masks[torch.arange(c.rows, device=dev()) % 4] & ~members(c), -INF)
    return c


# (slices of one turn and of two in one launch, of four and of eight in three, of more than a wave looks for; a slice that is a row's last few ids)
SIZES = [(4, 300, "f32"), (5, 24581, "f32"), (5, 24581, "bf16"), (40, 100003, "bf16"), (300, 40000, "f32"), (2400, 33001, "bf16"), (4, 1100003, "f32")]


@pytest.mark.parametrize("rows, vocab, x", SIZES)
@pytest.mark.parametrize("temperature, top", [(1.0, -100.0), (0.1, -9.5)])
@pytest.mark.parametrize("teacher, rest", D.KINDS)
def test_masked_rows_far_below_zero(sampler, rows, vocab, x, temperature, top, teacher, rest):
    """A q of 0 at -inf, whatever the row's largest logit: exp(-top / T) is beyond f32 here."""
    D.check(sampler, far_below(D.Case(rows, vocab, 12, x, "f32", x, teacher, rest, temperature, weights=True), top))


@pytest.mark.parametrize("name, value", [("LILY_SAMPLER_DISTILL_LOOKS", "0"), ("LILY_SAMPLER_HANDOVER", "strict")])
@pytest.mark.parametrize("teacher, rest", D.KINDS)
def test_masked_rows_far_below_zero_by_the_other_ways(monkeypatch, name, value, teacher, rest):
    monkeypatch.setenv(name, value)
    s = LS.Sampler(0)
    for rows, vocab, x in ((5, 24581, "f32"), (300, 40000, "f32"), (2400, 33001, "bf16")):
        c = far_below(D.Case(rows, vocab, 12, x, "f32", x, teacher, rest, 1.0, weights=True), -100.0)
        D.check(s, c)
        z, want = c.logits.clone(), torch.empty_like(c.grad)
        torch.cuda.synchronize()
        s.distill(c.logits, c.ids, c.values, c.loss, grad=want, **c.lists(), **c.grads())
        s.distill(z, c.ids, c.values, c.loss, grad=z, **c.lists(), **c.grads())
        torch.cuda.synchronize()
        assert torch.equal(z, want)
    s.close()
