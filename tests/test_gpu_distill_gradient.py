"""The gradient of a distillation, against its formula in 64 bits, where a row's largest logit lies far below zero and much of the row is
masked, where nothing is left outside the list, and where a list's probabilities come to more than 1.

Bars are those of test_gpu_distill.py: they count distances from the row's largest value, wherever that lies.  With S = sum p + P, 1 unless the
list has more, the gradient of the loss is
    w T (S q_v - p_v) in the list,   w T (S q_v - P q_v / Q) outside.
S is as far off as the list's sum, the sum of p times its own bar and (k + 100) u of rounding, and its product with q rounds some times more (8 u);
every bar of a q grows S-fold, and so does the loss's, to which the row's logarithm adds its own bar S times."""
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


@pytest.mark.parametrize("rows, vocab", [(4, 300), (5, 24581), (300, 40000), (4, 1100003)])
@pytest.mark.parametrize("teacher, rest", D.KINDS)
def test_a_value_that_is_no_number_where_nothing_is_left_outside_the_list(sampler, rows, vocab, teacher, rest):
    """It makes the row's loss and whole gradient a NaN there too, and no other row's."""
    c = D.Case(rows, vocab, 12, "f32", "f32", "f32", teacher, rest, 1.0)
    c.logits[:2].masked_fill_(~members(c)[:2], -INF)
    c.values[0, 3] = float("nan")
    c.outputs()
    again = torch.empty_like(c.grad)
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.grad, **c.lists(), **c.grads())
    sampler.distill_backward(c.logits, c.ids, c.values, stats=c.stats, grad=again, **c.lists(), **c.grads())
    sampler.synchronize()
    assert bool(torch.isnan(c.loss[0])) and bool(torch.isfinite(c.loss[2:]).all())
    for grad in (c.grad, again):
        assert bool(torch.isnan(grad[0]).all()) and bool(torch.isfinite(grad[1:]).all())


class Heavy(D.Case):
    """Lists whose probabilities, with the rest as one outcome, come to what `bring` says; the gradient without S taken from D.Case."""

    def bring(self, masses):
        masses = torch.tensor(masses, device=dev(), dtype=torch.float64)[torch.arange(self.rows, device=dev()) % len(masses)]
        if self.teacher == "probs":
            self.values.copy_(self.values.double() * (masses / self.values.double().sum(1))[:, None])
        else:
            self.lse = (torch.logsumexp(self.values.double() / self.T, 1) - torch.log(masses)).float()
        return self

    def p(self):
        v = self.values.double()
        return v if self.teacher == "probs" else torch.exp(v / self.T - self.lse.double()[:, None])

    def formula(self):
        out, self.out = self.out, "f32"
        loss, loss_tol, stats, stats_tol, grad, tol = super().formula()
        self.out = out
        p, q = self.p(), torch.softmax(self.logits.double() / self.T, 1)
        mass = p.sum(1, keepdim=True)
        total = mass.clamp_min(1.0)
        off = (130 if self.teacher == "probs" else 4) * D.U * mass + (self.k + 100) * D.U
        w = self.T * self.scale * (self.weights.double()[:, None] if self.weights is not None else torch.ones_like(mass))
        grad, tol = grad + w * (total - 1.0) * q, total * tol + w.abs() * q * (off + 8 * D.U * total)
        if out == "bf16":
            tol = tol + 2.0 ** -8 * (grad.abs() + tol)
        return loss, total[:, 0] * loss_tol, stats, stats_tol, grad, tol


MASSES = [0.4, 1.03, 1.0, 1.5, 1.0 + 2.0 ** -20, 4.0]


@pytest.mark.parametrize("rows, vocab, k, x, out", [(6, 300, 7, "f32", "f32"), (6, 24581, 40, "bf16", "bf16"), (9, 100003, 64, "f32", "f32"),
                                                    (300, 40000, 300, "f32", "bf16"), (2400, 33001, 20, "bf16", "f32"), (6, 1100003, 64, "f32", "f32"),
                                                    (6, 40, 40, "f32", "f32")])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
@pytest.mark.parametrize("teacher", ["logits", "probs"])
def test_a_list_of_more_than_all(sampler, rows, vocab, k, x, out, t, temperature, teacher):
    """P is 0 there, and the row's softmax is held to all that the list has."""
    c = Heavy(rows, vocab, k, x, t, out, teacher, True, temperature, weights=True).bring(MASSES)
    c.ids[1, 1] = c.ids[1, 0]
    D.check(sampler, c)
    # a row adds up to S - sum p - P, which is 0 (where no id is outside the list nobody has the - P: it adds up to P)
    *_, tol = c.formula()
    left = torch.where(members(c).all(1), (1.0 - c.p().sum(1)).clamp_min(0.0), 0.0) * c.T * c.scale * c.weights.double()
    assert bool(((c.grad.double().sum(1) - left).abs() <= tol.sum(1)).all())


@pytest.mark.parametrize("name, value", [("LILY_SAMPLER_DISTILL_LOOKS", "0"), ("LILY_SAMPLER_HANDOVER", "strict")])
@pytest.mark.parametrize("teacher", ["logits", "probs"])
def test_a_list_of_more_than_all_by_the_other_ways(monkeypatch, name, value, teacher):
    monkeypatch.setenv(name, value)
    s = LS.Sampler(0)
    for rows, vocab, x in ((6, 24581, "f32"), (300, 40000, "f32"), (2400, 33001, "bf16")):
        D.check(s, Heavy(rows, vocab, 30, x, "f32", x, teacher, True, 1.0, weights=True).bring(MASSES))
    s.close()


@pytest.mark.parametrize("teacher", ["logits", "probs"])
def test_lists_that_rounding_brings_beyond_all(sampler, teacher):
    """Teacher logits of some 20, rounded to bf16 (by up to 2^-4), against the sum over the row as it was; probabilities rounded to bf16 of a list that
    holds the whole vocabulary."""
    g = torch.Generator(device=dev()).manual_seed(8)
    rows, vocab, k = (64, 9000, 20) if teacher == "logits" else (64, 12, 12)
    c = Heavy(rows, vocab, k, "f32", "bf16", "f32", teacher, True, 1.0)
    t = 18.0 + 4.0 * torch.rand(rows, k, generator=g, device=dev())
    if teacher == "logits":
        c.values.copy_(t)
        c.lse = (torch.logsumexp(t.double(), 1) + 1e-3).float()
    else:
        c.values.copy_(torch.softmax(t, 1))
    masses = c.p().sum(1)
    assert bool((masses > 1.0 + (0.01 if teacher == "logits" else 0.0005)).any()) and bool((masses < 1.0).any())
    D.check(sampler, c)


@pytest.mark.parametrize("temperature", [2.0 ** -100, 1e-6, 1e6])
@pytest.mark.parametrize("rows", [3, 900])
def test_lists_that_a_small_temperature_brings_beyond_all(sampler, rows, temperature):
    """The teacher's sum in f32: at T = 1e-6 it lies at some 5e6 and is rounded by up to 1 / 4."""
    c = Heavy(rows, 9001, 40, "f32", "f32", "f32", "logits", True, temperature, weights=True)
    D.check(sampler, c)
    assert temperature != 1e-6 or rows == 3 or bool((c.p().sum(1) > 1.0).any())


@pytest.mark.parametrize("teacher", ["logits", "probs"])
def test_the_gradient_is_the_loss_differentiated_there_too(sampler, teacher):
    """Central differences of the loss in 64 bits: their own error is some step^2 = 1e-10 and 1e-15 / step = 1e-10."""
    c = Heavy(4, 60, 7, "f32", "f32", "f32", teacher, True, 1.7, spread=1.0, weights=True).bring([1.03, 2.0, 0.7, 1.3])
    c.ids[1, 2] = c.ids[1, 5]
    c.outputs()
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, grad=c.grad, **c.lists(), **c.grads())
    sampler.synchronize()
    keep, step = c.logits, 1e-5
    want = torch.empty(4, 60, dtype=torch.float64, device=dev())
    for v in range(60):
        sides = []
        for e in (step, -step):
            c.logits = keep.double()
            c.logits[:, v] += e
            sides.append(c.formula()[0])
        want[:, v] = (sides[0] - sides[1]) / (2 * step)
    c.logits = keep
    want *= c.scale * c.weights.double()[:, None]
    assert float((c.grad.double() - want).abs().max()) <= c.formula()[5].max() + 1e-8
