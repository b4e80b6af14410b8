"""Distillation from a teacher's lists (lily_distill, lily_distill_backward) against its formulas in 64 bits.

Bars (u = 2^-24), a = (z - z0) / T a value's distance from its row's largest, q = softmax:
  * an exponential: its argument's difference and product with log2(e) / T round three times (3 u |a|), the exponential 2 u;
    values meet their row's reference in two steps whose distances add up to |a|;
  * a sum of them: sum q (3 |a| + 6) u, and up to 65 additions in a thread, 8 in its wave, 8 of waves and 8 of slices: (3 E + 100) u
    relative, E = sum q |a|;
    a stored logarithm rounds u |log sum| more, and what is formed of it so much again: (3 E + 140) u in all, call it s;
  * q: (3 |a| + 8) u + s relative; r, the same outside the list; a probability of the list: (3 |t - t0| / T + 140) u + its own
    sum's (3 E_t + 140) u, or from the teacher's sum one exponential of an argument in 64 bits, 4 u (a probability given as such: 130 u with
    its sum).  P = 1 - sum p is as far off as all of them and their sum (k + 100) u;
  * the gradient: each of q sum(p), p and P r times its own, and 8 u of them; bf16 2^-8 of the result;
  * the loss, formed in 64 bits of these: T^2 (sum p rel(p) (|log p - log q| + 1) + s + rel(list's sum) + dP (|log(P / Q)| + 1) + P (s + s_rest))
    + u |loss|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
INF = math.inf


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def rows_of(t, pad, start=0):
    """The values as rows of a wider buffer whose other elements hold NaN, starting at element `start`."""
    rows, n = t.shape
    fill = float("nan") if t.is_floating_point() else 12345
    buf = torch.full((rows * (n + pad) + start + 8,), fill, dtype=t.dtype, device=t.device)
    m = torch.as_strided(buf, (rows, n), (n + pad, 1), start)
    m.copy_(t)
    return buf, m


class Case:
    def __init__(self, rows, vocab, k, x="f32", t="f32", out="f32", teacher="logits", rest=False, temperature=1.0, counts=None, pad=0, start=0,
                 weights=False, seed=0, spread=3.0):
        g = torch.Generator(device=dev()).manual_seed(rows * 17 + vocab + k + seed)
        temperature = float(torch.tensor(temperature, dtype=torch.float32))   # what the call is given: 1e-6 is 2.5e-9 of itself off, of z / T some hundredths
        self.rows, self.vocab, self.k, self.T, self.teacher, self.rest = rows, vocab, k, temperature, teacher, rest
        self.pad, self.start, self.out = pad, start, out
        z = spread * torch.randn(rows, vocab, generator=g, device=dev())
        ids = torch.rand(rows, vocab, generator=g, device=dev()).topk(min(k, vocab), 1).indices
        if k > vocab:
            ids = torch.nn.functional.pad(ids, (0, k - vocab), value=-1)
        t_ = 2.0 * torch.randn(rows, k, generator=g, device=dev())
        z.scatter_add_(1, ids.clamp_min(0), torch.where(ids >= 0, 4.0, 0.0))
        share = 0.05 + 0.9 * torch.rand(rows, generator=g, device=dev())      # of the teacher's mass, in its list
        if teacher == "probs":
            t_ = torch.softmax(t_.masked_fill(ids < 0, -INF), 1) * (share[:, None] if rest else 3.0)
        self.values = rows_of(t_.to(DT[t]), pad, start)[1]
        self.logits = rows_of(z.to(DT[x]), pad, start)[1]
        self.ids = rows_of(ids.to(torch.int32), pad, start)[1]
        self.counts = None if counts is None else torch.tensor([counts(r) for r in range(rows)], dtype=torch.int32, device=dev())
        self.weights = torch.rand(rows, generator=g, device=dev()) + 0.5 if weights else None
        self.scale = 0.37 if weights else 1.0
        self.lse = None
        if teacher == "logits" and rest:
            on = torch.where(self.ids >= 0, self.values.double() / temperature, -INF)
            self.lse = (torch.logsumexp(on, 1) - torch.log(share.double())).float()

    def outputs(self):
        self.loss, self.stats = torch.full((self.rows,), 9.0, device=dev()), torch.full((self.rows, 4), 9.0, device=dev())
        self.buf, self.grad = rows_of(torch.zeros(self.rows, self.vocab, dtype=DT[self.out], device=dev()), self.pad, self.start)
        self.before = self.buf.clone()

    def lists(self):
        return dict(temperature=self.T, teacher=self.teacher, rest=self.rest, teacher_lse=self.lse, counts=self.counts)

    def grads(self):
        return dict(row_weights=self.weights, grad_scale=self.scale)

    def formula(self):
        """(loss, its bar, stats, their bars, gradient, its bar)."""
        T, rows, vocab, k = self.T, self.rows, self.vocab, self.k
        z = self.logits.double() / T
        ids = self.ids.long() & 0xffffffff
        on = ids < vocab
        if self.counts is not None:
            on &= torch.arange(k, device=dev())[None, :] < (self.counts.long() & 0xffffffff)[:, None]
        ids = torch.where(on, ids, 0)
        t = self.values.double()
        if self.teacher == "logits":
            t = torch.where(on, t / T, torch.full_like(t, -INF))
            top = t.amax(1, keepdim=True)
            if self.rest:
                logp = t - self.lse.double()[:, None]
                rel, listed = torch.full_like(t, 4 * U), torch.zeros(rows, 1, device=dev(), dtype=torch.float64)
            else:
                logp = t - torch.logsumexp(t, 1, keepdim=True)
                e_t = (torch.exp(logp) * (top - t)).nan_to_num(0.0).sum(1, keepdim=True)
                listed = (3 * e_t + 140) * U
                rel = (3 * (top - t).nan_to_num(0.0, posinf=0.0) + 140) * U + listed
        else:
            t = torch.where(on, t.clamp_min(0.0), torch.zeros_like(t))
            logp = torch.log(t if self.rest else t / t.sum(1, keepdim=True))
            rel, listed = torch.full_like(t, 130 * U), torch.full((rows, 1), 130 * U, device=dev(), dtype=torch.float64)
        p = torch.where(on, torch.exp(logp), torch.zeros_like(t)).nan_to_num(0.0)
        live = on.any(1) if self.rest else p.sum(1) > 0
        P = (1.0 - p.sum(1, keepdim=True)).clamp_min(0.0) if self.rest else torch.zeros(rows, 1, device=dev(), dtype=torch.float64)
        dP = (p * rel).sum(1, keepdim=True) + (k + 100) * U if self.rest else 0.0 * P

        def whole(v):
            v0 = v.amax(1, keepdim=True)
            logs = torch.logsumexp(v, 1, keepdim=True)
            a = v0 - v
            e = (torch.exp(v - logs) * a).nan_to_num(0.0).sum(1, keepdim=True)
            return v0, logs - v0, torch.exp(v - logs), a, (3 * e + 140) * U + 2 * U * (logs - v0).abs()

        z0, ls, q, a, s = whole(z)
        member = torch.zeros(rows, vocab + 1, dtype=torch.bool, device=dev())
        member.scatter_(1, torch.where(on, ids, vocab), True)
        member = member[:, :vocab]
        dense = torch.zeros_like(z).scatter_add_(1, ids, p)
        dense_err = torch.zeros_like(z).scatter_add_(1, ids, p * (rel + 8 * U))
        q_err = q * ((3 * a.nan_to_num(0.0, posinf=0.0) + 16) * U + s)
        logq = (z - z0 - ls).gather(1, ids)
        mine = torch.where(p > 0, logp - logq, torch.zeros_like(p))
        loss = (p * mine).sum(1)
        loss_tol = (p * rel * (mine.abs() + 1)).sum(1) + s[:, 0] + listed[:, 0]
        raw = self.logits.double()              # (a quotient times T is not the value again)
        stats = torch.cat([raw.amax(1, keepdim=True), ls, 0 * ls, 0 * ls], 1)
        stats_tol = torch.cat([0 * s, s, 0 * s, 0 * s], 1)
        if self.rest:
            zr = z.masked_fill(member, -INF)
            some = (~member & (z > -INF)).any(1, keepdim=True)
            r0, rs, r, ar, sr = whole(torch.where(some, zr, torch.zeros_like(zr)))
            logQ = torch.where(some, r0 + rs - z0 - ls, -INF)   # (where exp(logQ) is below what 64 bits hold, log of it is not it)
            r, Q = torch.where(some, r, 0.0), torch.exp(logQ)
            term = torch.where(P > 0, P * (torch.log(P) - logQ), 0.0 * P)
            loss = loss + term[:, 0]
            gap = torch.where((P > 0) & some, (torch.log(P) - logQ).abs(), 0.0 * P)
            loss_tol = loss_tol + (dP * (gap + 1) + P * (s + sr))[:, 0]
            stats[:, 2:] = torch.where(some, torch.cat([raw.masked_fill(member, -INF).amax(1, keepdim=True), rs], 1), torch.tensor([-INF, 0.0], device=dev(), dtype=torch.float64))
            stats_tol[:, 3:] = torch.where(some, sr, 0.0)
            grad = torch.where(member, q - dense, q - P * r)
            r_err = torch.where(some, r * ((3 * ar.nan_to_num(0.0, posinf=0.0) + 16) * U + sr), 0.0)
            # (formed as r (Q - P): Q as far off as both sums, and by the distance of the two largest values)
            Q_err = Q * (s + sr + (3 * (z0 - r0).abs() + 16) * U)
            grad_tol = torch.where(member, q_err + dense_err, (Q + P) * r_err + r * (Q_err + dP))
        else:
            total = p.sum(1, keepdim=True)
            grad, grad_tol = q * total - dense, q_err + 140 * U * q + dense_err
        w = T * self.scale * (self.weights.double()[:, None] if self.weights is not None else torch.ones(rows, 1, device=dev(), dtype=torch.float64))
        w = torch.where(live[:, None], w, 0.0 * w)
        grad, grad_tol = w * grad, w.abs() * grad_tol + 4 * U * (w * grad).abs()
        if self.out == "bf16":
            grad_tol = grad_tol + 2.0 ** -8 * (grad.abs() + grad_tol)
        loss = torch.where(live, T * T * loss, 0.0 * z0[:, 0])
        return loss, T * T * loss_tol + U * loss.abs(), stats, stats_tol, grad, grad_tol


def near(got, want, tol):
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine])
    # (a value whose bar reaches beyond f32's largest, 2^128 (1 - 2^-24), by half a step or more may have been rounded to infinity:
    # a loss of p times 3.4028235e38, the p off by 1e-7 of themselves)
    over = fine & (got == INF) & (want + tol >= 2.0 ** 128 * (1.0 - 2.0 ** -25))
    fine = fine & ~over
    err = (got - want)[fine].abs()
    assert bool((err <= tol[fine] + 2.0 ** -125).all()), float((err - tol[fine]).max())


def check(sampler, c, loss_only=True):
    c.outputs()
    want = c.formula()
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.grad, **c.lists(), **c.grads())
    sampler.synchronize()
    near(c.loss, want[0], want[1])
    near(c.stats, want[2], want[3])
    near(c.grad, want[4], want[5])
    mask = torch.ones_like(c.buf, dtype=torch.bool)
    torch.as_strided(mask, (c.rows, c.vocab), (c.vocab + c.pad, 1), c.start).fill_(False)
    bits = torch.int16 if c.out == "bf16" else torch.int32
    assert torch.equal(c.buf.view(bits)[mask], c.before.view(bits)[mask])
    if not loss_only:
        return
    # the gradient from the stats, and the loss alone
    again = torch.full_like(c.grad, 5.0)
    sampler.distill_backward(c.logits, c.ids, c.values, stats=c.stats, grad=again, **c.lists(), **c.grads())
    loss, stats = torch.full_like(c.loss, 5.0), torch.full_like(c.stats, 5.0)
    sampler.distill(c.logits, c.ids, c.values, loss, stats=stats, **c.lists())
    sampler.synchronize()
    near(again, want[4], want[5])
    near(loss, want[0], want[1])
    near(stats, want[2], want[3])


KINDS = [("logits", False), ("logits", True), ("probs", False), ("probs", True)]


@pytest.mark.parametrize("rows, vocab, k", [(1, 1, 1), (2, 7, 3), (1, 8, 8), (3, 64, 5), (5, 1000, 20), (2, 8191, 64), (2, 8192, 1), (2, 8193, 300),
                                            (9, 16385, 64), (3, 30011, 1024), (1, 151936, 20), (4, 248320, 64), (2, 100, 130)])
@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("x, t, out, pad, start", [("f32", "f32", "f32", 0, 0), ("bf16", "bf16", "bf16", 8, 8), ("bf16", "f32", "f32", 3, 1),
                                                   ("f32", "bf16", "bf16", 5, 3)])
def test_against_the_formula(sampler, rows, vocab, k, teacher, rest, x, t, out, pad, start):
    check(sampler, Case(rows, vocab, k, x, t, out, teacher, rest, 1.0, None, pad, start, weights=pad != 0))


@pytest.mark.parametrize("temperature", [0.1, 0.7, 2.0, 20.0])
@pytest.mark.parametrize("teacher, rest", KINDS)
def test_temperatures(sampler, temperature, teacher, rest):
    check(sampler, Case(6, 20000, 50, "f32", "f32", "f32", teacher, rest, temperature))
    check(sampler, Case(6, 20000, 50, "bf16", "bf16", "bf16", teacher, rest, temperature))


@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("rows, vocab", [(600, 5000), (300, 40000), (2100, 130), (257, 70001), (260, 153607), (256, 248320)])
def test_many_rows(sampler, teacher, rest, rows, vocab):
    check(sampler, Case(rows, vocab, 40, "bf16", "f32", "bf16", teacher, rest, 1.5, lambda r: r % 45, weights=True))


@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("rows", [40, 280])
def test_lists_of_every_length(sampler, teacher, rest, rows):
    """Counts from none to more than there is room for, and ids that pad."""
    c = Case(rows, 9000, 33, "f32", "f32", "f32", teacher, rest, 1.0, lambda r: r if r < 39 else -1)
    c.ids[:, 5] = -1
    c.ids[:, 6] = 9000            # the first id beyond the vocabulary
    c.ids[::3, 7:] = -1
    check(sampler, c)
    assert float(c.loss[0]) == 0.0 and bool((c.grad[0] == 0).all())


@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("k", [4, 70, 1000])
@pytest.mark.parametrize("rows", [8, 300])
def test_an_id_that_stands_there_twice(sampler, teacher, rest, k, rows):
    c = Case(rows, 20000, k, "f32", "f32", "f32", teacher, rest, 1.0)
    c.ids[0, :] = 17                           # every entry the same id
    c.ids[1, 1] = c.ids[1, 0]
    c.ids[2, k - 1] = c.ids[2, 0]
    c.ids[3, : k // 2] = c.ids[3, k // 2: 2 * (k // 2)].clone()
    c.ids[4, ::3] = 8191
    c.ids[4, 1::3] = 8192
    check(sampler, c)


@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("rows", [6, 260])
def test_masked_logits(sampler, teacher, rest, rows):
    """-inf in the student's rows, outside its list, in it where the teacher has nothing and where it has something."""
    c = Case(rows, 12000, 16, "f32", "f32", "f32", teacher, rest, 1.0)
    none = -INF if teacher == "logits" else 0.0
    outside = torch.ones(12000, dtype=torch.bool, device=dev())
    outside[c.ids[0].long()] = False
    c.logits[0, outside] = -INF                # nothing is left outside the list
    c.logits[1, ::2] = -INF                    # half the row, parts of the list among it
    c.logits[2, 4000:] = -INF
    c.values[2, :] = torch.where(c.ids[2] >= 4000, torch.tensor(none, device=dev()), c.values[2])
    c.logits[3, c.ids[3, 3].long()] = -INF     # an infinite loss
    c.logits[4, :] = torch.finfo(torch.float32).min
    c.logits[4, 77] = 1.0
    check(sampler, c)
    assert float(c.loss[3]) == INF and bool(torch.isfinite(c.grad[3]).all())


@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("rows, vocab", [(9, 300), (9, 20000), (270, 60000), (270, 200000)])
def test_what_is_not_finite(sampler, teacher, rest, rows, vocab):
    """NaN, +inf and rows of -inf make their row a NaN and no other; rows without an entry that counts or without weight stay zeros."""
    c = Case(rows, vocab, 8, "f32", "f32", "f32", teacher, rest, 1.0, lambda r: 0 if r in (6, 7) else 8, weights=True)
    free = next(i for i in range(vocab) if i not in set(c.ids[0].tolist()))
    c.logits[0, free] = float("nan")
    c.logits[1, c.ids[1, 2].long()] = float("nan")
    c.logits[2, vocab // 2] = INF
    c.logits[3, :] = -INF
    c.values[4, 1] = float("nan")
    c.logits[6, 3] = float("nan")              # no entry counts
    c.logits[8, :] = float("nan")
    c.weights[8] = 0.0
    c.weights[7] = 0.0
    c.outputs()
    again = torch.full_like(c.grad, 5.0)
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.grad, **c.lists(), **c.grads())
    sampler.distill_backward(c.logits, c.ids, c.values, stats=c.stats, grad=again, **c.lists(), **c.grads())
    sampler.synchronize()
    for grad in (c.grad, again):
        assert bool(torch.isnan(grad[:5]).all()), [bool(torch.isnan(grad[r]).all()) for r in range(5)]
        assert bool(torch.isfinite(grad[5]).all()) and bool((grad[6:9] == 0).all()) and bool(torch.isfinite(grad[9:]).all())
    assert bool(torch.isnan(c.loss[:5]).all()) and bool(torch.isfinite(c.loss[5])) and bool((c.loss[6:8] == 0).all())
    assert bool(torch.isfinite(c.loss[9:]).all())


def test_a_list_without_mass(sampler):
    """Without `rest` a list of zeros or of -inf is none."""
    for teacher, none in (("probs", 0.0), ("probs", -1.0), ("logits", -INF)):
        c = Case(3, 500, 4, teacher=teacher)
        c.values[1, :] = none
        check(sampler, c)
        assert float(c.loss[1]) == 0.0 and bool((c.grad[1] == 0).all())


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab, k", [(3, 20000, 50), (700, 3001, 17), (2, 200, 190), (300, 50001, 60)])
@pytest.mark.parametrize("teacher, rest", KINDS)
def test_in_place(sampler, x, rows, vocab, k, teacher, rest):
    c = Case(rows, vocab, k, x, "f32", x, teacher, rest, 1.0)
    c.outputs()
    want = c.formula()
    torch.cuda.synchronize()
    keep = c.logits.clone()
    sampler.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.logits, **c.lists(), **c.grads())
    sampler.synchronize()
    near(c.loss, want[0], want[1])
    near(c.logits, want[4], want[5])
    first = c.logits.clone()
    c.logits.copy_(keep)
    torch.cuda.synchronize()
    sampler.distill_backward(c.logits, c.ids, c.values, stats=c.stats, grad=c.logits, **c.lists(), **c.grads())
    sampler.synchronize()
    near(c.logits, want[4], want[5])
    c.logits.copy_(keep)
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.logits, **c.lists(), **c.grads())
    sampler.synchronize()
    assert torch.equal(first, c.logits)        # the same bits again


@pytest.mark.parametrize("teacher, rest", KINDS)
def test_the_gradient_is_the_loss_differentiated(sampler, teacher, rest):
    """Central differences of the loss in 64 bits: their own error is some step^2 = 1e-10 and 1e-15 / step = 1e-10."""
    c = Case(2, 60, 7, "f32", "f32", "f32", teacher, rest, 1.7, spread=1.0, weights=True)
    c.ids[1, 2] = c.ids[1, 5]
    c.outputs()
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, grad=c.grad, **c.lists(), **c.grads())
    sampler.synchronize()
    keep, step = c.logits, 1e-5
    want = torch.empty(2, 60, dtype=torch.float64, device=dev())
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


def test_more_rows_than_the_workspace_holds(sampler):
    """Lists of 1 024 logits each: some 8 000 rows fill the workspace."""
    check(sampler, Case(9000, 300, 1024, "bf16", "bf16", "bf16", "logits", True, 1.0, lambda r: (r * 7) % 300))


def test_rows_that_lie_further_apart_than_32_bits(sampler):
    c = Case(3, 9000, 20, "bf16", "f32", "bf16", "logits", True, 1.0)
    far = (1 << 31) + 24
    for name in ("logits", "grad"):
        wide = torch.as_strided(torch.empty(2 * far + 9000, dtype=torch.bfloat16, device=dev()), (3, 9000), (far, 1))
        if name == "logits":
            wide.copy_(c.logits)
            c.logits = wide
    c.outputs()
    want = c.formula()
    torch.cuda.synchronize()
    sampler.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=wide, **c.lists())
    sampler.synchronize()
    near(c.loss, want[0], want[1])
    near(wide, want[4], want[5])
    wide.zero_()
    torch.cuda.synchronize()
    sampler.distill_backward(c.logits, c.ids, c.values, stats=c.stats, grad=wide, **c.lists())
    sampler.synchronize()
    near(wide, want[4], want[5])


@pytest.mark.parametrize("rows, vocab", [(3, 30000), (400, 3000), (300, 9000)])
def test_a_captured_graph(rows, vocab):
    stream = torch.cuda.Stream()
    s = LS.Sampler(0, stream)
    c = Case(rows, vocab, 20, "bf16", "f32", "bf16", "logits", True, 1.0, weights=True)
    c.outputs()
    g = torch.Generator(device=dev()).manual_seed(4)

    def step():
        s.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.grad, **c.lists(), **c.grads())

    torch.cuda.synchronize()
    step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for turn in range(4):
        c.logits.copy_(torch.randn(rows, vocab, generator=g, device=dev()) * (turn + 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = c.loss.clone(), c.grad.clone()
        c.loss.zero_(), c.grad.zero_()
        torch.cuda.synchronize()
        step()
        s.synchronize()
        assert torch.equal(replayed[0], c.loss) and torch.equal(replayed[1], c.grad)
        want = c.formula()
        near(c.loss, want[0], want[1])
        near(c.grad, want[4], want[5])
    s.close()


def test_what_the_python_mirror_refuses(sampler):
    c = Case(2, 100, 5)
    c.outputs()
    good = dict(logits=c.logits, ids=c.ids, values=c.values, loss=c.loss, stats=c.stats, grad=c.grad)
    row = torch.zeros(2, device=dev())
    for bad in (dict(logits=c.logits.half()), dict(logits=c.logits[:, ::2]), dict(ids=c.ids.long()), dict(ids=c.ids[:, :4]), dict(values=c.values[:1]),
                dict(loss=row[:1]), dict(loss=row.double()), dict(stats=c.stats[:, :3]), dict(grad=c.grad[:, :50]), dict(teacher="ids"),
                dict(temperature=0.0), dict(temperature=INF), dict(rest=True), dict(teacher_lse=row), dict(teacher="probs", rest=True, teacher_lse=row),
                dict(counts=row), dict(row_weights=row[:1]), dict(grad_scale=float("nan")), dict(grad=c.logits[:, :100].bfloat16()[:, ::1].t()),
                dict(loss=None, stats=None, grad=None)):
        with pytest.raises(LS.SamplerError):
            sampler.distill(**{**good, **bad})
    good.pop("loss")
    for bad in (dict(stats=None), dict(grad=None)):
        with pytest.raises(LS.SamplerError):
            sampler.distill_backward(**{**good, **bad})


@pytest.mark.parametrize("looks", [0, 1, 3])
@pytest.mark.parametrize("teacher, rest", KINDS)
def test_slices_whose_neighbours_are_not_seen(monkeypatch, looks, teacher, rest):
    """A workgroup that does not find its row's other sums forms them itself: by the same operations, so the bits are the same."""
    monkeypatch.setenv("LILY_SAMPLER_DISTILL_LOOKS", str(looks))
    s, usual = LS.Sampler(0), None
    for rows, vocab, k, x in ((3, 40003, 30, "f32"), (200, 33001, 60, "bf16"), (2, 100000, 1000, "bf16"), (150, 70001, 5, "f32"), (2400, 33001, 20, "bf16")):
        c = Case(rows, vocab, k, x, "f32", x, teacher, rest, 1.0, weights=True)
        c.ids[1, 1] = c.ids[1, 0]
        c.logits[0, ::3] = -INF
        check(s, c)
        monkeypatch.delenv("LILY_SAMPLER_DISTILL_LOOKS", raising=False)
        usual = usual or LS.Sampler(0)
        loss, grad, stats = torch.empty_like(c.loss), torch.empty_like(c.grad), torch.empty_like(c.stats)
        torch.cuda.synchronize()
        s.distill(c.logits, c.ids, c.values, c.loss, stats=c.stats, grad=c.grad, **c.lists(), **c.grads())
        usual.distill(c.logits, c.ids, c.values, loss, stats=stats, grad=grad, **c.lists(), **c.grads())
        torch.cuda.synchronize()
        assert torch.equal(loss, c.loss) and torch.equal(stats, c.stats) and torch.equal(grad, c.grad)
    s.close()
    usual.close()


@pytest.mark.parametrize("looks", [0, 2, 4096])
@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 30])
def test_in_place_whether_neighbours_are_seen_or_not(monkeypatch, looks, x, rows):
    """A workgroup that adds up a neighbour's slice itself takes no gradient for a logit; what a call leaves is what the next one finds."""
    monkeypatch.setenv("LILY_SAMPLER_DISTILL_LOOKS", str(looks))
    s = LS.Sampler(0)
    c = Case(rows, 100003, 40, x, "f32", x, "logits", True, 1.0, weights=True)
    kept = c.logits.clone()
    check(s, c)
    first = c.grad.clone(), c.loss.clone()
    for _ in range(20):
        z, loss = kept.clone(), torch.empty_like(c.loss)
        torch.cuda.synchronize()
        s.distill(z, c.ids, c.values, loss, grad=z, **c.lists(), **c.grads())
        torch.cuda.synchronize()
        assert torch.equal(z, first[0]) and torch.equal(loss, first[1])
        s.distill(kept, c.ids, c.values, loss, **c.lists())      # the loss alone, the same way
        torch.cuda.synchronize()
        assert torch.equal(loss, first[1])
    s.close()


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("teacher, rest", KINDS)
def test_lists_of_one_id_and_of_pairs(sampler, rows, teacher, rest):
    """The first entry of an id speaks for all of them: lists that name one id throughout, and every id twice, apart and side by side."""
    c = Case(rows, 30011, 1000, "bf16", "f32", "f32", teacher, rest, 1.0, weights=True)
    c.ids[0] = 17
    c.ids[1, 500:] = c.ids[1, :500]
    c.ids[2, 1::2] = c.ids[2, ::2]
    if teacher == "probs":
        c.values.mul_(0.9 / c.values.sum(1, keepdim=True))
    check(sampler, c)


@pytest.mark.parametrize("looks", ["4096", "0"])
@pytest.mark.parametrize("teacher, rest", KINDS)
def test_few_rows_by_three_launches(monkeypatch, looks, teacher, rest):
    """LILY_SAMPLER_HANDOVER=strict: sums that pass between launches, or as whole words."""
    monkeypatch.setenv("LILY_SAMPLER_HANDOVER", "strict")
    monkeypatch.setenv("LILY_SAMPLER_DISTILL_LOOKS", looks)
    s = LS.Sampler(0)
    for rows, vocab, k, x in ((3, 40003, 30, "f32"), (2, 100000, 1000, "bf16"), (30, 7, 3, "f32")):
        c = Case(rows, vocab, k, x, "f32", x, teacher, rest, 1.0, weights=True)
        check(s, c)
        want = c.grad.clone()
        z = c.logits.clone()
        torch.cuda.synchronize()
        s.distill(z, c.ids, c.values, c.loss, grad=z, **c.lists(), **c.grads())
        s.synchronize()
        assert torch.equal(z, want)
    s.close()


@pytest.mark.parametrize("rows, vocab, x", [(2, 1 << 24, "bf16"), (3, 1100003, "f32"), (1, 2097160, "bf16")])
def test_vocabularies_of_more_slices_than_a_wave_looks_for(sampler, rows, vocab, x):
    check(sampler, Case(rows, vocab, 64, x, "f32", x, "logits", True, 1.0, weights=True))


@pytest.mark.parametrize("temperature", [2.0 ** -100, 1e-6, 1e6])
@pytest.mark.parametrize("teacher, rest", KINDS)
@pytest.mark.parametrize("rows", [3, 900])
def test_temperatures_that_leave_one_outcome_or_all_alike(sampler, temperature, teacher, rest, rows):
    check(sampler, Case(rows, 9001, 40, "f32", "f32", "f32", teacher, rest, temperature, weights=True))
