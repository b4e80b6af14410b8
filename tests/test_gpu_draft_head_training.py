"""A draft head trained and served, by the operators one after the other: the norm, the head's product, the distillation from a target
model's lists, the gradient back through the head and the norm; and its way to a token through 8-bit blocks.  Every stage is held to its
formula in 64 bits on what the stage before left (bars as for each alone), and the gradient at the head's input to the formula of them all.

The gradient through everything, as lengths (s the head's largest singular value, |.| a row's length, T = 1, a row's weight 1): the normed
row rounds 2^-8 of itself, which moves its logits by s |y| 2^-8 (their own f32 sums 2^-12 of |y| s more at most); a softmax's Jacobian is
no longer than 1/2; the gradient at the logits rounds 2^-8, and so does the one at the normed row; the norm's backward pass lengthens
nothing by more than rstd max|w|.  Together
    |dx| <= rstd max|w| (s (s |y| 2^-8 1.1 / 2 + 2^-8 |g|) + 2^-8 1.1 |dy|) + 2^-8 1.1 |gx|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import test_gpu_blocks as B
import test_gpu_distill as D
import test_gpu_layer_norm as L
import test_gpu_project as P
from gpu_util import dev, ls_params

EPS = 1e-5
BF16 = torch.bfloat16


class Training:
    """A step's resident buffers.  The target's logits are drawn from (the draws leave its lists) before the student learns from them."""

    def __init__(self, stream, seed, rows, d, vocab, rest):
        self.s = LS.Sampler(0, stream)
        self.rows, self.d, self.vocab, self.rest, self.k = rows, d, vocab, rest, 50
        self.g = torch.Generator(device=dev()).manual_seed(seed)
        normal = lambda *shape: torch.randn(*shape, generator=self.g, device=dev())
        empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=dev())
        self.x, self.past, self.target = empty(rows, d, dtype=BF16), empty(rows, d, dtype=BF16), empty(rows, vocab)
        self.h, self.normed, self.dy, self.dx = (empty(rows, d, dtype=BF16) for _ in range(4))
        self.w_norm, self.b_norm = 1 + 0.1 * normal(d), 0.1 * normal(d)
        self.head = (normal(vocab, d) / math.sqrt(d)).to(BF16)
        # (the product back through the head takes whole eights: the gradient's rows and the turned head end in zeros)
        pad = -vocab % 8
        self.head_t = torch.nn.functional.pad(self.head.T, (0, pad)).contiguous()
        self.dz_wide = torch.zeros(rows, vocab + pad, dtype=BF16, device=dev())
        self.dz = self.dz_wide[:, :vocab]
        self.mean, self.rstd, self.loss, self.stats = empty(rows), empty(rows), empty(rows), empty(rows, 4)
        self.logits = empty(rows, vocab)
        self.dw, self.db = empty(d), empty(d)
        self.drawn = empty(rows, dtype=torch.int32)
        self.ids, self.probs = empty(rows, LS.SAMPLE_K_CAP, dtype=torch.int32), empty(rows, LS.SAMPLE_K_CAP)
        self.counts = empty(rows, 2, dtype=torch.int32)
        self.kept, self.teacher = empty(rows, dtype=torch.int32), empty(rows, LS.SAMPLE_K_CAP)
        self.adjusted, self.lse = empty(rows, vocab), empty(rows)
        params = [ls_params(temperature=1.0, top_k=self.k, top_p=1.0, seed=r) for r in range(rows)]
        self.draw = self.s.plan(self.target, params, [1] * rows, self.drawn, dbg_ids=self.ids, dbg_probs=self.probs, dbg_counts=self.counts)

    def feed(self):
        for t in (self.x, self.past):
            t.copy_(torch.randn(t.shape, generator=self.g, device=dev()))
        self.target.copy_(2 * torch.randn(self.target.shape, generator=self.g, device=dev()))

    def run(self):
        s = self.s
        self.draw.run(0)
        self.kept.copy_(self.counts[:, 0])
        if self.rest:   # the target's logits and its row's log-sum-exp
            self.draw.process_logits(self.adjusted, log_sum_exp=self.lse)
            torch.gather(self.adjusted, 1, self.ids.long().clamp(0, self.vocab - 1), out=self.teacher)
        else:           # what the draw says, exp(adjusted - top)
            self.teacher.copy_(self.probs)
        s.layer_norm(self.x, self.w_norm, self.b_norm, self.normed, eps=EPS, residual=self.past, summed=self.h, mean=self.mean, rstd=self.rstd)
        s.project(self.normed, self.head, self.logits)
        s.distill(self.logits, self.ids, self.teacher, self.loss, teacher=("probs", "logits")[self.rest], rest=self.rest,
                  teacher_lse=self.lse if self.rest else None, counts=self.kept, stats=self.stats, grad=self.dz)
        s.project(self.dz_wide, self.head_t, self.dy)
        s.layer_norm_backward(self.dy, self.h, self.mean, self.rstd, self.w_norm, grad_x=self.dx, grad_weight=self.dw, grad_bias=self.db)

    def outputs(self):
        return [t.clone() for t in (self.normed, self.logits, self.loss, self.stats, self.dz, self.dy, self.dx, self.dw, self.db)]

    def check(self):
        h, y, tol, mean, *_ = L.forward(self.x, self.past, "bf16", self.w_norm, self.b_norm)
        assert torch.equal(h.to(BF16), self.h)
        L.check_out(y, tol, self.normed, None, "bf16")
        P._check(self.logits, *P._formula(self.normed, self.head, None, None, None, "none", None))
        assert bool((self.kept == min(self.k, self.vocab)).all())
        c = D.Case.__new__(D.Case)
        c.rows, c.vocab, c.k, c.T, c.teacher, c.rest = self.rows, self.vocab, LS.SAMPLE_K_CAP, 1.0, ("probs", "logits")[self.rest], self.rest
        c.logits, c.ids, c.values, c.counts, c.lse, c.weights, c.scale = self.logits, self.ids, self.teacher, self.kept, self.lse, None, 1.0
        c.out = "bf16"
        want = c.formula()
        D.near(self.loss, want[0], want[1])
        D.near(self.dz, want[4], want[5])
        P._check(self.dy, *P._formula(self.dz_wide, self.head_t, None, None, None, "none", None))
        want = L.backward(self.dy, self.h, self.mean, self.rstd, self.w_norm, None)
        L.check_grad(self.dx, want[0], want[1])
        L.check_grad(self.dw, want[2], want[3])
        L.check_grad(self.db, want[4], want[5])

    def check_through(self):
        """The gradient at the head's input against all of it in 64 bits."""
        x = (self.x.float() + self.past.float()).to(BF16).double().requires_grad_(True)
        head = self.head.double()
        y = torch.nn.functional.layer_norm(x, (self.d,), self.w_norm.double(), self.b_norm.double(), EPS)
        z = y @ head.T
        z.retain_grad()
        y.retain_grad()
        on = torch.arange(LS.SAMPLE_K_CAP, device=dev())[None, :] < self.kept[:, None]
        t = self.teacher.double()
        p = torch.where(on, torch.exp(t - self.lse.double()[:, None]) if self.rest else t, 0.0)
        p = p if self.rest else p / p.sum(1, keepdim=True)
        dense = torch.zeros(self.rows, self.vocab, dtype=torch.float64, device=dev()).scatter_add_(1, torch.where(on, self.ids.long(), 0), p)
        logq = torch.log_softmax(z, 1)
        loss = -(dense * logq).sum(1)
        if self.rest:
            listed = dense > 0
            loss = loss - (1 - p.sum(1)).clamp_min(0) * torch.logsumexp(logq.masked_fill(listed, -math.inf), 1)
        loss.sum().backward()
        size = lambda t: t.double().norm(dim=1)
        s = float(torch.linalg.matrix_norm(head, 2))
        rstd = torch.rsqrt(x.detach().var(1, unbiased=False) + EPS)
        # (the rest as one outcome: two softmaxes, of all and of what is outside, each with its own Jacobian)
        jacobian = 1.0 if self.rest else 0.5
        far = rstd * float(self.w_norm.abs().max()) * (s * (s * size(y.detach()) * 2 ** -8 * 1.1 * jacobian + 2 ** -8 * size(z.grad)) + 2 ** -8 * 1.1 * size(y.grad))
        err = size(self.dx.double() - x.grad)
        assert bool((err <= far + 2 ** -8 * 1.1 * size(x.grad)).all()), (float(err.max()), float(far.min()))


@pytest.mark.parametrize("rows, d, vocab", [(1, 64, 1000), (5, 640, 10007), (70, 512, 32000), (300, 256, 20011)])
@pytest.mark.parametrize("rest", [False, True])
def test_a_training_step(rows, d, vocab, rest):
    t = Training(None, rows + vocab, rows, d, vocab, rest)
    for _ in range(2):
        t.feed()
        torch.cuda.synchronize()
        t.run()
        torch.cuda.synchronize()
        t.check()
        t.check_through()
    t.s.close()


@pytest.mark.parametrize("rest", [False, True])
def test_differences(rest, rows=3, d=400, k=20):
    """The norm in f32 as the logits themselves: the loss moves with the norm's weight, its bias and its rows as their gradients say.  A
    central difference over a step h = 2^-4 along the gradient u (unit length): the third derivative of a log-sum-exp along a move m of the
    logits is at most |m|max^3 (of the rest's, twice so), the norm's own along a move of a row, with rstd <= 1.2 here, at most 8 rstd^3 of
    it times the gradient; the losses are off by 2^-20 of (1 + their size) each."""
    s = LS.Sampler(0)
    g = torch.Generator(device=dev()).manual_seed(5)
    x = torch.randn(rows, d, generator=g, device=dev())
    w, b = 1 + 0.1 * torch.randn(d, generator=g, device=dev()), 0.1 * torch.randn(d, generator=g, device=dev())
    ids = torch.rand(rows, d, generator=g, device=dev()).topk(k, 1).indices.int()
    values = torch.rand(rows, k, generator=g, device=dev()) / k
    z, dz, dx = torch.empty(rows, d, device=dev()), torch.empty(rows, d, device=dev()), torch.empty(rows, d, device=dev())
    mean, rstd, loss = (torch.empty(rows, device=dev()) for _ in range(3))
    stats = torch.empty(rows, 4, device=dev())
    dw, db = torch.empty(d, device=dev()), torch.empty(d, device=dev())

    def run(x, w, b):
        torch.cuda.synchronize()
        s.layer_norm(x, w, b, z, eps=EPS, mean=mean, rstd=rstd)
        s.distill(z, ids, values, loss, teacher="probs", rest=rest, stats=stats, grad=dz)
        s.layer_norm_backward(dz, x, mean, rstd, w, grad_x=dx, grad_weight=dw, grad_bias=db)
        s.synchronize()
        return loss.double()

    base = run(x, w, b)
    xhat = ((x - mean[:, None]) * rstd[:, None]).abs().max()
    assert float(rstd.max()) <= 1.2
    grads = [t.clone().double() for t in (dx, dw, db)]
    h = 2.0 ** -4
    for i, grad in enumerate(grads):
        u = (grad / grad.norm()).float()
        moved = []
        for sign in (1.0, -1.0):
            at = [x, w, b]
            at[i] = at[i] + sign * h * u
            moved.append(run(*at))
        slope = float((moved[0] - moved[1]).sum()) / (2 * h)
        m = 1.2 * float(w.abs().max()) * float(u.norm(dim=1).max()) if i == 0 else float(u.abs().max()) * (float(xhat) if i == 1 else 1.0)
        third = rows * (1 + rest) * 2 * m ** 3 + (8 * 1.2 ** 3 * float(grad.norm()) if i == 0 else 0.0)
        bar = h * h / 6 * third + 2.0 ** -20 * float((1 + base.abs()).sum()) / h
        assert bar < 0.2 * float(grad.norm())
        assert abs(slope - float(grad.norm())) <= bar, (i, slope, float(grad.norm()), bar)
    s.close()


@pytest.mark.parametrize("rows, d, vocab", [(3, 256, 9001), (200, 128, 5003)])
def test_a_captured_training_step(rows, d, vocab):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        t = Training(stream, 3, rows, d, vocab, True)
        t.feed()
        t.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            t.run()
        for _ in range(4):
            t.feed()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            replayed = t.outputs()
            for o in (t.normed, t.logits, t.loss, t.stats, t.dz, t.dy, t.dx, t.dw, t.db):
                o.zero_()
            t.run()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(replayed, t.outputs()))
            t.check()
    t.s.close()


def test_two_samplers_at_once():
    """Two programs on streams of their own: what each computes is what it computes alone."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    steps, alone = [], []
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            t = Training(stream, 40 + i, (30, 260)[i], 256, (50021, 7001)[i], bool(i))
            t.feed()
            t.run()
            torch.cuda.synchronize()
            alone.append(t.outputs())
            steps.append(t)
    for _ in range(5):
        for t in steps:
            for o in (t.loss, t.dz, t.dx, t.dw):
                o.zero_()
        torch.cuda.synchronize()
        for turn in range(3):
            for t, stream in zip(steps, streams):
                with torch.cuda.stream(stream):
                    t.run()
        torch.cuda.synchronize()
        for t, want in zip(steps, alone):
            assert all(torch.equal(a, b) for a, b in zip(want, t.outputs()))
    for t in steps:
        t.s.close()


@pytest.mark.parametrize("rows", [1, 8, 40, 300])
def test_a_draft_through_8_bit_blocks(rows, d=896, vocab=9001, inner=500):
    """The weights laid out once; then the norm into blocks, a layer's product, the norm again, the head's, a greedy draw; and the distillation's
    teacher is the distribution that a draft left in its slot."""
    s = LS.Sampler(0)
    g = torch.Generator(device=dev()).manual_seed(rows)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev())
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=dev())
    weights = []
    for n, k in ((inner, d), (vocab, inner)):
        w, codes, scales = normal(n, k) / math.sqrt(k), empty(n, k, dtype=torch.float8_e4m3fn), empty(B.over(n), B.over(k))
        torch.cuda.synchronize()
        s.quantize_blocks(w, codes, scales)
        s.synchronize()
        pad = -k % 16   # (products take whole sixteens)
        weights.append((torch.nn.functional.pad(codes.view(torch.uint8), (0, pad)).view(torch.float8_e4m3fn), scales))
    x, b = normal(rows, d).to(BF16), normal(inner)
    q, qs = empty(rows, d, dtype=torch.float8_e4m3fn), empty(rows, B.over(d))
    wide = torch.zeros(rows, inner + (-inner % 16), dtype=torch.float8_e4m3fn, device=dev())
    inner_rows, inner_q, inner_s = empty(rows, inner, dtype=BF16), wide[:, :inner], empty(rows, B.over(inner))
    logits, drawn = empty(rows, vocab), empty(rows, dtype=torch.int32)
    torch.cuda.synchronize()
    s.layer_norm(x, None, None, q, eps=EPS, scales=qs)
    s.project_blocks(q, qs, *weights[0], inner_rows, bias=b, activation="gelu")
    s.layer_norm(inner_rows, None, None, inner_q, eps=EPS, scales=inner_s)
    s.project_blocks(wide, inner_s, *weights[1], logits)
    s.sample_rows(logits, [ls_params() for _ in range(rows)], [0] * rows, drawn)
    s.synchronize()
    _, y, tol, *_ = L.forward(x, None, None, None, None)
    L.check_out(y, tol, q, qs, "e4m3")
    P._check(inner_rows, *B.formula(q, qs, *weights[0], b, "gelu", None), B.cut(q, qs, *weights[0]) if rows > 16 else None)
    _, y, tol, *_ = L.forward(inner_rows, None, None, None, None)
    L.check_out(y, tol, inner_q, inner_s, "e4m3")
    P._check(logits, *B.formula(wide, inner_s, *weights[1], None, "none", None))
    assert torch.equal(drawn.long(), logits.argmax(1))
    # a draft's slot as the teacher of the row that it was drawn from: the loss is the list's own share, no gradient outside rounding
    dists, scratch, token = LS.DraftDists(s, 1), LS.SamplerScratch(s, vocab), empty(1, dtype=torch.int32)
    s.sample_draft_f32(logits[0], scratch, ls_params(temperature=1.0, top_k=30, top_p=0.9, seed=1), 0, token, dists.slot(0))
    ids, probs = dists.read(0)
    n, slot = len(ids), dists.slot(0)
    c = D.Case.__new__(D.Case)
    c.rows, c.vocab, c.k, c.T, c.teacher, c.rest, c.pad, c.start, c.out = 1, vocab, n, 1.0, "probs", False, 0, 0, "f32"
    c.logits, c.counts, c.lse, c.weights, c.scale = logits[:1], LS._device_view(slot.count_dev, 1, 0), None, None, 1.0
    c.ids = LS._device_view(slot.ids_dev, n, 0)[None]
    c.values = LS._device_view(slot.probs_dev, n, 0).view(torch.float32)[None]
    assert torch.equal(c.ids[0].cpu(), ids) and torch.equal(c.values[0].cpu(), probs)
    D.check(s, c)
    s.close()


def far_rows(rows, n, dtype, stride):
    """[rows, n] whose rows lie `stride` elements apart."""
    return torch.as_strided(torch.empty((rows - 1) * stride + n, dtype=dtype, device=dev()), (rows, n), (stride, 1))


def test_rows_further_apart_than_32_bits_reach():
    s = LS.Sampler(0)
    g = torch.Generator(device=dev()).manual_seed(9)
    rows, d = 3, 1000
    stride = (1 << 31) + 24   # elements: 4 GiB in bf16, 8 GiB in f32
    x, out = far_rows(rows, d, BF16, stride), far_rows(rows, d, BF16, stride + 8)
    x.copy_(torch.randn(rows, d, generator=g, device=dev()))
    mean, rstd = torch.empty(rows, device=dev()), torch.empty(rows, device=dev())
    torch.cuda.synchronize()
    s.layer_norm(x, None, None, out, eps=EPS, mean=mean, rstd=rstd)
    s.synchronize()
    _, y, tol, *_ = L.forward(x, None, None, None, None)
    L.check_out(y, tol, out, None, "bf16")
    for wide in (d, 9000):   # (one launch for gradient and sums, and one each)
        h, gx = (far_rows(rows, wide, BF16, stride + 16 * i) for i in (0, 1))
        h.copy_(torch.randn(rows, wide, generator=g, device=dev()))
        grad = torch.randn(rows, wide, generator=g, device=dev())
        mean, rstd = L.statistics(h)
        dw, db = torch.empty(wide, device=dev()), torch.empty(wide, device=dev())
        torch.cuda.synchronize()
        s.layer_norm_backward(grad, h, mean, rstd, None, grad_x=gx, grad_weight=dw, grad_bias=db)
        s.synchronize()
        want = L.backward(grad, h, mean, rstd, None, None)
        for got, k in ((gx, 0), (dw, 2), (db, 4)):
            L.check_grad(got, want[k], want[k + 1])
    del h, gx, out
    q = far_rows(rows, d, torch.float8_e4m3fn, 2 * stride)
    for block_rows in (1, 128):
        scales = torch.empty(rows if block_rows == 1 else 1, B.over(d), device=dev())
        torch.cuda.synchronize()
        s.quantize_blocks(x, q, scales)
        s.synchronize()
        near, again = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty_like(scales)
        close = x.contiguous()
        torch.cuda.synchronize()
        s.quantize_blocks(close, near, again)
        s.synchronize()
        assert torch.equal(q.contiguous().view(torch.uint8), near.view(torch.uint8)) and torch.equal(scales, again)
    s.close()


def test_a_product_over_more_bytes_than_32_bits_reach():
    """Rows 8 MiB apart, the widest that the product takes: 600 of them lie over 4.9 GB."""
    s = LS.Sampler(0)
    g = torch.Generator(device=dev()).manual_seed(2)
    for rows, n in ((600, 30), (20, 600), (600, 600)):
        d, stride = 1024, 1 << 23
        x0, xs, w0, ws = B.operands(g, rows, n, d)
        x, w = far_rows(rows, d, torch.float8_e4m3fn, stride), far_rows(n, d, torch.float8_e4m3fn, stride)
        x.view(torch.uint8).copy_(x0.view(torch.uint8)), w.view(torch.uint8).copy_(w0.view(torch.uint8))
        out = torch.empty(rows, n, dtype=BF16, device=dev())
        near = torch.empty_like(out)
        torch.cuda.synchronize()
        s.project_blocks(x, xs, w, ws, out)
        s.project_blocks(x0, xs, w0, ws, near)
        s.synchronize()
        P._check(out, *B.formula(x0, xs, w0, ws, None, "none", None), B.cut(x0, xs, w0, ws) if rows > 16 else None)
        P._check(near, *B.formula(x0, xs, w0, ws, None, "none", None), B.cut(x0, xs, w0, ws) if rows > 16 else None)
    s.close()
