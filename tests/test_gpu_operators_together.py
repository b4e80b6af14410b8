"""What a decode step does from its last layer to the token, by the operators one after the other: the residual's
addition and the norm, a draft head's block, the norm into 8 bits, a head held in 8-bit floats, processed logits and
the draw.  Every stage is held to its formula in 64 bits on what the stage before left (bars as for each alone)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import test_gpu_norm as N
import test_gpu_project as P
from gpu_util import dev, ls_params

EPS = 1e-6


class Step:
    """A program's resident buffers for `rows` conversations; they share a wider hidden buffer."""

    def __init__(self, stream, seed, rows, d, vocab):
        self.s = LS.Sampler(0, stream)
        self.stream, self.rows, self.d, self.vocab = stream, rows, d, vocab
        self.g = g = torch.Generator(device=dev())
        g.manual_seed(seed)
        normal = lambda *shape: torch.randn(*shape, generator=g, device=dev())
        bf16 = torch.bfloat16
        wide = torch.zeros(rows, 2 * d, dtype=bf16, device=dev())
        self.x, self.h = wide[:, :d], wide[:, d:]           # side by side, one stride
        self.h0 = torch.empty(rows, d, dtype=bf16, device=dev())
        self.w_norm, self.w_last = (1 + 0.1 * normal(d)).to(bf16), 0.1 * normal(d)
        self.w_block, self.b_block = (normal(d, d) / math.sqrt(d)).to(bf16), 0.1 * normal(d)
        head = normal(vocab, d)
        self.head_scales = head.abs().amax(1) / 448.0
        self.head = (head / self.head_scales[:, None]).to(torch.float8_e4m3fn)
        self.head_scales /= math.sqrt(d)
        self.normed, self.block = torch.empty(rows, d, dtype=bf16, device=dev()), torch.empty(rows, d, dtype=bf16, device=dev())
        self.q, self.q_scales = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(rows, device=dev())
        self.logits, self.adjusted = torch.empty(rows, vocab, device=dev()), torch.empty(rows, vocab, device=dev())
        self.lse, self.ids, self.again = (torch.empty(rows, device=dev(), dtype=t) for t in (torch.float32, torch.int32, torch.int32))
        self.scratch, self.history = [], torch.randint(vocab, (rows, 40), generator=g, device=dev(), dtype=torch.int32)
        for r in range(rows):
            self.scratch.append(LS.SamplerScratch(self.s, vocab))
        params = [ls_params(temperature=0.7, top_k=30, top_p=0.9, seed=r, repetition_penalty=1.1, presence_penalty=0.5) for r in range(rows)]
        plain = [ls_params(temperature=1.0, top_k=30, top_p=0.9, seed=r) for r in range(rows)]
        self.plan = self.s.plan(self.logits, params, [3] * rows, self.ids, scratch=self.scratch)
        self.from_adjusted = self.s.plan(self.adjusted, plain, [3] * rows, self.again)

    def feed(self):
        self.x.copy_(torch.randn(self.rows, self.d, generator=self.g, device=dev()))
        self.h0.copy_(torch.randn(self.rows, self.d, generator=self.g, device=dev()))

    def begin(self):
        """The state a step changes, as it was (an eager step or a replay may follow)."""
        self.h.copy_(self.h0)
        for r, c in enumerate(self.scratch):
            c.reset_counts()
            c.add_history(self.history[r])

    def run(self):
        s = self.s
        s.rms_norm(self.x, self.w_norm, self.normed, eps=EPS, residual=self.h, summed=self.h)
        s.project(self.normed, self.w_block, self.block, bias=self.b_block, activation="silu", residual=self.h)
        s.rms_norm(self.block, self.w_last, self.q, eps=EPS, weight_offset=1.0, scales=self.q_scales)
        s.project(self.q, self.head, self.logits, x_scales=self.q_scales, weight_scales=self.head_scales)
        self.plan.process_logits(self.adjusted, log_sum_exp=self.lse)
        self.plan.run(0)
        self.from_adjusted.run(0)

    def outputs(self):
        return [t.clone() for t in (self.h, self.normed, self.block, self.q.view(torch.uint8), self.q_scales, self.logits,
                                    self.adjusted, self.lse, self.ids, self.again)]

    def check(self):
        h, y = N._formula(self.x, self.h0, "bf16", self.w_norm, 0.0, EPS)
        assert torch.equal(h, self.h)
        N._check(y, self.normed, None, "bf16")
        P._check(self.block, *P._formula(self.normed, self.w_block, None, None, self.b_block, "silu", self.h))
        _, y = N._formula(self.block, None, None, self.w_last, 1.0, EPS)
        N._check(y, self.q, self.q_scales, "e4m3")
        P._check(self.logits, *P._formula(self.q, self.head, self.q_scales, self.head_scales, None, "none", None))
        # sums of at most 0.001 vocab + 8 terms a thread, each rounded three times
        lse = torch.logsumexp(self.adjusted.double(), 1)
        assert bool(((self.lse - lse).abs() <= (1.25 * max(8, self.vocab / 1024) + 8 + lse.abs()) * 2.0 ** -24).all())
        # a count of the history lowers a logit, everything else is the logit over the temperature
        counted = torch.zeros(self.rows, self.vocab, dtype=torch.bool, device=dev())
        counted.scatter_(1, self.history.long(), True)
        assert torch.equal(self.adjusted[~counted], (self.logits / torch.tensor(0.7, device=dev()))[~counted])
        assert bool((self.adjusted[counted] < self.logits[counted] / 0.7).all())
        assert torch.equal(self.ids, self.again)             # the draw from the written rows is the raw rows' draw
        assert bool(((self.ids >= 0) & (self.ids < self.vocab)).all())

    def close(self):
        self.plan.close()
        self.from_adjusted.close()
        for c in self.scratch:
            c.close()
        self.s.close()


@pytest.mark.parametrize("rows, d, vocab", [(1, 256, 1000), (4, 512, 12345), (13, 1040, 5000), (70, 512, 9001), (300, 512, 3001)])
def test_a_step_from_the_last_layer_to_the_token(rows, d, vocab):
    step = Step(torch.cuda.Stream(), rows, rows, d, vocab)
    for _ in range(2):
        step.feed()
        torch.cuda.synchronize()
        step.begin()
        torch.cuda.synchronize()
        step.run()
        step.s.synchronize()
        step.check()
    step.close()


def test_two_programs_at_once():
    """Two samplers' steps enqueued in turn on their own streams, with nothing waited for between them."""
    steps = [Step(torch.cuda.Stream(), 10 + i, rows, 512, 20011) for i, rows in enumerate((40, 130))]
    for step in steps:
        step.feed()
    torch.cuda.synchronize()
    for step in steps:
        step.begin()
    torch.cuda.synchronize()
    for step in steps:
        step.run()
    torch.cuda.synchronize()
    alone = [step.outputs() for step in steps]
    for step in steps:
        step.check()
    for _ in range(4):
        for step in steps:
            step.begin()
        torch.cuda.synchronize()
        for i in range(6):
            for step in steps:
                step.s.rms_norm(step.x, step.w_norm, step.normed, eps=EPS, residual=step.h0, summed=step.h)
                step.s.project(step.normed, step.w_block, step.block, bias=step.b_block, activation="silu", residual=step.h)
                step.plan.process_logits(step.adjusted, log_sum_exp=step.lse, logprobs=True)
        torch.cuda.synchronize()
        for step in steps:
            step.h.copy_(step.h0)   # (torch's stream, not the samplers')
        torch.cuda.synchronize()
        for step in steps:
            step.run()
        torch.cuda.synchronize()
        for step, first in zip(steps, alone):
            assert all(torch.equal(a, b) for a, b in zip(first, step.outputs()))
    for step in steps:
        step.close()


@pytest.mark.parametrize("rows", [4, 70])
def test_a_captured_step(rows):
    """The whole step as one graph, replayed over changing inputs, with eager steps and waits between the replays."""
    stream = torch.cuda.Stream()
    step = Step(stream, 20 + rows, rows, 512, 30011)
    step.feed()
    step.begin()
    torch.cuda.synchronize()
    step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step.run()
    for _ in range(4):
        step.feed()
        step.begin()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step.check()
        replayed = step.outputs()
        step.begin()
        torch.cuda.synchronize()
        step.run()
        step.s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, step.outputs()))
    step.close()


FAR = (1 << 31) + 24   # elements between two rows: their bytes, and in f32 their elements' bytes twice over, pass 32 bits


def _far(rows, cols, dtype):
    """[rows, cols] with FAR elements from row to row (what lies between is not touched, nor ever written)."""
    return torch.as_strided(torch.empty((rows - 1) * FAR + cols, dtype=dtype, device=dev()), (rows, cols), (FAR, 1))


def test_rows_that_lie_further_apart_than_32_bits():
    s = LS.Sampler(0)
    g = torch.Generator(device=dev())
    g.manual_seed(5)
    rows, d, n, vocab = 3, 512, 300, 9000
    x, h, out = (_far(rows, d, torch.bfloat16) for _ in range(3))
    x.copy_(torch.randn(rows, d, generator=g, device=dev()))
    h.copy_(torch.randn(rows, d, generator=g, device=dev()))
    w = torch.ones(d, device=dev())
    torch.cuda.synchronize()
    before = h.clone()
    s.rms_norm(x, w, out, eps=EPS, residual=h, summed=h)
    s.synchronize()
    want_h, y = N._formula(x, before, "bf16", w, 0.0, EPS)
    assert torch.equal(want_h, h)
    N._check(y, out, None, "bf16")
    del x, h
    torch.cuda.empty_cache()
    for many in (rows, 20):   # few rows, and tiles (of rows side by side)
        res, o = _far(rows, n, torch.bfloat16), _far(rows, n, torch.float32)
        a = out.contiguous() if many == rows else torch.randn(many, d, generator=g, device=dev()).bfloat16()
        if many != rows:
            del res, o
            torch.cuda.empty_cache()
            stride = (1 << 28) + 8
            res, o = (torch.as_strided(torch.empty((many - 1) * stride + n, dtype=t, device=dev()), (many, n), (stride, 1))
                      for t in (torch.bfloat16, torch.float32))
        res.copy_(torch.randn(many, n, generator=g, device=dev()))
        weight = (torch.randn(n, d, generator=g, device=dev()) / math.sqrt(d)).bfloat16()
        torch.cuda.synchronize()
        s.project(a, weight, o, activation="silu", residual=res)
        s.synchronize()
        P._check(o, *P._formula(a, weight, None, None, None, "silu", res))
        del res, o
        torch.cuda.empty_cache()
    logits, adjusted = _far(rows, vocab, torch.bfloat16), _far(rows, vocab, torch.float32)
    logits.copy_(torch.randn(rows, vocab, generator=g, device=dev()) * 3)
    lse = torch.empty(rows, device=dev())
    params = [ls_params(temperature=0.5, top_k=5, seed=r) for r in range(rows)]
    torch.cuda.synchronize()
    keep = s.process_logits(logits, params, adjusted, log_sum_exp=lse)
    s.synchronize()
    assert torch.equal(adjusted, logits.float() / 0.5)
    ref = torch.logsumexp(adjusted.double(), 1)
    assert bool(((lse - ref).abs() <= (1.25 * 9 + 8 + ref.abs()) * 2.0 ** -24).all())
    del keep
    s.close()
