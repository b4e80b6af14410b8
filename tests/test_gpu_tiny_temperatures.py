"""Temperatures so small that logits divided by them lie far from zero, ties at the top among them: the draws' and the
head's log-probabilities against the oracle (ids exact, 1e-5, relative above 1), processed logits against 64 bits by
test_gpu_finite_fills.py's bar."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import lily_workloads as W
import oracle as O
from gpu_util import dev, run_rows
from test_gpu_finite_fills import _as, _check_rows

TEMPERATURES = [1e-4, 1e-6, 1e-8, 1e-10, 1e-12, 1e-16, 1e-20]
F = np.float32


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def _logits(rng, rows, vocab):
    x = rng.normal(0, 3, (rows, vocab)).astype(F)
    x[::2, [5, vocab // 2, vocab - 1]] = 16.0   # (a value of bf16)
    return x


@pytest.mark.parametrize("rows, vocab", [(1, 151_936), (20, 30_011), (300, 4100)])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("k", [1, 20, 64, 200, 0])
@pytest.mark.parametrize("masked", [False, True])
def test_draws(sampler, rows, vocab, bf16, k, masked):
    rng = np.random.default_rng(rows + k + bf16)
    for temperature in TEMPERATURES:
        x = _logits(rng, rows, vocab)
        given = W.to_bf16_bits(x) if bf16 else x
        allow = rng.integers(0, 2 ** 32, (rows, (vocab + 31) // 32), dtype=np.uint32) if masked else None
        kw = [dict(temperature=temperature, top_k=k, top_p=1.0, seed=r) for r in range(rows)]
        got = run_rows(sampler, given, kw, [3] * rows, allow=allow, logprobs=True)
        for r in range(0, rows, max(1, rows // 6)):
            d = O.sample(given[r], None, O.params(**kw[r]), 3, want_logprob=True, allow=None if allow is None else allow[r])
            what = (temperature, r, got.ids[r], d.chosen, got.logprobs[r], d.logprob)
            assert got.ids[r] == d.chosen, what
            assert abs(got.logprobs[r] - d.logprob) <= 1e-5 * max(1.0, abs(d.logprob)), what


@pytest.mark.parametrize("rows, vocab, d", [(3, 2048, 128), (4, 30_080, 256), (200, 8192, 256)])
@pytest.mark.parametrize("bf16", [False, True])
def test_the_head(sampler, rows, vocab, d, bf16):
    g = torch.Generator(device=dev())
    g.manual_seed(rows)
    hidden = torch.randn(rows, d, generator=g, device=dev()).bfloat16()
    weights = (torch.randn(vocab, d, generator=g, device=dev()) * 0.3).bfloat16()
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16 if bf16 else torch.float32, device=dev())
    tiles = (vocab + LS.LOGIT_TILE_COLS - 1) // LS.LOGIT_TILE_COLS
    top, part, lp = (torch.zeros(rows, n, device=dev()) for n in (tiles, tiles, 1))
    lp, ids = lp[:, 0].contiguous(), torch.zeros(rows, dtype=torch.int32, device=dev())
    for temperature in TEMPERATURES:
        for k in (1, 20, 64):
            kw = [dict(temperature=temperature, top_k=k, top_p=1.0, seed=r) for r in range(rows)]
            torch.cuda.synchronize()
            sampler.lm_head_sample_rows(hidden, weights, logits, top, part, [LS.SamplingParams.greedy(**q) for q in kw], [2] * rows, ids,
                                        out_logprobs=lp)
            sampler.synchronize()
            stored = logits.view(torch.int16).cpu().numpy().view(np.uint16) if bf16 else logits.cpu().numpy()
            for r in range(0, rows, max(1, rows // 4)):
                o = O.sample(stored[r], None, O.params(**kw[r]), 2, want_logprob=True)
                what = (temperature, k, r, int(ids[r]), o.chosen, float(lp[r]), o.logprob)
                assert int(ids[r]) == o.chosen, what
                assert abs(float(lp[r]) - o.logprob) <= 1e-5 * max(1.0, abs(o.logprob)), what


@pytest.mark.parametrize("temperature", TEMPERATURES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab", [(3, 30_011), (300, 4100)])
def test_processed_logits(sampler, temperature, dtype, rows, vocab):
    _check_rows(sampler, _as(_logits(np.random.default_rng(rows), rows, vocab), dtype), dtype, temperature)
