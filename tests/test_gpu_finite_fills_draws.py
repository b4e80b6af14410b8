"""The draws' log-probabilities for rows that hold finite values of any size, against the oracle: ids that a host bars with
a large negative number (a few, most, a thread's, a slice's), rows of nothing else, rows raised by a large positive one.
The ids are exact; a log-probability is within the 1e-5 (relative above 1) that every draw's is held to."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import lily_workloads as W
import oracle as O
from gpu_util import dev, run_rows

F = np.float32
FILLS = [-1e8, -1e9, -2e9, -5e9, -1e10, -1e12, -1e20, -1e30]
PATTERNS = ["most", "front", "back", "few", "one left", "all", "high", "two high"]


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def _rows(rng, n, vocab):
    """n rows of the patterns and fills in turn, their temperatures, an id of each that is not barred."""
    x, temps, free = rng.normal(0, 3, (n, vocab)).astype(F), [], []
    for r in range(n):
        pattern, fill = PATTERNS[r % len(PATTERNS)], FILLS[(r // len(PATTERNS) + r) % len(FILLS)]
        temps.append([1.0, 0.3, 1.0, 1.3][(r // 3) % 4])
        keep = vocab // 2
        if pattern == "most":
            kept = x[r, keep]
            x[r, rng.random(vocab) < 0.98] = fill
            x[r, keep] = kept
        elif pattern == "front":
            x[r, : int(vocab * 0.9)] = fill
            keep = vocab - 1
        elif pattern == "back":
            x[r, int(vocab * 0.3):] = fill
            keep = 0
        elif pattern == "few":
            x[r, 40:60] = fill
        elif pattern == "one left":
            kept = x[r, keep]
            x[r] = fill
            x[r, keep] = kept
        elif pattern == "all":
            x[r] = fill
        else:
            # (the oracle rounds every quotient by the temperature: no temperature, no rounding)
            temps[r] = 1.0
            if pattern == "high":
                x[r] = -fill
            else:
                x[r, vocab // 3] = x[r, vocab // 3 + 5] = -fill
                keep = vocab // 3
        free.append(keep)
    return x, temps, free


@pytest.mark.parametrize("rows, vocab", [(8, 151_936), (64, 9001), (136, 3001), (320, 4100)])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("k", [1, 20, 64, 200, 0])
@pytest.mark.parametrize("kind", ["plain", "penalties", "mask", "biases", "forced"])
def test_log_probabilities(sampler, rows, vocab, bf16, k, kind):
    rng = np.random.default_rng(rows * 31 + k * 7 + len(kind) + bf16)
    x, temps, free = _rows(rng, rows, vocab)
    given = W.to_bf16_bits(x) if bf16 else x
    kw = [dict(temperature=temps[r], top_k=k, top_p=0.98, seed=r) for r in range(rows)]
    scratch = allow = bias = forced = None
    counts = [None] * rows
    if kind == "penalties":
        scratch = []
        for r in range(rows):
            kw[r].update(repetition_penalty=1.05, presence_penalty=0.3, frequency_penalty=0.2)
            scratch.append(LS.SamplerScratch(sampler, vocab))
            h = rng.integers(0, vocab, 50).astype(np.int32)
            scratch[-1].add_history(torch.from_numpy(h).to(dev()))
            counts[r] = np.bincount(h, minlength=vocab).astype(np.uint32)
    elif kind == "mask":
        allow = rng.integers(0, 2 ** 32, (rows, (vocab + 31) // 32), dtype=np.uint32)
        for r in range(rows):
            allow[r, free[r] >> 5] |= np.uint32(1) << np.uint32(free[r] & 31)
    elif kind == "biases":
        # (integers: a sum with a value whose step they lie below is rounded the same way by both)
        bias = [[(int(i), float(d)) for i, d in zip(rng.choice(vocab, 10, replace=False), rng.integers(-3, 4, 10))] for _ in range(rows)]
        temps = [1.0] * rows
        for d in kw:
            d["temperature"] = 1.0
    elif kind == "forced":
        forced = [free[r] if r % 3 else LS.NO_TOKEN for r in range(rows)]
    got = run_rows(sampler, given, kw, [3] * rows, scratch=scratch, allow=allow, bias=bias, forced=forced, logprobs=True, use_plan=bool(k % 3))
    for r in range(0, rows, max(1, rows // 64)):
        d = O.sample(given[r], counts[r], O.params(**kw[r]), 3, want_logprob=True, allow=None if allow is None else allow[r],
                     bias=None if bias is None else bias[r], forced=None if forced is None or forced[r] == LS.NO_TOKEN else forced[r])
        what = (r, PATTERNS[r % len(PATTERNS)], temps[r], got.ids[r], d.chosen, got.logprobs[r], d.logprob)
        assert got.ids[r] == d.chosen, what
        assert abs(got.logprobs[r] - d.logprob) <= 1e-5 * max(1.0, abs(d.logprob)), what
