"""Processed logits of rows that hold finite values of any size: ids that a host bars with a large negative number, rows
of nothing else, rows that lie together far from zero.

Bar: adjusted values bit for bit; with top the row's largest value and s = log sum exp(a - top) in f64, what a row's sum and its
logarithm lose is off = (1.25 n + 8) 2^-24, n = max(8, V / 1024) (a thread's additions, exponents and exponentials
rounded); log_sum_exp is top + s rounded once, off + |top + s| 2^-24; a log-probability p = (a - top) - s has the
roundings of a - top, of s and of their difference besides, none of them larger than p: off + 3 |p| 2^-24.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import lily_workloads as W
from gpu_util import dev, ls_params, upload_logits

U = 2.0 ** -24
F = np.float32


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def _check_rows(sampler, x, dtype, temperature):
    """x: f32 rows (of bf16 values where dtype says so), none of them empty or with an infinity."""
    rows, vocab = x.shape
    logits = upload_logits(W.to_bf16_bits(x) if dtype == "bf16" else x)
    params = [ls_params(temperature=temperature, top_k=20, seed=r) for r in range(rows)]
    a = (x / F(temperature)).astype(F)
    wide = a.astype(np.float64)
    top = wide.max(1, keepdims=True)
    s = np.log(np.exp(wide - top).sum(1, keepdims=True))
    off = (1.25 * max(8, vocab / 1024) + 8) * U
    for logprobs in (False, True):
        out, lse = torch.empty(rows, vocab, device=dev()), torch.empty(rows, device=dev())
        torch.cuda.synchronize()
        keep = sampler.process_logits(logits, params, out, log_sum_exp=lse, logprobs=logprobs)
        sampler.synchronize()
        got, got_lse = out.cpu().numpy(), lse.cpu().numpy().astype(np.float64)
        want = (top + s)[:, 0]
        bad = ~(np.abs(got_lse - want) <= off + np.abs(want) * U)
        assert not bad.any(), (logprobs, np.nonzero(bad)[0][:4], got_lse[bad][:4], want[bad][:4])
        if logprobs:
            p = (wide - top) - s
            bad = ~(np.abs(got.astype(np.float64) - p) <= off + 3 * U * np.abs(p))
            assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], p[bad][:4])
        else:
            assert np.array_equal(got.view(np.uint32), a.view(np.uint32))
        del keep


def _as(x, dtype):
    x = np.ascontiguousarray(x, dtype=F)
    return W.bf16_bits_to_f32(W.to_bf16_bits(x)) if dtype == "bf16" else x


# every row of a batch once: few ids left, most of them, a thread's share barred among ordinary ones, nothing but fill
@pytest.mark.parametrize("fill", [-1e6, -1e8, -1e9, -1e10, -1e12, -1e20, -1e30])
@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.0, 1.3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("copies, vocab", [(1, 30001), (75, 9001)])
def test_barred_by_a_large_negative_number(sampler, fill, temperature, dtype, copies, vocab):
    rng = np.random.default_rng(int(-fill) % 1009 + vocab)
    x = rng.normal(0, 3, (4 * copies, vocab)).astype(F)
    x[0::4][rng.random((copies, vocab)) < 0.98] = fill
    x[1::4][rng.random((copies, vocab)) < 0.3] = fill
    for u in range(8):                               # the ids of neighbouring threads, in every group they hold
        x[2::4, 1024 * u + 40:1024 * u + 60] = fill
    x[3::4] = fill
    _check_rows(sampler, _as(x, dtype), dtype, temperature)


@pytest.mark.parametrize("temperature", [0.3, 1.0])
@pytest.mark.parametrize("fill", [-1e10, -1e30])
def test_a_whole_vocabulary_of_which_little_is_left(sampler, temperature, fill):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 3, (3, 151_936)).astype(F)
    x[rng.random(x.shape) < 0.98] = fill
    _check_rows(sampler, x, "f32", temperature)


# (the steps of f32 are 2^-24 of the middle: values of a few steps apart, and all the same)
@pytest.mark.parametrize("middle", [2.0 ** 22, 2.0 ** 24 - 8, 2.0 ** 24, 2.0 ** 26, 2.0 ** 30, 1e10, 1e20, 1e30, 3e38])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("temperature", [0.9, 1.0])
def test_rows_that_lie_together_far_from_zero(sampler, middle, sign, temperature):
    if middle == 3e38 and temperature < 1.0:
        middle = 2.9e38                              # (its quotient is a number still)
    rng = np.random.default_rng(7)
    m = F(sign * middle)
    x = np.full((4, 8200), m, F)
    x[1] = m + rng.integers(-4, 5, 8200) * np.spacing(np.abs(m))
    x[2, ::3] = 0.0
    x[3, rng.random(8200) < 0.5] = rng.normal(0, 2, 1)
    _check_rows(sampler, x.astype(F), "f32", temperature)
