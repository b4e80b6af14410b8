"""lily_rms_norm where f32 ends, as include/lily_sampler.h states it: infinite weights, products that overflow, squares that
do."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def _norm(sampler, x, w, eps=1e-6):
    rows, d = x.shape
    q, sc = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(rows, device=dev())
    y = torch.empty(rows, d, device=dev())
    torch.cuda.synchronize()
    sampler.rms_norm(x, w, q, eps=eps, scales=sc)
    sampler.rms_norm(x, w, y, eps=eps)
    sampler.synchronize()
    return q.float().cpu(), sc.cpu(), y.cpu()


@pytest.mark.parametrize("big", [math.inf, 3e38])
def test_products_with_the_weight_that_are_not_finite(sampler, big):
    x = torch.ones(2, 128, device=dev())
    x[:, 9] = 4.0                        # (its product with 3e38 overflows: the row's root is about 1.06)
    w = torch.ones(128, device=dev())
    w[9] = big
    q, sc, y = _norm(sampler, x, w)
    assert bool((y[:, 9] == math.inf).all()) and bool(torch.isfinite(y[:, :9]).all())
    assert bool((sc == math.inf).all())
    assert bool(torch.isnan(q[:, 9]).all()) and bool((q[:, :9] == 0).all()) and bool((q[:, 10:] == 0).all())


@pytest.mark.parametrize("d", [64, 4096, 32768])
def test_squares_that_overflow(sampler, d):
    x = torch.full((2, d), 2.0 ** 65, device=dev())
    x[1] = 2.0 ** 55
    q, sc, y = _norm(sampler, x, None)
    assert bool((y[0] == 0).all()) and float(sc[0]) == 0.0 and bool((q[0] == 0).all())
    assert bool(((y[1] - 1.0).abs() <= 40 * 2.0 ** -24).all()) and bool((q[1] == 448.0).all())


def test_small_rows_without_an_eps(sampler):
    x = torch.full((1, 256), 2.0 ** -63, device=dev())
    q, sc, y = _norm(sampler, x, None, 0.0)
    assert bool(((y - 1.0).abs() <= 40 * 2.0 ** -24).all()) and bool((q == 448.0).all())
