"""The norm in front of the head (lily_rms_norm) against its formula in 64 bits.

Bar, derived from the arithmetic (u = 2^-24, half a step of f32):
  * h: bit-exact (one f32 addition of values that are f32 or bf16, one rounding to the stream's type);
  * y in f32: the sum of squares adds at most d / n_threads + 6 + waves <= 60 terms one after the other
    in any order of addition, each addition and product rounded: 62 u relative on a sum of positive
    terms, halved by the root (31 u), then division by d, + eps, root, reciprocal, two products and the
    addition of the offset: 8 u more.  40 u in all.  (The f64 value is taken of the f32-rounded weight
    plus offset, where the f32 addition of the offset may cancel.)
  * bf16: half a step more, 2^-8 relative;
  * E4M3: q * scale within half a step of y: 2^-4 relative for normal codes, half of 2^-9 * scale below,
    plus 45 u of y (the product with 448 / max); the scale within 42 u.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def _matrix(rng, rows, d, dtype, pad, scale=1.0, start=0):
    """[rows, d] of a buffer `pad` elements wider whose other elements hold NaN."""
    buf = torch.full((rows * (d + pad) + start + 8,), float("nan"), dtype=DT[dtype], device=dev())
    m = torch.as_strided(buf, (rows, d), (d + pad, 1), start)
    m.copy_(torch.from_numpy(rng.normal(0, scale, (rows, d)).astype(np.float32)))
    return buf, m


def _formula(x, residual, stream, weight, offset, eps):
    h = x.float()
    if residual is not None:
        h = (h + residual.float()).to(DT[stream])
    hd = h.double()
    w = (weight.float() + offset).double() if weight is not None else torch.ones(x.shape[1], device=x.device).double()
    return h, hd / torch.sqrt(hd.square().mean(1, keepdim=True) + eps) * w


def _check(y, out, scales, dtype):
    err = (out.double() * (scales.double()[:, None] if scales is not None else 1.0) - y).abs()
    if dtype == "f32":
        tol = 40 * U * y.abs()
    elif dtype == "bf16":
        tol = (2.0 ** -8 + 40 * U) * y.abs()
    else:
        top = y.abs().amax(1)
        assert bool(((scales.double() * 448.0 - top).abs() <= 42 * U * top).all())
        tol = torch.maximum((2.0 ** -4 + 90 * U) * y.abs(), 2.0 ** -10 * 1.0001 * scales.double()[:, None])
    assert bool((err <= tol + 1e-300).all()), float((err - tol).max())


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 63), (5, 64), (1, 4096), (61, 2560), (4, 5120), (3, 8193), (2, 16384), (2, 16392),
          (1, 32768), (2, 32767), (300, 520), (1, 511), (2, 513)]


@pytest.mark.parametrize("rows, d", SHAPES)
@pytest.mark.parametrize("xt, st, ot, wt", [("bf16", "bf16", "bf16", "bf16"), ("bf16", "f32", "e4m3", "f32"),
                                            ("f32", "f32", "f32", "f32"), ("f32", "bf16", "e4m3", "bf16"),
                                            ("bf16", None, "f32", "bf16"), ("f32", None, "bf16", None)])
@pytest.mark.parametrize("pad, start", [(0, 0), (8, 8), (3, 1)])
def test_against_the_formula(sampler, rows, d, xt, st, ot, wt, pad, start):
    rng = np.random.default_rng(rows * 1000 + d + pad)
    _, x = _matrix(rng, rows, d, xt, pad, 2.0, start)
    res = _matrix(rng, rows, d, st, pad, 3.0, start)[1] if st else None
    summed_buf, summed = _matrix(rng, rows, d, st, pad, 1.0, start) if st else (None, None)
    weight = torch.from_numpy(rng.normal(0, 1, d).astype(np.float32)).to(dev()).to(DT[wt]) if wt else None
    offset = 1.0 if wt == "bf16" else 0.0
    out_buf, out = _matrix(rng, rows, d, ot, pad, 1.0, start)
    before = out_buf.clone()
    scales = torch.full((rows,), -1.0, device=dev()) if ot == "e4m3" else None
    h, y = _formula(x, res, st, weight, offset, 1e-5)
    torch.cuda.synchronize()
    sampler.rms_norm(x, weight, out, eps=1e-5, residual=res, summed=summed, weight_offset=offset, scales=scales)
    sampler.synchronize()
    if st:
        assert torch.equal(summed, h)
    _check(y, out, scales, ot)
    # what lies between and behind the rows stays as it was
    if ot == "e4m3":
        out_buf, before = out_buf.view(torch.uint8), before.view(torch.uint8)
    mask = torch.ones_like(out_buf, dtype=torch.bool)
    torch.as_strided(mask, (rows, d), (d + pad, 1), start).fill_(False)
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[out_buf.element_size()]
    assert torch.equal(out_buf.view(bits)[mask], before.view(bits)[mask])


@pytest.mark.parametrize("d", [4096, 1001])
@pytest.mark.parametrize("where", ["sum is residual", "sum is x", "out is x", "out is residual, sum is x"])
def test_in_place(sampler, d, where):
    rng = np.random.default_rng(d)
    x = _matrix(rng, 9, d, "bf16", 0)[1]
    res = _matrix(rng, 9, d, "bf16", 0)[1]
    w = torch.from_numpy(rng.normal(0, 1, d).astype(np.float32)).to(dev())
    h, y = _formula(x, res, "bf16", w, 0.0, 1e-6)
    summed, out = torch.empty_like(x), torch.empty_like(x)
    summed = res if where == "sum is residual" else x if "sum is x" in where else summed
    out = x if where == "out is x" else res if "out is residual" in where else out
    torch.cuda.synchronize()
    sampler.rms_norm(x, w, out, residual=res, summed=summed)
    sampler.synchronize()
    assert torch.equal(summed.float(), h.float())
    _check(y, out, None, "bf16")


def test_rows_of_zeros_tiny_rows_and_rows_that_are_not_finite(sampler):
    x = torch.zeros(6, 256, device=dev())
    x[1] = 1e-30
    x[2] = 1e-42
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    x[5, 0] = 3.0
    out = torch.empty(6, 256, dtype=torch.float8_e4m3fn, device=dev())
    scales = torch.empty(6, device=dev())
    plain = torch.empty(6, 256, device=dev())
    torch.cuda.synchronize()
    sampler.rms_norm(x, None, out, eps=1e-6, scales=scales)
    sampler.rms_norm(x, None, plain, eps=1e-6)
    sampler.synchronize()
    q, sc, p = out.float().cpu(), scales.cpu(), plain.cpu()
    assert float(sc[0]) == 0.0 and bool((q[0] == 0).all())
    assert abs(float(sc[1]) * 448.0 / 1e-27 - 1.0) < 1e-5 and bool((q[1] == 448.0).all())
    assert float(sc[2]) == 0.0 and bool((q[2] == 0).all())      # 1e-39: below 2^-116
    assert bool(torch.isnan(sc[3])) and bool(torch.isnan(q[3]).all()) and bool(torch.isnan(p[3]).all())
    assert bool(torch.isnan(sc[4])) and bool(torch.isnan(q[4]).all())
    assert bool(torch.isnan(p[4, 7])) and bool((p[4, :7] == 0).all())
    assert float(q[5, 0]) == 448.0 and bool((q[5, 1:] == 0).all())


def test_an_eps_of_zero_over_a_row_of_zeros_is_what_the_formula_gives(sampler):
    x = torch.zeros(1, 64, device=dev())
    out = torch.empty(1, 64, device=dev())
    torch.cuda.synchronize()
    sampler.rms_norm(x, None, out, eps=0.0)
    sampler.synchronize()
    assert bool(torch.isnan(out).all())


def test_another_stream_and_a_captured_graph(sampler):
    """The call works on its sampler's stream, whatever stream torch is on, and allocates nothing: it can be
    captured, and every replay gives the eager result for what the buffers then hold."""
    stream = torch.cuda.Stream()
    s = LS.Sampler(0, stream)
    rng = np.random.default_rng(5)
    x = _matrix(rng, 33, 2560, "bf16", 0)[1]
    w = torch.from_numpy(rng.normal(1, 0.1, 2560).astype(np.float32)).to(dev())
    out = torch.empty(33, 2560, dtype=torch.float8_e4m3fn, device=dev())
    scales = torch.empty(33, device=dev())
    torch.cuda.synchronize()
    s.rms_norm(x, w, out, scales=scales)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.rms_norm(x, w, out, scales=scales)
    for turn in range(4):
        x.copy_(torch.from_numpy(rng.normal(0, 1 + turn, (33, 2560)).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.view(torch.uint8).clone(), scales.clone()
        out.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        s.rms_norm(x, w, out, scales=scales)
        s.synchronize()
        assert torch.equal(got[0], out.view(torch.uint8)) and torch.equal(got[1], scales)
        _check(_formula(x, None, None, w, 0.0, 1e-6)[1], out, scales, "e4m3")
    s.close()


def test_what_the_python_mirror_refuses(sampler):
    x = torch.zeros(2, 64, device=dev())
    w = torch.ones(64, device=dev())
    good = torch.empty(2, 64, device=dev())
    for bad in (dict(x=x.half()), dict(x=x.cpu()), dict(x=x[:, ::2]), dict(out=good[:1]), dict(weight=w[:32]),
                dict(residual=x[:1]), dict(summed=x), dict(residual=x, summed=x.bfloat16()),
                dict(out=good.to(torch.float8_e4m3fn)), dict(scales=torch.zeros(2, device=dev())), dict(eps=-1.0)):
        kw = dict(x=x, weight=w, out=good)
        kw.update(bad)
        with pytest.raises(LS.SamplerError):
            sampler.rms_norm(**kw)
