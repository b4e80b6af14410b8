"""The matrix product's tile of 256 x 256 (lily_project) against the formula in 64 bits; the bar is test_gpu_project.py's.

Sizes that get the tile by themselves (test_project_plan.py asks for each of them), and small and ragged ones through
LILY_SAMPLER_PROJECT=256, which gives it to every product of more than 16 rows.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev
from project_sizes import LARGE_TILE
from test_gpu_project import U, _check, _formula, _rows, _run


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def _with_tile(tile, stream=None):
    patch = pytest.MonkeyPatch()
    patch.setenv("LILY_SAMPLER_PROJECT", str(tile))
    try:
        return LS.Sampler(0, stream) if stream is not None else LS.Sampler(0)
    finally:
        patch.undo()


@pytest.fixture(scope="module")
def large():
    s = _with_tile(256)
    yield s
    s.close()


# Rows of the residual that start at any element, whose lines the tile asks for ahead of its epilogue (from eleven
# stages on): tiles that end inside rows and outputs, a d that ends inside a stage.
@pytest.mark.parametrize("rows, n, d, dtype, out, residual, start", [
    (4090, 4090, 4112, "bf16", "bf16", "bf16", 3), (4090, 4090, 4112, "bf16", "f32", "f32", 3),
    (4096, 4096, 4096, "bf16", "bf16", "bf16", 1), (4090, 4090, 4112, "bf16", "f32", "bf16", 1),
    (1020, 16380, 8208, "e4m3", "bf16", "bf16", 1), (1020, 16380, 8208, "e4m3", "bf16", "f32", 5)])
def test_residuals_at_any_element(sampler, rows, n, d, dtype, out, residual, start):
    _run(sampler, rows, n, d, dtype, out, "silu", "f32", residual, start=start)


@pytest.mark.parametrize("size", [s for s in LARGE_TILE if s[6] == 0], ids=lambda s: "-".join(map(str, s[:6])))
def test_sizes_that_get_the_tile(sampler, size):
    rows, n, d, dtype, out, residual, start = size
    _run(sampler, rows, n, d, dtype, out, "gelu", "bf16", residual, start=start)


KINDS = [("bf16", "f32"), ("bf16", "bf16"), ("e4m3", "f32"), ("e4m3", "bf16")]


# rows and outputs around the tile's, a wave's, a block's edges
@pytest.mark.parametrize("rows", [17, 32, 33, 127, 129, 255, 256, 257, 385, 513])
@pytest.mark.parametrize("n", [1, 3, 7, 8, 31, 129, 255, 256, 257, 383, 520])
@pytest.mark.parametrize("dtype, out", KINDS)
def test_rows_and_outputs(large, rows, n, dtype, out):
    _run(large, rows, n, 256, dtype, out, scales=dtype == "e4m3")


# d from one piece of 16 bytes on: part of a stage, one to many stages, odd and even numbers of them, the last whole or not
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 128, 144, 192, 256, 320, 384, 400, 512, 640, 656, 704, 768, 896, 1008, 1088, 1408, 1536,
                               1552, 4096, 4112])
@pytest.mark.parametrize("dtype, out", KINDS)
def test_widths(large, d, dtype, out):
    _run(large, 300, 270, d, dtype, out, pad=1)


# the epilogue: residuals and outputs of both types at any element, every activation, with few stages and with enough that the
# residual's lines are asked for early; whole tiles among ragged ones
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("out_dtype, residual, bias, scales", [
    ("bf16", "bf16", "f32", True), ("f32", "f32", "bf16", True), ("f32", "bf16", None, False), ("bf16", "f32", "bf16", False),
    ("bf16", None, None, True), ("f32", "f32", None, False)])
@pytest.mark.parametrize("rows, n, d, start", [(257, 300, 320, 0), (300, 261, 64, 1), (520, 514, 1040, 3), (512, 512, 768, 4), (270, 256, 2064, 5)])
def test_epilogues(large, act, out_dtype, residual, bias, scales, rows, n, d, start):
    for dtype in ("bf16", "e4m3"):
        # (the bound of the 8-bit products asks for scales)
        _run(large, rows, n, d, dtype, out_dtype, act, bias, residual, scales or dtype == "e4m3", pad=2, start=start)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows, n, d, forced", [(4096, 4096, 4096, False), (300, 513, 1552, True), (512, 256, 144, True)])
def test_in_place_of_the_residual(sampler, large, dtype, rows, n, d, forced):
    s = large if forced else sampler
    g = torch.Generator(device=dev())
    g.manual_seed(8)
    x, w = _rows(g, rows, d, "bf16")[1], _rows(g, n, d, "bf16", 0, 0.02)[1]
    res = _rows(g, rows, n, dtype, 3)[1]
    want, tol = _formula(x, w, None, None, None, "silu", res)
    apart = torch.empty(rows, n, dtype=res.dtype, device=dev())
    torch.cuda.synchronize()
    s.project(x, w, apart, activation="silu", residual=res)
    s.project(x, w, res, activation="silu", residual=res)
    s.synchronize()
    _check(res, want, tol)
    assert torch.equal(apart, res)


def test_values_that_are_not_finite(large):
    """A NaN or an infinity stays in its row (of x) or column (of the weights)."""
    for rows, n in ((40, 70), (300, 500)):
        x = torch.ones(rows, 192, dtype=torch.bfloat16, device=dev())
        w = torch.ones(n, 192, dtype=torch.bfloat16, device=dev())
        x[1, 5] = float("nan")
        x[rows - 1, 7] = float("inf")
        w[9, 191] = float("-inf")
        out = torch.empty(rows, n, device=dev())
        torch.cuda.synchronize()
        large.project(x, w, out)
        large.synchronize()
        got, others = out.cpu(), torch.arange(n) != 9
        assert bool(torch.isnan(got[1]).all())
        assert bool((got[-1][others] == math.inf).all()) and bool(torch.isnan(got[-1, 9]))
        rest = torch.ones(rows, dtype=torch.bool)
        rest[1] = rest[-1] = False
        assert bool((got[rest][:, 9] == -math.inf).all()) and bool((got[rest][:, others] == 192.0).all())


@pytest.mark.parametrize("dtype, out_dtype", KINDS)
def test_the_same_bits_every_time_and_wherever_a_row_lies(large, dtype, out_dtype):
    """A call repeats its bits, and a row's values are the same wherever it lies among the tiles."""
    g = torch.Generator(device=dev())
    g.manual_seed(4)
    x, w = _rows(g, 600, 1040, dtype)[1], _rows(g, 300, 1040, dtype)[1]
    whole = [torch.empty(600, 300, dtype=torch.bfloat16 if out_dtype == "bf16" else torch.float32, device=dev()) for _ in range(6)]
    part = torch.empty(301, 300, dtype=whole[0].dtype, device=dev())
    torch.cuda.synchronize()
    for o in whole:
        large.project(x, w, o)
    large.project(x[299:], w, part)
    large.synchronize()
    assert all(torch.equal(whole[0], o) for o in whole[1:])
    assert torch.equal(whole[0][299:], part)


def test_another_stream_and_a_captured_graph():
    stream = torch.cuda.Stream()
    s = _with_tile(256, stream)
    g = torch.Generator(device=dev())
    g.manual_seed(9)
    for rows, n, d in ((300, 700, 2048), (40, 512, 400)):
        x, w = _rows(g, rows, d, "bf16")[1], _rows(g, n, d, "bf16", 0, 1 / math.sqrt(d))[1]
        bias, res = torch.randn(n, generator=g, device=dev()), torch.randn(rows, n, generator=g, device=dev())
        out = torch.empty(rows, n, dtype=torch.bfloat16, device=dev())
        torch.cuda.synchronize()
        s.project(x, w, out, bias=bias, activation="gelu", residual=res)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.project(x, w, out, bias=bias, activation="gelu", residual=res)
        for _ in range(3):
            x.copy_(torch.randn(rows, d, generator=g, device=dev()))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            out.zero_()
            torch.cuda.synchronize()
            s.project(x, w, out, bias=bias, activation="gelu", residual=res)
            s.synchronize()
            assert torch.equal(got, out)
            want, tol = _formula(x, w, None, None, bias, "gelu", res)
            _check(out, want, tol)
    s.close()


@pytest.mark.parametrize("out_dtype", ["f32", "bf16"])
def test_gelu_over_its_range(large, out_dtype):
    """Rows of zeros, so that the bias is the argument; the bar is test_gpu_project.py's for it."""
    n = 20001
    v = torch.cat([torch.linspace(-14, 14, n - 2000, dtype=torch.float64), torch.logspace(-30, 0, 1000, dtype=torch.float64),
                   -torch.logspace(-30, 0, 1000, dtype=torch.float64)]).float().to(dev())
    v[7], v[8], v[9], v[10] = 0.0, -0.0, 1e30, float("inf")
    x = torch.zeros(20, 64, dtype=torch.bfloat16, device=dev())
    w = torch.ones(n, 64, dtype=torch.bfloat16, device=dev())
    out = torch.empty(20, n, dtype=torch.bfloat16 if out_dtype == "bf16" else torch.float32, device=dev())
    torch.cuda.synchronize()
    large.project(x, w, out, bias=v, activation="gelu")
    large.synchronize()
    d = v.double()
    low = (0.5 * torch.special.erfc(d.abs().cpu() * math.sqrt(0.5))).to(dev())
    want, tail = d * torch.where(d > 0, 1.0 - low, low), low
    want[8], want[10] = 0.0, float("inf")
    near = 8 + d.square().clamp_max(1e4)
    tol = torch.where(d < 0, (near + 1) * U * want.abs(), d.abs() * U * (near * tail + 2)) + 2.0 ** -126 * d.abs().clamp_max(100.0)
    if out_dtype == "bf16":
        tol = tol + 2.0 ** -8 * want.abs()
    ok = ((out.double() - want).abs() <= tol) | (out.double() == want)
    assert bool(ok.all()), (v[~ok.all(0)][:5], out[:, ~ok.all(0)][0, :5], want[~ok.all(0)][:5])


# the other two tiles by the switch, where the estimate would take another: parts of d as it chooses among them
@pytest.mark.parametrize("tile", [64, 128])
def test_the_other_tiles_by_the_switch(tile):
    s = _with_tile(tile)
    for rows, n, d in ((17, 33, 64), (40, 1000, 8192), (300, 257, 2064), (2051, 4100, 1040)):
        for dtype, out in KINDS:
            _run(s, rows, n, d, dtype, out, "silu", "f32", out, start=1)
    s.close()
