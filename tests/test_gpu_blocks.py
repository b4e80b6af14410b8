"""8-bit floats with a scale for each block (lily_quantize_blocks) and their product (lily_project_blocks) against the formulas in
64 bits.

Bars (u = 2^-24).  Quantisation: a scale is one division, equal to f32(max / 448); q is x times 448 / max rounded (3 u) and then half a
step of E4M3 (2^-4 relative, half of 2^-9 below the normal codes).
Product: with S_b = sum |x_i w_i| of a block and S = sum_b S_b xs ws, a block's sum of up to 128 exact products is within
128 u S_b in any order, its scales' product, the multiplication and the addition of the B blocks (up to 16 parts are joined) round
(B + 20) u S: 1.13 ((min(d, 128) + B + 24) u S + 4 u |bias|) + 12 u |act| + 2 u |out| with what bias, activation and
residual add (1.13 the activations' largest slope), and for bf16 2^-8 |out| more.  More than 16 rows with a bf16 output may go
through the matrix cores' 8-bit products, which cut each of eight neighbouring products off at 2^-13 of the largest one: less than
7 * 2^-13 max|x_i| max|w_i| a group, scaled with its block, and in the mean square four times 7 / 3 (2^-13 max max)^2 a group.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
import test_gpu_project as P
from gpu_util import dev

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def over(n, m=128):
    return -(-n // m)


def spread(scales, block_rows, rows, d):
    return scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :d]


def check_quantized(x, out, scales, block_rows):
    rows, d = x.shape
    xd = x.double()
    padded = torch.nn.functional.pad(xd.abs(), (0, over(d) * 128 - d, 0, over(rows, block_rows) * block_rows - rows))
    top = padded.view(over(rows, block_rows), block_rows, over(d), 128).amax((1, 3))
    # (a tensor's quotient by a number is torch's product with the reciprocal; 64 bits rounded to f32 are the f32 quotient)
    want = (torch.where(top < 2.0 ** -116, torch.zeros_like(top), top) / torch.full_like(top, 448.0)).float()
    assert torch.equal(scales, want)
    wide = spread(scales, block_rows, rows, d)
    err = (out.double() * wide - xd).abs()
    bar = torch.maximum((2.0 ** -4 + 8 * U) * xd.abs(), 2.0 ** -10 * 1.0001 * wide) + 4 * U * xd.abs()
    zero = wide == 0
    assert bool((out.double()[zero] == 0).all())
    assert bool((err <= bar)[~zero].all()), float((err - bar)[~zero].max())


@pytest.mark.parametrize("rows, d", [(1, 1), (1, 128), (2, 129), (3, 1000), (61, 2560), (127, 127), (128, 128), (129, 257), (300, 640), (5, 5001),
                                     (1000, 72), (7, 33000)])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("pad, start", [(0, 0), (16, 16), (3, 1)])
def test_quantized_blocks(sampler, rows, d, xt, block_rows, pad, start):
    g = torch.Generator(device=dev()).manual_seed(rows * 7 + d)
    _, x = P._rows(g, rows, d, xt, pad, 3.0, start)
    x.mul_(torch.exp2(torch.randint(-20, 20, (1, d), generator=g, device=dev()).float()).to(x.dtype))
    buf, out = P._rows(g, rows, d, "e4m3", pad, 1.0, start)
    before = buf.clone()
    down = rows if block_rows == 1 else over(rows)
    wide = torch.full((down, over(d) + 3), -1.0, device=dev())
    scales = wide[:, : over(d)]
    torch.cuda.synchronize()
    sampler.quantize_blocks(x, out, scales)
    sampler.synchronize()
    check_quantized(x, out, scales.contiguous(), block_rows if rows > 1 else 1)
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, (rows, d), (d + pad, 1), start).fill_(False)
    assert torch.equal(buf.view(torch.uint8)[mask], before.view(torch.uint8)[mask])
    assert bool((wide[:, over(d):] == -1.0).all())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_blocks_of_zeros_tiny_values_and_what_is_not_finite(sampler, block_rows):
    rows, d = 128, 128 * 7 + 5
    x = torch.randn(rows, d, generator=torch.Generator(device=dev()).manual_seed(2), device=dev())
    x[:, :128] = 0.0
    x[:, 128:256] *= 2.0 ** -125
    x[5, 300] = float("nan")
    x[5, 400] = float("inf")
    x[:, 512:640] *= 2.0 ** -110
    x[:, 640:768] = 1e38
    out, scales = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(rows if block_rows == 1 else 1, 8, device=dev())
    torch.cuda.synchronize()
    sampler.quantize_blocks(x, out, scales)
    sampler.synchronize()
    q = out.float()
    assert bool((scales[:, :2] == 0).all()) and bool((q[:, :256] == 0).all())
    hit = slice(5, 6) if block_rows == 1 else slice(0, rows)
    at = slice(5, 6) if block_rows == 1 else slice(0, 1)
    assert bool(torch.isnan(scales[at, 2]).all()) and bool(torch.isnan(q[hit, 256:384]).all())
    assert bool(torch.isinf(scales[at, 3]).all()) and bool(torch.isnan(q[5, 400])) and bool((q[5, 384:400] == 0).all())
    keep = [r for r in range(rows) if r != 5] if block_rows == 1 else range(rows)
    check_quantized(x[keep][:, 512:].contiguous(), out[keep][:, 512:].contiguous(), scales[keep if block_rows == 1 else [0]][:, 4:].contiguous(), block_rows)


# ---- the product


def operands(g, rows, n, d, pad=0):
    """Values of every size within a block's range, scales of very different sizes, as strided matrices."""
    _, x = P._rows(g, rows, d, "e4m3", pad * 16, 20.0)
    _, w = P._rows(g, n, d, "e4m3", pad * 16, 20.0)
    xs = torch.exp2(torch.rand(rows, over(d) + pad, generator=g, device=dev()) * 8 - 8)[:, : over(d)]
    ws = torch.exp2(torch.rand(over(n), over(d) + 2 * pad, generator=g, device=dev()) * 8 - 8)[:, : over(d)] / math.sqrt(d)
    return x, xs, w, ws


def formula(x, xs, w, ws, bias, act, residual):
    (rows, d), n = x.shape, w.shape[0]
    xd, wd = x.double() * spread(xs, 1, rows, d), w.double() * spread(ws, 128, n, d)
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    a = P._act(xd @ wd.T + b, act)
    out = a if residual is None else a + residual.double()
    tol = 1.13 * ((min(d, 128) + over(d) + 24) * U * (xd.abs() @ wd.abs().T) + 4 * U * b.abs()) + 12 * U * a.abs() + 2 * U * out.abs()
    return out, tol


def cut(x, xs, w, ws):
    """(bound, mean square) of what the 8-bit products cut off."""
    (rows, d), n = x.shape, w.shape[0]
    groups = lambda t: torch.nn.functional.pad(t.abs(), (0, -d % 8)).unflatten(1, (-1, 8)).amax(2)
    gx, gw = groups(x.double() * spread(xs, 1, rows, d)), groups(w.double() * spread(ws, 128, n, d))
    return 7 * 2.0 ** -13 * (gx @ gw.T), 7 / 3 * 2.0 ** -26 * (gx.square() @ gw.square().T)


def run(sampler, rows, n, d, out_dtype, act="none", bias=None, residual=None, pad=0, start=0, seed=0):
    g = torch.Generator(device=dev()).manual_seed(rows * 131 + n * 7 + d + seed)
    x, xs, w, ws = operands(g, rows, n, d, pad)
    b = None if bias is None else torch.randn(n, generator=g, device=dev()).to(DT[bias])
    res = None if residual is None else P._rows(g, rows, n, residual, start)[1]
    buf, out = P._rows(g, rows, n, out_dtype, start, 1.0, start)
    before = buf.clone()
    want, tol = formula(x, xs, w, ws, b, act, res)
    torch.cuda.synchronize()
    sampler.project_blocks(x, xs, w, ws, out, bias=b, activation=act, residual=res)
    sampler.synchronize()
    P._check(out, want, tol, cut(x, xs, w, ws) if out_dtype == "bf16" and rows > 16 else None)
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, (rows, n), (n + start, 1), start).fill_(False)
    bits = torch.int16 if out_dtype == "bf16" else torch.int32
    assert torch.equal(buf.view(bits)[mask], before.view(bits)[mask])


# rows and outputs around every tile's edges, one row to many
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 100, 128, 129, 300])
@pytest.mark.parametrize("n", [1, 3, 16, 127, 128, 129, 1000])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_shapes(sampler, rows, n, out):
    run(sampler, rows, n, 528, out)


@pytest.mark.parametrize("rows", [1, 17, 40, 70, 200])
@pytest.mark.parametrize("d", [16, 112, 128, 144, 256, 384, 1040, 2048, 4096 + 16, 8208, 128 * 67, 128 * 130 + 64])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_depths(sampler, rows, d, out):
    run(sampler, rows, 200, d, out)


def test_a_run_of_blocks_longer_than_a_wave_holds(sampler):
    """65 lines of weights' scales and more for one wave, in one part of d: 8 waves, 16 rows."""
    run(sampler, 3, 32, 128 * 8 * 65 + 16, "f32")
    run(sampler, 40, 16, 128 * 8 * 65 + 16, "f32")


@pytest.mark.parametrize("rows", [3, 30, 130, 260])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("bias, residual, out", [("f32", "bf16", "bf16"), ("bf16", "f32", "f32"), (None, "f32", "bf16"), ("f32", None, "f32")])
def test_epilogues(sampler, rows, act, bias, residual, out):
    run(sampler, rows, 333, 640, out, act, bias, residual)


@pytest.mark.parametrize("rows", [5, 90, 400])
@pytest.mark.parametrize("pad, start", [(1, 1), (3, 2), (0, 5)])
def test_strides_and_odd_starts(sampler, rows, pad, start):
    run(sampler, rows, 259, 1040, "bf16", "silu", "f32", "bf16", pad, start)
    run(sampler, rows, 259, 1040, "f32", "silu", "bf16", "f32", pad, start)


@pytest.mark.parametrize("rows, n, d", [(300, 4096, 1024), (2048, 2048, 512), (1000, 3000, 2064), (4100, 1030, 272), (64, 20000, 512), (100, 10007, 1024)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_larger(sampler, rows, n, d, out):
    run(sampler, rows, n, d, out, "silu", "f32", "bf16", 0, 1)


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("rows, n, d", [(20, 40, 144), (130, 129, 4112), (257, 300, 1040), (500, 513, 8208), (260, 260, 128), (300, 700, 128 * 66)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_each_tile(monkeypatch, tile, rows, n, d, out):
    monkeypatch.setenv("LILY_SAMPLER_PROJECT", str(tile))
    s = LS.Sampler(0)
    run(s, rows, n, d, out, "gelu", "bf16", "bf16", 1, 3)
    run(s, rows, n, d, out)
    s.close()


@pytest.mark.parametrize("lines", [1, 2, 3, 4, 8, 9, 17, 63, 64, 65, 129])
@pytest.mark.parametrize("rows, n", [(1, 1), (255, 257), (256, 512), (600, 300)])
def test_whole_lines_of_the_largest_tile(monkeypatch, rows, n, lines):
    """Stages that follow each other in two places of shared memory, eight stages' scales, sixty-four stages' scales of the weights."""
    monkeypatch.setenv("LILY_SAMPLER_PROJECT", "256")
    s = LS.Sampler(0)
    run(s, rows, n, 128 * lines, "bf16")
    run(s, rows, n, 128 * lines, "bf16", "silu", "f32", "bf16", 1, 3)
    s.close()


@pytest.mark.parametrize("rows", [4, 40, 300])
def test_scales_of_zero_infinite_scales_and_values_that_are_not_finite(sampler, rows):
    g = torch.Generator(device=dev()).manual_seed(8)
    n, d = 300, 640
    x, xs, w, ws = operands(g, rows, n, d)
    xs[1, :] = 0.0                       # a row of zeros, whatever its codes
    ws[1, 2] = 0.0                       # a block of weights that adds nothing
    xs[2, 3] = float("inf")
    x[2, 3 * 128:4 * 128] = 1.0
    w[:, 3 * 128:4 * 128] = 1.0
    x.view(torch.uint8)[3, 70] = 0x7f    # a NaN
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.empty(rows, n, dtype=dtype, device=dev())
        torch.cuda.synchronize()
        sampler.project_blocks(x, xs, w, ws, out)
        sampler.synchronize()
        assert bool((out[1] == 0).all())
        assert bool(torch.isinf(out[2]).all()) and bool(torch.isnan(out[3]).all())
        fine = [r for r in range(rows) if r not in (2, 3)]
        want, tol = formula(x[fine], xs[fine], w, ws, None, "none", None)
        P._check(out[fine], want, tol, cut(x[fine], xs[fine], w, ws) if dtype == torch.bfloat16 and rows > 16 else None)


def test_in_place_of_the_residual_and_the_same_bits_again(sampler):
    g = torch.Generator(device=dev()).manual_seed(3)
    for rows in (7, 77, 500):
        x, xs, w, ws = operands(g, rows, 384, 1024)
        res = torch.randn(rows, 384, generator=g, device=dev()).bfloat16()
        want, tol = formula(x, xs, w, ws, None, "silu", res)
        first, out = torch.empty_like(res), res.clone()
        torch.cuda.synchronize()
        sampler.project_blocks(x, xs, w, ws, first, activation="silu", residual=res)
        sampler.project_blocks(x, xs, w, ws, out, activation="silu", residual=out)
        sampler.synchronize()
        P._check(out, want, tol, cut(x, xs, w, ws) if rows > 16 else None)
        assert torch.equal(first, out)


def test_a_quantized_matrix_multiplied(sampler):
    """What lily_quantize_blocks leaves of rows and weights, multiplied, is the product of the matrices within what eight bits hold:
    each operand within 2^-4 of itself or 2^-10 of its block's largest value / 448."""
    g = torch.Generator(device=dev()).manual_seed(6)
    rows, n, d = 130, 500, 2000
    a, b = torch.randn(rows, d, generator=g, device=dev()), torch.randn(n, d, generator=g, device=dev()) / math.sqrt(d)
    x, w = (torch.empty(t.shape, dtype=torch.float8_e4m3fn, device=dev()) for t in (a, b))
    xs, ws = torch.empty(rows, over(d), device=dev()), torch.empty(over(n), over(d), device=dev())
    out = torch.empty(rows, n, device=dev())
    torch.cuda.synchronize()
    sampler.quantize_blocks(a, x, xs)
    sampler.quantize_blocks(b, w, ws)
    sampler.project_blocks(x, xs, w, ws, out)
    sampler.synchronize()
    want, tol = formula(x, xs, w, ws, None, "none", None)
    P._check(out, want, tol)
    # independent roundings, evenly spread over half a step (2^-4 at most): 2^-4 / sqrt(3) each, sqrt(2) of it together
    exact = a.double() @ b.double().T
    assert float((out.double() - exact).norm() / exact.norm()) < 2.0 ** -4 * math.sqrt(2.0 / 3.0)


@pytest.mark.parametrize("rows, n, d", [(4, 300, 512), (100, 300, 4096)])
def test_a_captured_graph(rows, n, d):
    stream = torch.cuda.Stream()
    s = LS.Sampler(0, stream)
    g = torch.Generator(device=dev()).manual_seed(4)
    a = torch.randn(rows, d, generator=g, device=dev())
    _, _, w, ws = operands(g, 1, n, d)
    x, xs, out = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(rows, over(d), device=dev()), torch.empty(rows, n, device=dev())

    def step():
        s.quantize_blocks(a, x, xs)
        s.project_blocks(x, xs, w, ws, out)

    torch.cuda.synchronize()
    step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for turn in range(4):
        a.copy_(torch.randn(rows, d, generator=g, device=dev()) * (turn + 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        step()
        s.synchronize()
        assert torch.equal(replayed, out)
        P._check(out, *formula(x, xs, w, ws, None, "none", None))
    s.close()


def test_what_the_python_mirror_refuses(sampler):
    x, w = (torch.zeros(r, 256, dtype=torch.float8_e4m3fn, device=dev()) for r in (4, 300))
    xs, ws, out = torch.zeros(4, 2, device=dev()), torch.zeros(3, 2, device=dev()), torch.zeros(4, 300, device=dev())
    for bad in (dict(x=x.float()), dict(weight=w.bfloat16()), dict(x_scales=xs[:, :1]), dict(weight_scales=ws[:2]), dict(x_scales=xs.bfloat16()),
                dict(out=out[:3]), dict(out=out.cpu()), dict(activation="tanh"), dict(x=x[:, 8:]), dict(weight=w[:, :128])):
        kw = dict(x=x, x_scales=xs, weight=w, weight_scales=ws, out=out)
        kw.update(bad)
        with pytest.raises(LS.SamplerError):
            sampler.project_blocks(**kw)
    for bad in (dict(x=w), dict(out=out[:, :256]), dict(scales=xs[:3]), dict(scales=xs[:, :1]), dict(scales=xs.bfloat16())):
        kw = dict(x=torch.zeros(4, 256, device=dev()), out=x, scales=xs)
        kw.update(bad)
        with pytest.raises(LS.SamplerError):
            sampler.quantize_blocks(**kw)
