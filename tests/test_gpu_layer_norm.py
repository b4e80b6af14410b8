"""The layer norm (lily_layer_norm) and its backward pass (lily_layer_norm_backward) against their formulas in 64 bits.

Bars, derived from the arithmetic (u = 2^-24, half a step of f32; A the mean of |h|, x = (h - mean) rstd):
  * h: bit-exact (one f32 addition, one rounding to the stream's type);
  * mean: at most 8 + 4 + 8 + 16 additions one after the other (a piece, pieces, a wave, waves) and a division: dm = 38 u A;
  * rstd: the squares' sum takes up to 32 + 8 + 16 steps, its differences are rounded once (2 u in a square) and lie dm off, which adds dm^2 to
    the variance and nothing of first order (differences from a mean cancel); halved by the root; division, + eps, root and
    reciprocal 4 u: (40 u + dm^2 rstd^2) relative;
  * y in f32: |x w| (48 u + dm^2 rstd^2) + dm rstd |w| + 4 u (|b| + |y|);
  * bf16: half a step more, 2^-8 relative;
  * E4M3: half a step of q (2^-4 relative, half of 2^-9 scale below the normal codes), 4 u for the product with 448 / max; a scale
    is as far off as the value it is made of.
Backward, of given mean and rstd: x is off by 2 u |x|, g = grad w by u |g|; a row's sums take up to 64 steps, so their means are
off by 66 u mean|g| and 70 u mean|g x|; then
    rstd (3 u |g| + 68 u mean|g| + 72 u |x| mean|g x| + 5 u |x mean(g x)|) + 3 u |grad_x|, half a step of bf16 on top;
sums over the rows in any order: (rows + 8) u sum|grad x| and (rows + 8) u sum|grad|.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
EPS = 1e-5


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
    yield s
    s.close()


def matrix(rng, rows, d, dtype, pad=0, scale=1.0, start=0, mean=0.0):
    """(buffer, [rows, d] of it), `pad` elements wider, whose other elements hold NaN."""
    buf = torch.full((rows * (d + pad) + start + 8,), float("nan"), dtype=DT[dtype], device=dev())
    m = torch.as_strided(buf, (rows, d), (d + pad, 1), start)
    m.copy_(torch.from_numpy((rng.normal(0, scale, (rows, d)) + mean).astype(np.float32)))
    return buf, m


def untouched(buf, before, rows, d, pad, start):
    """What lies between and behind the rows is as it was."""
    mask = torch.ones(buf.shape, dtype=torch.bool, device=buf.device)
    torch.as_strided(mask, (rows, d), (d + pad, 1), start).fill_(False)
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[buf.element_size()]
    return torch.equal(buf.view(bits)[mask], before.view(bits)[mask])


def forward(x, residual, stream, weight, bias, eps=EPS):
    """(h, y, its bar, mean, its bar, rstd, its relative bar)."""
    h = x.float()
    if residual is not None:
        h = (h + residual.float()).to(DT[stream])
    hd = h.double()
    mean = hd.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((hd - mean).square().mean(1, keepdim=True) + eps)
    w = weight.double() if weight is not None else torch.ones(x.shape[1], device=x.device, dtype=torch.float64)
    b = bias.double() if bias is not None else torch.zeros(x.shape[1], device=x.device, dtype=torch.float64)
    off = (hd - mean) * rstd
    y = off * w + b
    dm = 38 * U * hd.abs().mean(1, keepdim=True)
    tol = (off * w).abs() * (48 * U + (dm * rstd) ** 2) + dm * rstd * w.abs() + 4 * U * (b.abs() + y.abs())
    return h, y, tol, mean[:, 0], dm[:, 0], rstd[:, 0], (40 * U + (dm * rstd) ** 2)[:, 0]


def check_out(y, tol, out, scales, dtype):
    if dtype != "e4m3":
        err = (out.double() - y).abs()
        if dtype == "bf16":
            tol = tol + 2.0 ** -8 * (y.abs() + tol)
        assert bool((err <= tol + 1e-300).all()), float((err - tol).max())
        return
    rows, d = y.shape
    blocks = 1 if scales.dim() == 1 else -(-d // 128)
    size = d if scales.dim() == 1 else 128
    pad = (0, blocks * size - d)
    top = torch.nn.functional.pad(y.abs(), pad).view(rows, blocks, size).amax(2)
    far = torch.nn.functional.pad(tol, pad).view(rows, blocks, size).amax(2)
    sc = scales.double().view(rows, blocks)
    assert bool(((sc * 448.0 - top).abs() <= far + 2 * U * top).all())
    wide = sc.repeat_interleave(size, 1)[:, :d]
    err = (out.double() * wide - y).abs()
    bar = torch.maximum((2.0 ** -4 + 8 * U) * (y.abs() + tol), 2.0 ** -10 * 1.0001 * wide) + tol
    assert bool((err <= bar).all()), float((err - bar).max())


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 63), (5, 64), (1, 4096), (61, 2560), (4, 5120), (3, 8193), (2, 16384), (2, 16392),
          (1, 32768), (2, 32767), (300, 520), (1, 511), (2, 513), (7, 129)]


@pytest.mark.parametrize("rows, d", SHAPES)
@pytest.mark.parametrize("xt, st, ot, wt, bt", [("bf16", "bf16", "bf16", "bf16", True), ("bf16", "f32", "e4m3", "f32", True),
                                                ("f32", "f32", "f32", "f32", True), ("f32", "bf16", "blocks", "bf16", True),
                                                ("bf16", None, "blocks", "bf16", False), ("f32", None, "bf16", None, False)])
@pytest.mark.parametrize("pad, start", [(0, 0), (8, 8), (3, 1)])
def test_against_the_formula(sampler, rows, d, xt, st, ot, wt, bt, pad, start):
    rng = np.random.default_rng(rows * 1000 + d + pad)
    _, x = matrix(rng, rows, d, xt, pad, 2.0, start, 0.7)
    res = matrix(rng, rows, d, st, pad, 3.0, start)[1] if st else None
    summed = matrix(rng, rows, d, st, pad, 1.0, start)[1] if st else None
    vector = lambda: torch.from_numpy(rng.normal(0, 1, d).astype(np.float32)).to(dev()).to(DT[wt])
    weight, bias = vector() if wt else None, vector() if bt else None
    blocks, ot = ot == "blocks", "e4m3" if ot == "blocks" else ot
    out_buf, out = matrix(rng, rows, d, ot, pad, 1.0, start)
    before = out_buf.clone()
    scales_buf = torch.full((rows, -(-d // 128) + 2), -1.0, device=dev())
    scales = None if ot != "e4m3" else scales_buf[:, :-2] if blocks else torch.full((rows,), -1.0, device=dev())
    mean, rstd = torch.empty(rows, device=dev()), torch.empty(rows, device=dev())
    h, y, tol, m, dm, r, dr = forward(x, res, st, weight, bias)
    torch.cuda.synchronize()
    sampler.layer_norm(x, weight, bias, out, eps=EPS, residual=res, summed=summed, scales=scales, mean=mean, rstd=rstd)
    sampler.synchronize()
    if st:
        assert torch.equal(summed, h)
    assert bool(((mean.double() - m).abs() <= dm + 1e-300).all())
    assert bool(((rstd.double() - r).abs() <= dr * r).all())
    check_out(y, tol, out, scales, ot)
    assert untouched(out_buf, before, rows, d, pad, start) and bool((scales_buf[:, -2:] == -1.0).all())


@pytest.mark.parametrize("d", [4096, 1001])
@pytest.mark.parametrize("where", ["sum is residual", "sum is x", "out is x", "out is residual, sum is x"])
def test_in_place(sampler, d, where):
    rng = np.random.default_rng(d)
    x, res = matrix(rng, 9, d, "bf16")[1], matrix(rng, 9, d, "bf16")[1]
    w = torch.from_numpy(rng.normal(0, 1, d).astype(np.float32)).to(dev())
    h, y, tol, *_ = forward(x, res, "bf16", w, None)
    summed, out = torch.empty_like(x), torch.empty_like(x)
    summed = res if where == "sum is residual" else x if "sum is x" in where else summed
    out = x if where == "out is x" else res if "out is residual" in where else out
    torch.cuda.synchronize()
    sampler.layer_norm(x, w, None, out, eps=EPS, residual=res, summed=summed)
    sampler.synchronize()
    assert torch.equal(summed.float(), h.float())
    check_out(y, tol, out, None, "bf16")


def test_constant_rows_far_means_and_rows_that_are_not_finite(sampler):
    """A variance of zero; a mean that is 2^12 deviations away; NaN and infinity in a row and in none of its neighbours."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.normal(0, 1, (6, 640)).astype(np.float32)).to(dev())
    x[0] = 3.0
    x[1] += 4096.0
    x[2, 600] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 0.0
    out, plain = torch.empty(6, 640, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(6, 640, device=dev())
    scales, mean, rstd = torch.empty(6, 5, device=dev()), torch.empty(6, device=dev()), torch.empty(6, device=dev())
    torch.cuda.synchronize()
    sampler.layer_norm(x, None, None, out, eps=EPS, scales=scales, mean=mean, rstd=rstd)
    sampler.layer_norm(x, None, None, plain, eps=EPS)
    sampler.synchronize()
    _, y, tol, *_ = forward(x, None, None, None, None)
    fine = [0, 1, 4, 5]
    check_out(y[fine], tol[fine], plain[fine], None, "f32")
    assert bool((out[[0, 4]].float() == 0).all()) and bool((scales[[0, 4]] == 0).all())
    check_out(y[[1, 5]], tol[[1, 5]], out[[1, 5]], scales[[1, 5]], "e4m3")
    assert bool(torch.isnan(plain[2:4]).all()) and bool(torch.isnan(scales[2:4]).all()) and bool(torch.isnan(out[2:4].float()).all())


def test_blocks_of_very_different_sizes(sampler):
    """Each block has the scale of its own largest value, zeros below 2^-116."""
    d = 1000
    x = torch.randn(4, d, device=dev(), generator=torch.Generator(device=dev()).manual_seed(1))
    w = torch.exp2(torch.arange(8, device=dev(), dtype=torch.float32) * -17.0).repeat_interleave(128)[:d]   # 1 to 2^-119
    out, scales = torch.empty(4, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(4, 8, device=dev())
    torch.cuda.synchronize()
    sampler.layer_norm(x, w, None, out, eps=EPS, scales=scales)
    sampler.synchronize()
    _, y, tol, *_ = forward(x, None, None, w, None)
    check_out(y[:, :896], tol[:, :896], out[:, :896], scales[:, :7], "e4m3")
    assert bool((scales[:, 7] == 0).all()) and bool((out[:, 896:].float() == 0).all())


# ---- the backward pass


def backward(grad, h, mean, rstd, weight, past):
    """(grad_x, its bar, grad_weight, its bar, grad_bias, its bar)."""
    dy, r = grad.double(), rstd.double()[:, None]
    x = (h.double() - mean.double()[:, None]) * r
    g = dy * weight.double() if weight is not None else dy
    mg, mgx = g.mean(1, keepdim=True), (g * x).mean(1, keepdim=True)
    gx = r * (g - mg - x * mgx)
    tol = r * (3 * U * g.abs() + 68 * U * g.abs().mean(1, keepdim=True) + 72 * U * x.abs() * (g * x).abs().mean(1, keepdim=True)
               + 5 * U * (x * mgx).abs()) + 3 * U * gx.abs()
    if past is not None:
        gx = gx + past.double()
        tol = tol + U * gx.abs()
    n = (grad.shape[0] + 8) * U
    return gx, tol, (dy * x).sum(0), n * (dy * x).abs().sum(0), dy.sum(0), n * dy.abs().sum(0)


def statistics(h):
    hd = h.double()
    return hd.mean(1).float(), (1.0 / torch.sqrt(hd.var(1, unbiased=False) + EPS)).float()


def check_grad(got, want, tol):
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    err = (got.double() - want).abs()
    assert bool((err <= tol + 1e-300).all()), float((err - tol).max())


GRAD_SHAPES = SHAPES + [(1000, 64), (700, 1000), (33, 9000), (2100, 256), (9, 20000)]


@pytest.mark.parametrize("rows, d", GRAD_SHAPES)
@pytest.mark.parametrize("gt, ht, wt, ot, with_past", [("bf16", "bf16", "bf16", "bf16", True), ("f32", "f32", "f32", "f32", False),
                                                      ("bf16", "f32", None, "f32", True), ("f32", "bf16", "f32", "bf16", False)])
@pytest.mark.parametrize("pad, start", [(0, 0), (3, 1)])
def test_backward_against_the_formula(sampler, rows, d, gt, ht, wt, ot, with_past, pad, start):
    rng = np.random.default_rng(rows * 1000 + d + pad)
    grad, h = matrix(rng, rows, d, gt, pad, 0.01, start)[1], matrix(rng, rows, d, ht, pad, 2.0, start, 0.5)[1]
    mean, rstd = statistics(h)
    weight = torch.from_numpy(rng.normal(0, 1, d).astype(np.float32)).to(dev()).to(DT[wt]) if wt else None
    past = matrix(rng, rows, d, ot, pad, 0.02, start)[1] if with_past else None
    buf, gx = matrix(rng, rows, d, ot, pad, 1.0, start)
    before = buf.clone()
    gw, gb = torch.full((d,), 7.0, device=dev()), torch.full((d,), 7.0, device=dev())
    want = backward(grad, h, mean, rstd, weight, past)
    torch.cuda.synchronize()
    sampler.layer_norm_backward(grad, h, mean, rstd, weight, grad_x=gx, grad_weight=gw, grad_bias=gb, past=past)
    sampler.synchronize()
    check_grad(gx, want[0], want[1])
    check_grad(gw, want[2], want[3])
    check_grad(gb, want[4], want[5])
    assert untouched(buf, before, rows, d, pad, start)
    again, first = torch.empty_like(gw), (gw.clone(), gb.clone(), gx.clone())
    sampler.layer_norm_backward(grad, h, mean, rstd, weight, grad_x=gx, grad_weight=again, grad_bias=gb, past=past)
    sampler.synchronize()
    assert torch.equal(again, first[0]) and torch.equal(gb, first[1]) and torch.equal(gx, first[2])   # the same bits again
    # only some of the outputs, and added to what is there
    sampler.layer_norm_backward(grad, h, mean, rstd, weight, grad_weight=gw, accumulate=True)
    sampler.layer_norm_backward(grad, h, mean, rstd, weight, grad_bias=gb)
    alone = torch.empty_like(gx)
    sampler.layer_norm_backward(grad, h, mean, rstd, weight, grad_x=alone, past=past)
    sampler.synchronize()
    check_grad(gw, 2 * want[2], 2 * want[3] + 2 * U * want[2].abs())
    check_grad(gb, want[4], want[5])
    check_grad(alone, want[0], want[1])


@pytest.mark.parametrize("d", list(range(8, 25)) + list(range(1025, 1032)) + list(range(8193, 8201)) + [12345, 16383])
@pytest.mark.parametrize("gt, ht, ot", [("bf16", "bf16", "bf16"), ("f32", "f32", "f32"), ("f32", "bf16", "f32"), ("bf16", "f32", "bf16")])
@pytest.mark.parametrize("pad, start", [(0, 0), (5, 1)])
def test_backward_where_a_row_ends_in_every_place_of_a_piece(sampler, d, gt, ht, ot, pad, start):
    """In place of its operands too: the piece that a row ends in is read with elements of the one before."""
    rng = np.random.default_rng(d + pad)
    rows = 777 if d < 8000 else 300
    grad, h = matrix(rng, rows, d, gt, pad, 1.0, start)[1], matrix(rng, rows, d, ht, pad, 2.0, start, 0.5)[1]
    past = matrix(rng, rows, d, ot, pad, 1.0, start)[1]
    mean, rstd = statistics(h)
    weight = torch.from_numpy(rng.normal(0, 1, d).astype(np.float32)).to(dev())
    want = backward(grad, h, mean, rstd, weight, past)
    for place in ("past", "grad") if gt == ot else ("past",):
        t = dict(grad=grad.clone(), past=past.clone())
        gx = t[place]
        gw, gb = torch.empty(d, device=dev()), torch.empty(d, device=dev())
        torch.cuda.synchronize()
        sampler.layer_norm_backward(t["grad"], h, mean, rstd, weight, grad_x=gx, grad_weight=gw, grad_bias=gb, past=t["past"])
        sampler.synchronize()
        for got, k in ((gx, 0), (gw, 2), (gb, 4)):
            check_grad(got, want[k], want[k + 1])


@pytest.mark.parametrize("rows, d", [(5, 640), (40, 1001), (3, 12000)])
@pytest.mark.parametrize("where", ["grad", "h", "past"])
def test_backward_in_place(sampler, rows, d, where):
    rng = np.random.default_rng(d + rows)
    t = dict(grad=matrix(rng, rows, d, "bf16")[1], h=matrix(rng, rows, d, "bf16", 0, 2.0)[1], past=matrix(rng, rows, d, "bf16")[1])
    mean, rstd = statistics(t["h"])
    w = torch.ones(d, device=dev())
    want = backward(t["grad"], t["h"], mean, rstd, w, t["past"])
    gw, gb = torch.empty(d, device=dev()), torch.empty(d, device=dev())
    torch.cuda.synchronize()
    sampler.layer_norm_backward(t["grad"], t["h"], mean, rstd, w, grad_x=t[where], grad_weight=gw, grad_bias=gb, past=t["past"])
    sampler.synchronize()
    check_grad(t[where], want[0], want[1])
    check_grad(gw, want[2], want[3])
    check_grad(gb, want[4], want[5])


def test_the_backward_pass_is_the_forward_pass_differentiated(sampler):
    """Central differences of the forward formula in 64 bits, of a random linear function of the outputs: their own error is some
    step^2 = 1e-10 and 1e-16 / step = 1e-11 of values of order one."""
    g = torch.Generator(device=dev()).manual_seed(9)
    rows, d = 3, 40
    x, w, b, dy = (torch.randn(*shape, generator=g, device=dev()) for shape in ((rows, d), (d,), (d,), (rows, d)))

    def loss(x, w, b):
        mean = x.mean(1, keepdim=True)
        return ((((x - mean) / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPS)) * w + b) * dy.double()).sum()

    def differences(i):
        args, step = [x.double(), w.double(), b.double()], 1e-5
        out = torch.empty_like(args[i])
        for at in range(args[i].numel()):
            keep = args[i].view(-1)[at].clone()
            args[i].view(-1)[at] = keep + step
            up = loss(*args)
            args[i].view(-1)[at] = keep - step
            out.view(-1)[at] = (up - loss(*args)) / (2 * step)
            args[i].view(-1)[at] = keep
        return out

    mean, rstd, out = torch.empty(rows, device=dev()), torch.empty(rows, device=dev()), torch.empty(rows, d, device=dev())
    gx, gw, gb = torch.empty(rows, d, device=dev()), torch.empty(d, device=dev()), torch.empty(d, device=dev())
    torch.cuda.synchronize()
    sampler.layer_norm(x, w, b, out, eps=EPS, mean=mean, rstd=rstd)
    sampler.layer_norm_backward(dy, x, mean, rstd, w, grad_x=gx, grad_weight=gw, grad_bias=gb)
    sampler.synchronize()
    # (mean and rstd were rounded to f32 on the way: some 50 u)
    for got, want in ((gx, differences(0)), (gw, differences(1)), (gb, differences(2))):
        assert float((got.double() - want).abs().max()) <= 2e-5 * max(1.0, float(want.abs().max()))


def test_captured_graphs_replayed_over_changing_inputs():
    stream = torch.cuda.Stream()
    s = LS.Sampler(0, stream)
    rng = np.random.default_rng(5)
    rows, d = 70, 2560
    x, dy = matrix(rng, rows, d, "bf16")[1], matrix(rng, rows, d, "bf16")[1]
    w, b = (torch.from_numpy(rng.normal(1, 0.1, d).astype(np.float32)).to(dev()) for _ in range(2))
    out, scales = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=dev()), torch.empty(rows, d // 128, device=dev())
    mean, rstd, gx = torch.empty(rows, device=dev()), torch.empty(rows, device=dev()), torch.empty_like(x)
    gw, gb = torch.empty(d, device=dev()), torch.empty(d, device=dev())

    def step():
        s.layer_norm(x, w, b, out, eps=EPS, scales=scales, mean=mean, rstd=rstd)
        s.layer_norm_backward(dy, x, mean, rstd, w, grad_x=gx, grad_weight=gw, grad_bias=gb)

    outputs = (out.view(torch.uint8), scales, mean, rstd, gx, gw, gb)
    torch.cuda.synchronize()
    step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for turn in range(4):
        x.copy_(torch.from_numpy(rng.normal(0, 1 + turn, (rows, d)).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outputs]
        for t in outputs:
            t.zero_()
        torch.cuda.synchronize()
        step()
        s.synchronize()
        assert all(torch.equal(a, t) for a, t in zip(replayed, outputs))
    s.close()


def test_what_the_python_mirror_refuses(sampler):
    x, w = torch.zeros(2, 64, device=dev()), torch.ones(64, device=dev())
    good, row = torch.empty(2, 64, device=dev()), torch.empty(2, device=dev())
    for bad in (dict(x=x.half()), dict(x=x.cpu()), dict(x=x[:, ::2]), dict(out=good[:1]), dict(weight=w[:32]), dict(bias=w.bfloat16()),
                dict(residual=x[:1]), dict(summed=x), dict(residual=x, summed=x.bfloat16()), dict(out=good.to(torch.float8_e4m3fn)),
                dict(scales=row), dict(eps=-1.0), dict(mean=row.double()), dict(rstd=row[:1])):
        kw = dict(x=x, weight=w, bias=w, out=good)
        kw.update(bad)
        with pytest.raises(LS.SamplerError):
            sampler.layer_norm(**kw)
    for bad in (dict(grad=x.half()), dict(h=x[:1]), dict(mean=None), dict(rstd=row[:1]), dict(weight=w[:3]), dict(grad_x=None), dict(past=x.bfloat16()),
                dict(grad_weight=w.bfloat16()), dict(grad_bias=w[:5])):
        kw = dict(grad=x, h=good, mean=row, rstd=row.clone(), weight=w, grad_x=torch.empty_like(x))
        kw.update(bad)
        with pytest.raises(LS.SamplerError):
            sampler.layer_norm_backward(**kw)


@pytest.mark.parametrize("rows, d", [(1, 140), (3, 8), (3, 2560), (16, 64), (17, 64), (2, 8191), (300, 1001), (5, 10000)])
@pytest.mark.parametrize("leave", [None, "grad_weight", "grad_bias"])
def test_all_gradients_added_to_what_is_there(sampler, rows, d, leave):
    """With one part of the rows and with several; what is not asked for is not touched."""
    rng = np.random.default_rng(rows * 7 + d)
    grad, h = matrix(rng, rows, d, "bf16")[1], matrix(rng, rows, d, "bf16", 0, 2.0)[1]
    mean, rstd = statistics(h)
    gx = torch.empty(rows, d, dtype=torch.bfloat16, device=dev())
    sums = dict(grad_weight=torch.full((d,), 3.0, device=dev()), grad_bias=torch.full((d,), -2.0, device=dev()))
    want = backward(grad, h, mean, rstd, None, None)
    torch.cuda.synchronize()
    given = {k: v for k, v in sums.items() if k != leave}
    sampler.layer_norm_backward(grad, h, mean, rstd, None, grad_x=gx, accumulate=True, **given)
    sampler.synchronize()
    check_grad(gx, want[0], want[1])
    for name, k, start in (("grad_weight", 2, 3.0), ("grad_bias", 4, -2.0)):
        if name == leave:
            assert bool((sums[name] == start).all())
        else:
            check_grad(sums[name], want[k] + start, want[k + 1] + U * (want[k].abs() + abs(start)))
