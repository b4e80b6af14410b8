"""The operators that train and serve a draft head in front of a large vocabulary, as cases that can be timed and compared.

`kind` says which operator a case is:
  layer         the residual's addition and the layer norm, in bf16, f32 or 8 bits with a scale for each row or each 128 elements
  layer_grad    its backward pass: the gradient of the rows (with what reaches them past the norm) and of weight and bias
  quantize      rows or weights in 8-bit floats with a scale for each 128 elements or each 128 x 128
  project       the matrix product of two such operands, with bias, activation and residual
  distill       a student's loss against a teacher's top logits, and its gradient, in one call
  distill_grad  the gradient alone, from what the loss left
Sizes are those of the benchmark and the tests (vocabularies 151 936 and 248 320, widths 2 560, 4 096).
`own` false: elementary torch operations in 32 bits; true: the library's calls.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
VOCAB = 151_936
VOCAB_LARGE = 248_320
BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -116     # rows and blocks whose largest magnitude lies below: zeros, scale 0
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}

_program = {}          # the library and its sampler, opened once as a program does


def listed():
    return [
        # The norm of four conversations' decode step: the smallest call there is.
        dict(name="layer_decode_b4", kind="layer", rows=4, d=4096, x="bf16", stream="bf16", out="bf16", block=0, stats=0, pad=0),
        # Prefill: residual and norm on their way into a block-scaled product.
        dict(name="layer_blocks_b8192", kind="layer", rows=8192, d=4096, x="bf16", stream="bf16", out="e4m3", block=128,
             stats=0, pad=0),
        # A training step's backward over a ragged batch of the smaller width, everything in f32.
        dict(name="layer_grad_f32_b2049", kind="layer_grad", rows=2049, d=2560, grad="f32", h="f32", out="f32", past=0, pad=0),
        # Mixed precision training: the gradient of the residual stream joins on the way.
        dict(name="layer_grad_bf16_b16384", kind="layer_grad", rows=16384, d=4096, grad="bf16", h="bf16", out="bf16", past=1, pad=0),
        # A server's ragged decode batch, rows of a wider buffer.
        dict(name="quantize_rows_b61", kind="quantize", rows=61, d=2560, x="bf16", block_rows=1, pad=64),
        # A layer's weights laid out for serving.
        dict(name="quantize_weights", kind="quantize", rows=12288, d=4096, x="f32", block_rows=128, pad=0),
        # A head in 8-bit blocks, the default batch of four, f32 logits.
        dict(name="head_blocks_b4", kind="project", rows=4, n=VOCAB, d=4096, out="f32", bias=0, act="none", residual=0, pad=0),
        # A middle batch through an odd-sized layer, rows of a wider buffer.
        dict(name="layer_blocks_b100", kind="project", rows=100, n=10007, d=4096, out="bf16", bias=1, act="gelu_tanh",
             residual=0, pad=32),
        # Prefill through a wide layer: bound by the matrix cores.
        dict(name="prefill_blocks_b8192", kind="project", rows=8192, n=12288, d=4096, out="bf16", bias=0, act="none",
             residual=0, pad=0),
        # A short fine-tuning batch: 37 positions of f32 logits against what a draw kept (ids and probabilities), ragged lists.
        dict(name="distill_kept_b37", kind="distill", rows=37, vocab=VOCAB, x="f32", out="f32", k=20, teacher="probs", t="f32",
             rest=0, temperature=1.0, ragged=1, weights=0, pad=0),
        # A training step of the headline size in mixed precision: 64 teacher logits, the rest of the vocabulary as one outcome.
        dict(name="distill_rest_b2048", kind="distill", rows=2048, vocab=VOCAB, x="bf16", out="bf16", k=64, teacher="logits",
             t="bf16", rest=1, temperature=2.0, ragged=0, weights=1, pad=0),
        # The backward pass by itself over the large vocabulary, long lists, padded positions.
        dict(name="distill_grad_b300", kind="distill_grad", rows=300, vocab=VOCAB_LARGE, x="bf16", out="f32", k=1000,
             teacher="logits", t="f32", rest=1, temperature=1.0, ragged=1, weights=1, pad=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layer", "layer_grad", "quantize", "project", "project", "distill", "distill", "distill_grad"])
    pad = rng.choice([0, 0, 16, 32])
    if kind in ("layer", "layer_grad", "quantize"):
        rows = _log_int(rng, 1, 16384)
        d = _log_int(rng, 64, min(16384, 16384 * 4096 // rows))
        if kind == "layer":
            out = rng.choice(["bf16", "e4m3", "e4m3", "f32"])
            return dict(kind=kind, rows=rows, d=d, x=rng.choice(["bf16", "bf16", "f32"]),
                        stream=rng.choice(["none", "bf16", "bf16", "f32"]), out=out,
                        block=rng.choice([0, 128, 128]) if out == "e4m3" else 0, stats=rng.randrange(2), pad=rng.choice([0, 0, 8, 3]))
        if kind == "layer_grad":
            return dict(kind=kind, rows=rows, d=d, grad=rng.choice(["bf16", "bf16", "f32"]), h=rng.choice(["bf16", "bf16", "f32"]),
                        out=rng.choice(["bf16", "bf16", "f32"]), past=rng.randrange(2), pad=rng.choice([0, 0, 8, 3]))
        return dict(kind=kind, rows=rows, d=d, x=rng.choice(["bf16", "f32"]), block_rows=rng.choice([1, 128]),
                    pad=rng.choice([0, 0, 8, 3]))
    if kind == "project":
        rows = _log_int(rng, 1, 8192)
        n = _log_int(rng, 64, 16384)
        d = 16 * _log_int(rng, 8, 512)
        while rows * n * d > 8192 * 12288 * 4096:
            n = (n + 1) // 2
        return dict(kind=kind, rows=rows, n=n, d=d, out=rng.choice(["bf16", "bf16", "f32"]), bias=rng.randrange(2),
                    act=rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]), residual=rng.randrange(2), pad=pad)
    rows = _log_int(rng, 1, 2048)
    vocab = _log_int(rng, 8000, VOCAB_LARGE)
    while rows * vocab > 2048 * VOCAB:
        rows = (rows + 1) // 2
    return dict(kind=kind, rows=rows, vocab=vocab, x=rng.choice(["bf16", "bf16", "f32"]), out=rng.choice(["bf16", "f32"]),
                k=_log_int(rng, 1, 1024), teacher=rng.choice(["logits", "logits", "probs"]), t=rng.choice(["f32", "bf16"]),
                rest=rng.randrange(2), temperature=rng.choice([1.0, 1.0, 2.0, 0.7]), ragged=rng.randrange(3),
                weights=rng.randrange(2), pad=rng.choice([0, 0, 8, 3]))


# ------------------------------------------------------------------ inputs


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _rows_of(t, pad):
    """`t` as the leading columns of a wider buffer."""
    if not pad:
        return t
    wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=t.device)
    wide[:, : t.shape[1]] = t
    return wide[:, : t.shape[1]]


def _empty(rows, columns, dtype):
    return torch.empty(rows, columns, dtype=DTYPES[dtype], device=DEVICE)


def _hidden(g, rows, d, scale):
    """Hidden states: channels differ in size, a few by much; rows have a mean of their own."""
    return (scale * _normal(g, rows, d) * torch.exp(_normal(g, d)) + scale * _normal(g, rows, 1))


def _prepare_layer(c, g):
    rows, d = c["rows"], c["d"]
    st = dict(x=_rows_of(_hidden(g, rows, d, 0.3).to(DTYPES[c["x"]]), c["pad"]), weight=(1.0 + 0.2 * _normal(g, d)).to(torch.bfloat16),
              bias=(0.1 * _normal(g, d)).to(torch.bfloat16), residual=None, summed=None, scales=None, mean=None, rstd=None)
    if c["stream"] != "none":
        st["residual"] = _rows_of(_hidden(g, rows, d, 1.0).to(DTYPES[c["stream"]]), c["pad"])
        st["summed"] = _empty(rows, d, c["stream"])
    st["out"] = _empty(rows, d, c["out"])
    if c["out"] == "e4m3":
        st["scales"] = _empty(rows, (d + BLOCK - 1) // BLOCK, "f32") if c["block"] else torch.empty(rows, device=DEVICE)
    if c["stats"]:
        st["mean"], st["rstd"] = torch.empty(rows, device=DEVICE), torch.empty(rows, device=DEVICE)
    return st


def _prepare_layer_grad(c, g):
    rows, d = c["rows"], c["d"]
    h = _hidden(g, rows, d, 1.0).to(DTYPES[c["h"]])
    wide = h.double()
    st = dict(h=_rows_of(h, c["pad"]), mean=wide.mean(1).float(), rstd=(1.0 / torch.sqrt(wide.var(1, unbiased=False) + EPS)).float(),
              grad=_rows_of((1e-3 * _normal(g, rows, d)).to(DTYPES[c["grad"]]), c["pad"]),
              weight=(1.0 + 0.2 * _normal(g, d)).to(torch.bfloat16), past=None, grad_x=_empty(rows, d, c["out"]),
              grad_weight=torch.empty(d, device=DEVICE), grad_bias=torch.empty(d, device=DEVICE))
    if c["past"]:
        st["past"] = _rows_of((1e-3 * _normal(g, rows, d)).to(DTYPES[c["out"]]), c["pad"])
    return st


def _blocks(n, block):
    return (n + block - 1) // block


def _prepare_quantize(c, g):
    rows, d = c["rows"], c["d"]
    x = _hidden(g, rows, d, 1.0) if c["block_rows"] == 1 else _normal(g, rows, d) / math.sqrt(d)
    return dict(x=_rows_of(x.to(DTYPES[c["x"]]), c["pad"]), out=_empty(rows, d, "e4m3"),
                scales=_empty(_blocks(rows, c["block_rows"]), _blocks(d, BLOCK), "f32"))


def _in_blocks(t, block_rows):
    """(E4M3, scales) of a matrix, a scale for each block_rows x 128."""
    rows, d = t.shape
    p = torch.nn.functional.pad(t, (0, -d % BLOCK, 0, -rows % block_rows))
    p = p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // BLOCK, BLOCK)
    scales = p.abs().amax((1, 3)) / E4M3_MAX
    q = (p / scales[:, None, :, None].clamp_min(1e-30)).clamp(-E4M3_MAX, E4M3_MAX)
    return q.reshape(p.shape[0] * block_rows, -1)[:rows, :d].to(torch.float8_e4m3fn), scales


def _prepare_project(c, g):
    rows, n, d = c["rows"], c["n"], c["d"]
    x, x_scales = _in_blocks(_hidden(g, rows, d, 0.5), 1)
    w = torch.empty(n, d, dtype=torch.float8_e4m3fn, device=DEVICE)
    w_scales = torch.empty(_blocks(n, BLOCK), _blocks(d, BLOCK), device=DEVICE)
    for lo in range(0, n, 32768):
        hi = min(lo + 32768, n)
        w[lo:hi], w_scales[lo // BLOCK:_blocks(hi, BLOCK)] = _in_blocks(_normal(g, hi - lo, d) / math.sqrt(d), BLOCK)
    return dict(x=_rows_of(x, c["pad"]), x_scales=x_scales, w=_rows_of(w, c["pad"]), w_scales=w_scales,
                bias=0.1 * _normal(g, n) if c["bias"] else None,
                residual=_normal(g, rows, n).to(DTYPES[c["out"]]) if c["residual"] else None, out=_empty(rows, n, c["out"]))


def _prepare_distill(c, g):
    rows, vocab, k, t = c["rows"], c["vocab"], c["k"], c["temperature"]
    x = 1.5 * _normal(g, rows, vocab)
    # the teacher's best k ids: one out of each k-th of the vocabulary, in no order; its values fall with the rank
    u = torch.rand(rows, k, generator=g, device=DEVICE, dtype=torch.float64)
    ids = ((torch.arange(k, device=DEVICE) + u) * (vocab / k)).long().clamp_max(vocab - 1)
    ids = ids.gather(1, torch.rand(rows, k, generator=g, device=DEVICE).argsort(1))
    values = 14.0 - 2.0 * torch.log1p(torch.arange(k, device=DEVICE, dtype=torch.float32)) + 0.5 * _normal(g, rows, k)
    # the student knows them by and large
    x.scatter_(1, ids, values + _normal(g, rows, k) - 1.0)
    rest = 0.01 + 0.2 * torch.rand(rows, generator=g, device=DEVICE)   # the teacher's mass outside its list
    if c["teacher"] == "probs":
        values = torch.softmax(values, 1) * (1.0 - rest[:, None] if c["rest"] else 1.0)
    values = values.to(DTYPES[c["t"]])
    st = dict(logits=_rows_of(x.to(DTYPES[c["x"]]), c["pad"]), ids=ids.to(torch.int32), teacher=values, counts=None, teacher_lse=None,
              weights=None, loss=torch.empty(rows, device=DEVICE), grad=_empty(rows, vocab, c["out"]), scale=1.0 / rows)
    del x
    if c["ragged"]:   # lists of many lengths, and positions without any
        counts = torch.randint(0, k + 1, (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        if c["ragged"] == 1:
            st["counts"] = counts
        else:
            st["ids"][torch.arange(k, device=DEVICE)[None, :] >= counts[:, None]] = -1
    if c["teacher"] == "logits" and c["rest"]:
        st["teacher_lse"] = (torch.logsumexp(values.double() / t, 1) - torch.log1p(-rest.double())).float()
    if c["weights"]:   # a padded batch: positions that do not count
        st["weights"] = torch.rand(rows, generator=g, device=DEVICE) + 0.5
        st["weights"][torch.rand(rows, generator=g, device=DEVICE) < 0.1] = 0.0
    if c["kind"] == "distill":
        st["stats"] = torch.empty(rows, 4, device=DEVICE)
        return st
    # what the loss left: largest value and logarithm of the sum, of the whole row and of the ids outside the list
    z = st["logits"].float()
    stats = torch.zeros(rows, 4, device=DEVICE)
    stats[:, 0] = z.amax(1)
    stats[:, 1] = torch.log(torch.exp((z - stats[:, :1]) / t).sum(1, dtype=torch.float64)).float()
    if c["rest"]:
        z = z.masked_fill(_members(st, c), -math.inf)
        stats[:, 2] = z.amax(1)
        stats[:, 3] = torch.log(torch.exp((z - stats[:, 2:3]) / t).sum(1, dtype=torch.float64)).float()
    st["stats"] = stats
    return st


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    st = {"layer": _prepare_layer, "layer_grad": _prepare_layer_grad, "quantize": _prepare_quantize, "project": _prepare_project,
          "distill": _prepare_distill, "distill_grad": _prepare_distill}[case["kind"]](case, g)
    st["case"] = dict(case)
    return st


def _sampler():
    if not _program:
        sys.path.insert(0, os.path.join(os.getcwd(), "lily-qwen3.8-flash-next_amd", "python"))
        import lily_sampler
        _program["sampler"] = lily_sampler.Sampler(0)
    return _program["sampler"]


# ------------------------------------------------------------------ the plain forms


def _plain_blocks(y, block_rows, block):
    """(E4M3, scales) of rows, `block_rows` x `block` values a scale."""
    rows, d = y.shape
    p = torch.nn.functional.pad(y, (0, -d % block, 0, -rows % block_rows))
    p = p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // block, block)
    top = p.abs().amax((1, 3))
    scales = torch.where(top < TINY, torch.zeros_like(top), top / E4M3_MAX)
    wide = scales[:, None, :, None]
    q = torch.where(wide == 0, torch.zeros_like(p), p / wide).clamp(-E4M3_MAX, E4M3_MAX)
    return q.reshape(p.shape[0] * block_rows, -1)[:rows, :d].to(torch.float8_e4m3fn), scales


def _plain_layer(st):
    c = st["case"]
    h = st["x"].float()
    outs = {}
    if st["residual"] is not None:
        outs["summed"] = (h + st["residual"].float()).to(DTYPES[c["stream"]])
        h = outs["summed"].float()
    mean = h.mean(1, keepdim=True)
    off = h - mean
    rstd = torch.rsqrt(off.square().mean(1, keepdim=True) + EPS)
    y = off * rstd * st["weight"].float() + st["bias"].float()
    if c["out"] == "e4m3":
        outs["out"], outs["scales"] = _plain_blocks(y, 1, BLOCK if c["block"] else c["d"])
        if not c["block"]:
            outs["scales"] = outs["scales"][:, 0]
    else:
        outs["out"] = y.to(DTYPES[c["out"]])
    if c["stats"]:
        outs["mean"], outs["rstd"] = mean[:, 0], rstd[:, 0]
    return outs


def _plain_layer_grad(st):
    grad = st["grad"].float()
    x = (st["h"].float() - st["mean"][:, None]) * st["rstd"][:, None]
    g = grad * st["weight"].float()
    gx = st["rstd"][:, None] * (g - g.mean(1, keepdim=True) - x * (g * x).mean(1, keepdim=True))
    if st["past"] is not None:
        gx = gx + st["past"].float()
    return dict(grad_x=gx.to(DTYPES[st["case"]["out"]]), grad_weight=(grad * x).sum(0), grad_bias=grad.sum(0))


def _plain_quantize(st):
    out, scales = _plain_blocks(st["x"].float(), st["case"]["block_rows"], BLOCK)
    return dict(out=out, scales=scales)


def _act(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _spread(scales, block_rows, rows, d):
    return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :d]


def _plain_project(st):
    c = st["case"]
    x = st["x"].float() * _spread(st["x_scales"], 1, c["rows"], c["d"])
    w = st["w"].float() * _spread(st["w_scales"], BLOCK, c["n"], c["d"])
    v = x @ w.T
    if st["bias"] is not None:
        v = v + st["bias"]
    v = _act(v, c["act"])
    if st["residual"] is not None:
        v = v + st["residual"].float()
    return v.to(DTYPES[c["out"]])


def _valid(st, c):
    """Which entries of the lists count."""
    valid = (st["ids"] >= 0) & (st["ids"] < c["vocab"])
    if st["counts"] is not None:
        valid = valid & (torch.arange(c["k"], device=DEVICE)[None, :] < st["counts"][:, None])
    return valid


def _members(st, c):
    member = torch.zeros(c["rows"], c["vocab"] + 1, dtype=torch.bool, device=DEVICE)
    member.scatter_(1, torch.where(_valid(st, c), st["ids"].long(), c["vocab"]), True)
    return member[:, : c["vocab"]]


def _plain_teacher(st, c, valid):
    """Probabilities and their logarithms over the list, and the mass of the rest."""
    t = st["teacher"].float()
    if c["teacher"] == "probs":
        p = torch.where(valid, t.clamp_min(0.0), torch.zeros_like(t))
        if not c["rest"]:
            p = p / p.sum(1, keepdim=True).clamp_min(1e-37)
        log_p = torch.log(p)
    else:
        t = torch.where(valid, t / c["temperature"], torch.full_like(t, -math.inf))
        top = t.amax(1, keepdim=True)
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        below = st["teacher_lse"][:, None] - top if c["rest"] else torch.log(torch.exp(t - top).sum(1, keepdim=True))
        log_p = torch.where(valid, t - top - below, torch.full_like(t, -math.inf))
        p = torch.exp(log_p)
    return p, torch.where(p > 0, log_p, torch.zeros_like(p)), (1.0 - p.sum(1)).clamp_min(0.0)


def _plain_distill(st):
    c = st["case"]
    t, vocab = c["temperature"], c["vocab"]
    z = st["logits"].float()
    valid = _valid(st, c)
    ids = torch.where(valid, st["ids"].long(), 0)
    p, log_p, p_rest = _plain_teacher(st, c, valid)
    if c["kind"] == "distill":
        stats = torch.zeros(c["rows"], 4, device=DEVICE)
        stats[:, 0] = z.amax(1)
        stats[:, 1] = torch.log(torch.exp((z - stats[:, :1]) / t).sum(1))
        if c["rest"]:
            outside = z.masked_fill(_members(st, c), -math.inf)
            stats[:, 2] = outside.amax(1)
            stats[:, 3] = torch.log(torch.exp((outside - stats[:, 2:3]) / t).sum(1))
    else:
        stats = st["stats"]
    below = (z - stats[:, :1]) / t - stats[:, 1:2]                 # log q
    outs = {}
    if c["kind"] == "distill":
        log_q = below.gather(1, ids)
        loss = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
        if c["rest"]:
            log_rest = (stats[:, 2] - stats[:, 0]) / t + stats[:, 3] - stats[:, 1]
            loss = loss + torch.where(p_rest > 0, p_rest * (torch.log(p_rest) - log_rest), torch.zeros_like(loss))
        outs["loss"] = torch.where(valid.any(1), t * t * loss, torch.zeros_like(loss))
        outs["stats"] = stats
    target = torch.zeros(c["rows"], vocab, device=DEVICE).scatter_add_(1, ids, torch.where(valid, p, torch.zeros_like(p)))
    if c["rest"]:
        target = torch.where(_members(st, c), target, p_rest[:, None] * torch.exp((z - stats[:, 2:3]) / t - stats[:, 3:4]))
        share = 1.0
    else:
        share = p.sum(1, keepdim=True)
    weight = t * st["scale"] * (st["weights"][:, None] if st["weights"] is not None else torch.ones(c["rows"], 1, device=DEVICE))
    weight = torch.where(valid.any(1, keepdim=True), weight, torch.zeros_like(weight))
    outs["grad"] = (weight * (torch.exp(below) * share - target)).to(DTYPES[c["out"]])
    return outs


# ------------------------------------------------------------------ one pass


def run(state):
    c = state["case"]
    if not own:
        return {"layer": _plain_layer, "layer_grad": _plain_layer_grad, "quantize": _plain_quantize, "project": _plain_project,
                "distill": _plain_distill, "distill_grad": _plain_distill}[c["kind"]](state)
    s, st = _sampler(), state
    if c["kind"] == "layer":
        s.layer_norm(st["x"], st["weight"], st["bias"], st["out"], eps=EPS, residual=st["residual"], summed=st["summed"],
                     scales=st["scales"], mean=st["mean"], rstd=st["rstd"])
        return {name: st[name] for name in ("summed", "out", "scales", "mean", "rstd") if st[name] is not None}
    if c["kind"] == "layer_grad":
        s.layer_norm_backward(st["grad"], st["h"], st["mean"], st["rstd"], st["weight"], grad_x=st["grad_x"],
                              grad_weight=st["grad_weight"], grad_bias=st["grad_bias"], past=st["past"])
        return {name: st[name] for name in ("grad_x", "grad_weight", "grad_bias")}
    if c["kind"] == "quantize":
        s.quantize_blocks(st["x"], st["out"], st["scales"])
        return dict(out=st["out"], scales=st["scales"])
    if c["kind"] == "project":
        s.project_blocks(st["x"], st["x_scales"], st["w"], st["w_scales"], st["out"], bias=st["bias"], activation=c["act"],
                         residual=st["residual"])
        return st["out"]
    lists = dict(temperature=c["temperature"], teacher=c["teacher"], rest=bool(c["rest"]), teacher_lse=st["teacher_lse"],
                 counts=st["counts"], stats=st["stats"], grad=st["grad"], row_weights=st["weights"], grad_scale=st["scale"])
    if c["kind"] == "distill":
        s.distill(st["logits"], st["ids"], st["teacher"], st["loss"], **lists)
        return dict(loss=st["loss"], stats=st["stats"], grad=st["grad"])
    s.distill_backward(st["logits"], st["ids"], st["teacher"], **lists)
    return dict(grad=st["grad"])


# ------------------------------------------------------------------ 64 bits, and the work


def _in_e4m3(q):
    """E4M3 by its definition: steps of 2^(e - 3), e the exponent, from 2^-9 on."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(q / step) * step


def _exact_quantized(y, block_rows, block):
    rows, d = y.shape
    r, b = torch.arange(rows, device=DEVICE) // block_rows, torch.arange(d, device=DEVICE) // block
    at = (r[:, None] * _blocks(d, block) + b[None, :]).reshape(-1)
    top = torch.zeros(_blocks(rows, block_rows) * _blocks(d, block), dtype=torch.float64, device=DEVICE)
    top.scatter_reduce_(0, at, y.abs().reshape(-1), "amax")
    top[top < TINY] = 0.0
    scales = top / E4M3_MAX
    q = torch.nan_to_num(y.reshape(-1) / scales[at]).reshape(rows, d)
    return _in_e4m3(q), scales.reshape(_blocks(rows, block_rows), -1)


def _exact_layer(st):
    c = st["case"]
    h = st["x"].double()
    outs = {}
    if st["residual"] is not None:
        h = (h + st["residual"].double()).to(DTYPES[c["stream"]]).double()
        outs["summed"] = h
    mean = torch.einsum("rd->r", h) / c["d"]
    var = torch.var(h, dim=1, correction=0)
    y = torch.addcmul(st["bias"].double(), (h - mean[:, None]) / torch.sqrt(var + EPS)[:, None], st["weight"].double())
    if c["out"] == "e4m3":
        outs["out"], outs["scales"] = _exact_quantized(y, 1, BLOCK if c["block"] else c["d"])
        if not c["block"]:
            outs["scales"] = outs["scales"].reshape(-1)
    else:
        outs["out"] = y
    if c["stats"]:
        outs["mean"], outs["rstd"] = mean, (var + EPS).pow(-0.5)
    return outs


def _exact_layer_grad(st):
    d = st["case"]["d"]
    dy, h = st["grad"].double(), st["h"].double()
    x = torch.einsum("rd,r->rd", h - st["mean"].double()[:, None], st["rstd"].double())
    gb, gw = torch.einsum("rd->d", dy), torch.einsum("rd,rd->d", dy, x)
    dy = dy * st["weight"].double()
    gx = dy - (torch.einsum("rd->r", dy)[:, None] + x * torch.einsum("rd,rd->r", dy, x)[:, None]) / d
    gx = gx * st["rstd"].double()[:, None]
    return dict(grad_x=gx if st["past"] is None else gx + st["past"].double(), grad_weight=gw, grad_bias=gb)


def _exact_project(st):
    c = st["case"]
    v = torch.zeros(c["rows"], c["n"], dtype=torch.float64, device=DEVICE)
    columns = torch.arange(c["n"], device=DEVICE) // BLOCK
    for b in range(_blocks(c["d"], BLOCK)):
        part = st["x"][:, b * BLOCK:(b + 1) * BLOCK].double() @ st["w"][:, b * BLOCK:(b + 1) * BLOCK].double().T
        part *= st["x_scales"][:, b, None].double()
        part *= st["w_scales"][:, b].double()[columns]
        v += part
    if st["bias"] is not None:
        v = v + st["bias"].double()
    if c["act"] == "silu":
        v = v * torch.sigmoid(v)
    elif c["act"] == "relu":
        v = v.clamp_min(0.0)
    elif c["act"] == "gelu":
        v = v * torch.special.ndtr(v)
    elif c["act"] == "gelu_tanh":
        v = v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    return v if st["residual"] is None else v + st["residual"].double()


def _exact_rows(st, c, lo, hi):
    t = c["temperature"]
    z = st["logits"][lo:hi].double() / t
    n = st["ids"].shape[1]
    count = st["counts"][lo:hi].long() if st["counts"] is not None else torch.full((hi - lo,), n, device=DEVICE)
    on = (torch.arange(n, device=DEVICE) < count[:, None]) & (st["ids"][lo:hi] >= 0)
    ids = st["ids"][lo:hi].long().clamp_min(0)
    v = st["teacher"][lo:hi].double()
    if c["teacher"] == "logits":
        v = (v / t).masked_fill(~on, -math.inf)
        p = torch.exp(v - st["teacher_lse"][lo:hi, None].double()) if c["rest"] else torch.softmax(v, 1).nan_to_num(0.0)
    else:
        v = v.masked_fill(~on, 0.0)
        p = v if c["rest"] else (v / v.sum(1, keepdim=True)).nan_to_num(0.0)
    dense = torch.zeros_like(z).scatter_add_(1, ids, p)
    hit = torch.zeros_like(z).scatter_add_(1, ids, on.double()) > 0
    logq = torch.log_softmax(z, 1)
    loss = torch.xlogy(p, p).sum(1) - (dense * logq).nan_to_num(0.0).sum(1)
    stats = torch.zeros(hi - lo, 4, dtype=torch.float64, device=DEVICE)
    stats[:, 0] = z.amax(1) * t
    stats[:, 1] = torch.logsumexp(z, 1) - z.amax(1)
    if c["rest"]:
        out = z.masked_fill(hit, -math.inf)
        stats[:, 2] = out.amax(1) * t
        rest_lse = torch.logsumexp(out, 1)
        stats[:, 3] = rest_lse - out.amax(1)
        left = (1.0 - p.sum(1)).clamp_min(0.0)
        loss = loss + torch.xlogy(left, left) - left * (rest_lse - torch.logsumexp(z, 1))
        want = torch.where(hit, dense, left[:, None] * torch.exp(z - rest_lse[:, None]))
        grad = torch.exp(logq) - want
    else:
        grad = torch.exp(logq) * p.sum(1, keepdim=True) - dense
    scale = torch.full((hi - lo,), st["scale"] * t, dtype=torch.float64, device=DEVICE)
    if st["weights"] is not None:
        scale = scale * st["weights"][lo:hi].double()
    some = on.any(1)
    grad = torch.where(some[:, None], grad * scale[:, None], 0.0)
    return torch.where(some, loss * t * t, 0.0), stats, grad


def _exact_distill(st):
    c = st["case"]
    loss, stats, grads = [], [], []
    for lo in range(0, c["rows"], 128):
        l, s, g = _exact_rows(st, c, lo, min(lo + 128, c["rows"]))
        loss.append(l)
        stats.append(s)
        grads.append(g.float() if c["out"] == "bf16" else g)
    if c["kind"] == "distill_grad":
        return dict(grad=torch.cat(grads))
    return dict(loss=torch.cat(loss), stats=torch.cat(stats), grad=torch.cat(grads))


def exact(case, seed):
    st = prepare(case, seed)
    return {"layer": _exact_layer, "layer_grad": _exact_layer_grad, "quantize": lambda s: dict(zip(("out", "scales"), _exact_quantized(
        s["x"].double(), s["case"]["block_rows"], BLOCK))), "project": _exact_project, "distill": _exact_distill,
        "distill_grad": _exact_distill}[case["kind"]](st)


def _bytes(name):
    return {"none": 0, "bf16": 2, "f32": 4, "e4m3": 1}[name]


def work(case):
    c, rows = case, case["rows"]
    if c["kind"] == "layer":
        d = c["d"]
        per = _bytes(c["x"]) + 2 * _bytes(c["stream"]) + _bytes(c["out"])
        scales = 0 if c["out"] != "e4m3" else 4 * rows * (_blocks(d, BLOCK) if c["block"] else 1)
        return dict(bytes=rows * d * per + 4 * d + scales + 8 * rows * c["stats"], flops=9 * rows * d)
    if c["kind"] == "layer_grad":
        d = c["d"]
        return dict(bytes=rows * d * (_bytes(c["grad"]) + _bytes(c["h"]) + _bytes(c["out"]) * (1 + c["past"])) + 10 * d + 8 * rows,
                    flops=14 * rows * d)
    if c["kind"] == "quantize":
        d = c["d"]
        return dict(bytes=rows * d * (_bytes(c["x"]) + 1) + 4 * _blocks(rows, c["block_rows"]) * _blocks(d, BLOCK), flops=3 * rows * d)
    if c["kind"] == "project":
        n, d, o = c["n"], c["d"], _bytes(c["out"])
        scales = 4 * _blocks(d, BLOCK) * (rows + _blocks(n, BLOCK))
        return dict(bytes=(rows + n) * d + rows * n * o * (1 + c["residual"]) + 4 * n * c["bias"] + scales, flops=2 * rows * n * d)
    v, k = c["vocab"], c["k"]
    lists = rows * (k * (4 + _bytes(c["t"])) + 32)
    return dict(bytes=rows * v * (_bytes(c["x"]) + _bytes(c["out"])) + lists, flops=(8 if c["kind"] == "distill" else 5) * rows * v)
