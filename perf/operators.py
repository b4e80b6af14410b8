"""The operators around the head, as cases that can be timed and compared: what a decode step does
between its last layer and the token.

`kind` says which operator a case is:
  norm     the residual's addition and the RMS norm in front of the head, in bf16, f32 or 8 bits
  project  a matrix product with bias, activation and residual in its epilogue, bf16 or 8-bit floats:
           a draft head's block, a projection ahead of the head, a head held in 8-bit floats
  logits   penalties, bias lists and grammar masks applied to rows of logits, the rows written out as
           adjusted logits or log-probabilities, with each row's log-sum-exp
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
E4M3_MAX = 448.0
TINY = 2.0 ** -116     # rows of 8-bit norms whose largest magnitude lies below: zeros, scale 0
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}

_program = {}          # the library and its sampler, opened once as a program does


def listed():
    return [
        # The final norm of four conversations' decode step: the smallest call there is.
        dict(name="norm_decode_b4", kind="norm", rows=4, d=4096, x="bf16", stream="bf16", out="bf16", offset=0, pad=0),
        # A server's ragged decode batch at the smaller width, its residual stream in f32, 8-bit rows out.
        dict(name="norm_q8_b61", kind="norm", rows=61, d=2560, x="bf16", stream="f32", out="e4m3", offset=1, pad=64),
        # Prefill: every position's row on its way into an 8-bit product.
        dict(name="norm_q8_b8192", kind="norm", rows=8192, d=4096, x="bf16", stream="bf16", out="e4m3", offset=0, pad=0),
        # One request's draft head: x + silu(W x + b).
        dict(name="draft_block_b1", kind="project", rows=1, n=4096, d=4096, dtype="bf16", out="bf16", bias=1, act="silu",
             residual=1, pad=0),
        # The same block for a verify pass's rows of four requests, at the smaller width.
        dict(name="draft_block_b12", kind="project", rows=12, n=2560, d=2560, dtype="bf16", out="bf16", bias=1, act="silu",
             residual=1, pad=0),
        # A head held in 8-bit floats, the default batch of four, f32 logits.
        dict(name="head_e4m3_b4", kind="project", rows=4, n=VOCAB, d=4096, dtype="e4m3", out="f32", bias=0, act="none",
             residual=0, pad=0),
        # A ragged middle batch through an odd-sized layer in 8-bit floats, rows of a wider buffer.
        dict(name="layer_e4m3_b100", kind="project", rows=100, n=10007, d=4096, dtype="e4m3", out="bf16", bias=1,
             act="gelu_tanh", residual=0, pad=32),
        # Prefill through the block: bound by the matrix cores.
        dict(name="prefill_bf16_b8192", kind="project", rows=8192, n=4096, d=4096, dtype="bf16", out="bf16", bias=1,
             act="silu", residual=1, pad=0),
        # Prefill in 8-bit floats, a wide layer.
        dict(name="prefill_e4m3_b8192", kind="project", rows=8192, n=12288, d=4096, dtype="e4m3", out="bf16", bias=0,
             act="none", residual=0, pad=0),
        # Four conversations under penalties: the adjusted logits a host's own sampler or ranking reads.
        dict(name="logits_decode_b4", kind="logits", rows=4, vocab=VOCAB, x="f32", out="f32", logprobs=0, history=8192,
             mask=0.0, bias=0, temperature=0.6),
        # Constrained decoding with bias lists; the log-probabilities a request asked for. One row's mask bars everything.
        dict(name="logprobs_masked_b64", kind="logits", rows=64, vocab=VOCAB, x="bf16", out="f32", logprobs=1, history=512,
             mask=0.02, bias=32, temperature=1.0),
        # Throughput serving: log-probabilities of the headline batch.
        dict(name="logprobs_b1024", kind="logits", rows=1024, vocab=VOCAB, x="bf16", out="f32", logprobs=1, history=2048,
             mask=0.0, bias=0, temperature=0.8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "project", "project", "logits"])
    if kind == "norm":
        rows = _log_int(rng, 1, 8192)
        d = _log_int(rng, 64, min(16384, 8192 * 4096 // rows))
        return dict(kind=kind, rows=rows, d=d, x=rng.choice(["bf16", "bf16", "f32"]),
                    stream=rng.choice(["none", "bf16", "bf16", "f32"]), out=rng.choice(["bf16", "e4m3", "e4m3", "f32"]),
                    offset=rng.randrange(2), pad=rng.choice([0, 0, 8, 3]))
    if kind == "project":
        dtype = rng.choice(["bf16", "e4m3"])
        rows = _log_int(rng, 1, 8192)
        n = _log_int(rng, 64, 16384)
        d = 16 * _log_int(rng, 8, 512)
        while rows * n * d > 8192 * 12288 * 4096:
            n = (n + 1) // 2
        return dict(kind=kind, rows=rows, n=n, d=d, dtype=dtype, out=rng.choice(["bf16", "bf16", "f32"]),
                    bias=rng.randrange(2), act=rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]),
                    residual=rng.randrange(2), pad=rng.choice([0, 0, 16, 32]))
    rows = _log_int(rng, 1, 1024)
    vocab = _log_int(rng, 8000, VOCAB_LARGE)
    while rows * vocab > 1024 * VOCAB:
        rows = (rows + 1) // 2
    return dict(kind=kind, rows=rows, vocab=vocab, x=rng.choice(["bf16", "f32"]),
                out=rng.choice(["f32", "f32", "bf16"]), logprobs=rng.randrange(2),
                history=rng.choice([0, _log_int(rng, 16, 8192)]), mask=rng.choice([0.0, 0.0, 0.02, 0.5, 0.95]),
                bias=rng.choice([0, 0, _log_int(rng, 1, 300)]), temperature=rng.choice([1.0, 0.6, 0.8, 1.3]))


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


def _in_e4m3(t):
    scale = t.abs().amax(1) / E4M3_MAX
    return (t / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _weights(g, n, d, dtype):
    """[n, d] of N(0, 1 / d), a block of rows at a time."""
    w = torch.empty(n, d, dtype=DTYPES[dtype], device=DEVICE)
    scales = torch.empty(n, dtype=torch.float32, device=DEVICE) if dtype == "e4m3" else None
    for lo in range(0, n, 32768):
        block = _normal(g, min(32768, n - lo), d) / math.sqrt(d)
        if dtype == "e4m3":
            w[lo:lo + 32768], scales[lo:lo + 32768] = _in_e4m3(block)
        else:
            w[lo:lo + 32768] = block.to(torch.bfloat16)
    return w, scales


def _prepare_norm(c, g):
    rows, d = c["rows"], c["d"]
    # a hidden state's channels differ in size, a few by much
    size = torch.exp(_normal(g, d))
    st = dict(x=_rows_of((_normal(g, rows, d) * 0.3 * size).to(DTYPES[c["x"]]), c["pad"]),
              weight=(1.0 - c["offset"] + 0.2 * _normal(g, d)).to(torch.bfloat16), residual=None)
    if c["stream"] != "none":
        st["residual"] = _rows_of((_normal(g, rows, d) * size).to(DTYPES[c["stream"]]), c["pad"])
    if own:
        st["out"] = torch.empty(rows, d, dtype=DTYPES[c["out"]], device=DEVICE)
        st["scales"] = torch.empty(rows, device=DEVICE) if c["out"] == "e4m3" else None
        st["summed"] = None if st["residual"] is None else torch.empty(rows, d, dtype=DTYPES[c["stream"]], device=DEVICE)
    return st


def _prepare_project(c, g):
    rows, n, d = c["rows"], c["n"], c["d"]
    x = _normal(g, rows, d)
    st = dict(x_scales=None)
    if c["dtype"] == "e4m3":
        x, st["x_scales"] = _in_e4m3(x)
    else:
        x = x.to(torch.bfloat16)
    st["x"] = _rows_of(x, c["pad"])
    w, st["w_scales"] = _weights(g, n, d, c["dtype"])
    st["w"] = _rows_of(w, c["pad"])
    st["bias"] = 0.1 * _normal(g, n) if c["bias"] else None
    st["residual"] = _normal(g, rows, n).to(DTYPES[c["out"]]) if c["residual"] else None
    if own:
        st["out"] = torch.empty(rows, n, dtype=DTYPES[c["out"]], device=DEVICE)
    return st


PENALTIES = dict(repetition_penalty=1.05, presence_penalty=0.3, frequency_penalty=0.2)


def _prepare_logits(c, g):
    rows, vocab = c["rows"], c["vocab"]
    x = 2.0 * _normal(g, rows, vocab)
    # a tenth with heavy tails, as a language model's rows have them (Student's t of 3 degrees, times 4)
    heavy = torch.rand(rows, vocab, generator=g, device=DEVICE) < 0.1
    at = heavy.nonzero(as_tuple=True)
    chi = _normal(g, 3, at[0].numel()).square().sum(0) / 3.0
    x[at] = 4.0 * _normal(g, at[0].numel()) / chi.sqrt()
    del heavy, at, chi
    st = dict(logits=x.to(DTYPES[c["x"]]), history=None, allow=None, bias=None)
    if c["history"]:
        # ids as running text has them: P(rank r) ~ r^-1.1
        below = torch.arange(1, vocab + 1, dtype=torch.float64).pow(-1.1).cumsum(0)
        u = torch.rand(rows, c["history"], generator=g, device=DEVICE, dtype=torch.float64) * float(below[-1])
        ranks = torch.searchsorted(below.to(DEVICE), u).clamp_max(vocab - 1)
        st["history"] = torch.randperm(vocab, generator=g, device=DEVICE)[ranks].to(torch.int32)
    if c["mask"]:
        # runs of 16 admitted ids; the last row's grammar has come to a dead end
        words = (vocab + 31) // 32
        halves = (torch.rand(rows, words, 2, generator=g, device=DEVICE) < c["mask"]).to(torch.int64) * 0xFFFF
        w = halves[..., 0] | (halves[..., 1] << 16)
        w[-1] = 0
        st["allow"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    if c["bias"]:
        ids = torch.rand(rows, vocab, generator=g, device=DEVICE).topk(c["bias"], dim=1).indices
        st["bias"] = (ids, 5.0 * _normal(g, rows, c["bias"]).sign())
    if not own:
        st["counts"] = None
        if c["history"]:
            st["counts"] = torch.zeros(rows, vocab, dtype=torch.int32, device=DEVICE)
            st["counts"].scatter_add_(1, st["history"].long(), torch.ones_like(st["history"]))
        return st
    # what a serving program keeps: the requests' histories as scratches, the batch as a resident plan
    LS, s = _library()
    params = [LS.SamplingParams.greedy(temperature=c["temperature"], top_k=64, seed=r,
                                       **(PENALTIES if c["history"] else {})) for r in range(rows)]
    kw = {}
    if c["history"]:
        kw["scratch"] = []
        for r in range(rows):
            kw["scratch"].append(LS.SamplerScratch(s, vocab))
            kw["scratch"][-1].add_history(st["history"][r])
    if c["bias"]:
        ids, delta = (t.tolist() for t in st["bias"])
        kw["bias"] = [list(zip(i, e)) for i, e in zip(ids, delta)]
    st["scratch"] = kw.get("scratch")
    st["ids"] = torch.empty(rows, dtype=torch.int32, device=DEVICE)
    st["plan"] = s.plan(st["logits"], params, [0] * rows, st["ids"], allow=st["allow"], **kw)
    st["out"] = torch.empty(rows, vocab, dtype=DTYPES[c["out"]], device=DEVICE)
    st["lse"] = torch.empty(rows, device=DEVICE)
    return st


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    st = {"norm": _prepare_norm, "project": _prepare_project, "logits": _prepare_logits}[case["kind"]](case, g)
    st["case"] = dict(case)
    if own:
        st["sampler"] = _library()[1]
    return st


def _library():
    if not _program:
        sys.path.insert(0, os.path.join(os.getcwd(), "lily-qwen3.8-flash-next_amd", "python"))
        import lily_sampler
        _program["library"] = lily_sampler
        _program["sampler"] = lily_sampler.Sampler(0)
    return _program["library"], _program["sampler"]


# ------------------------------------------------------------------ the plain forms


def _plain_norm(st):
    c = st["case"]
    h = st["x"].float()
    outs = {}
    if st["residual"] is not None:
        h = (h + st["residual"].float()).to(DTYPES[c["stream"]])
        outs["summed"] = h
        h = h.float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * (st["weight"].float() + c["offset"])
    if c["out"] != "e4m3":
        outs["out"] = y.to(DTYPES[c["out"]])
        return outs
    top = y.abs().amax(1)
    scale = torch.where(top < TINY, torch.zeros_like(top), top / E4M3_MAX)
    q = torch.where(top[:, None] < TINY, torch.zeros_like(y), y / scale[:, None])
    outs["out"] = q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    outs["scales"] = scale
    return outs


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


def _plain_project(st):
    c = st["case"]
    v = st["x"].float() @ st["w"].float().T
    if st["x_scales"] is not None:
        v = v * st["x_scales"][:, None] * st["w_scales"][None, :]
    if st["bias"] is not None:
        v = v + st["bias"]
    v = _act(v, c["act"])
    if st["residual"] is not None:
        v = v + st["residual"].float()
    return v.to(DTYPES[c["out"]])


def _plain_logits(st):
    c = st["case"]
    a = st["logits"].float()
    a = torch.where(torch.isnan(a), torch.full_like(a, -math.inf), a)
    if st["bias"] is not None:
        a = a.scatter_add(1, st["bias"][0], st["bias"][1])
    if st["allow"] is not None:
        ids = torch.arange(c["vocab"], device=DEVICE)
        allowed = (st["allow"][:, ids >> 5] >> (ids & 31)) & 1
        a = torch.where(allowed != 0, a, torch.full_like(a, -math.inf))
    if st["counts"] is not None:
        rep, n = PENALTIES["repetition_penalty"], st["counts"]
        lowered = torch.where(a > 0, a / rep, a * rep) - (PENALTIES["presence_penalty"] + PENALTIES["frequency_penalty"] * n)
        a = torch.where(n > 0, lowered, a)
    a = a / c["temperature"]
    top = a.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    lse = top + torch.log(torch.exp(a - top).sum(1, keepdim=True))
    if c["logprobs"]:
        a = torch.where(torch.isinf(a), a, a - lse)
    return dict(out=a.to(DTYPES[c["out"]]), lse=lse[:, 0])


# ------------------------------------------------------------------ one pass


def run(state):
    c = state["case"]
    if not own:
        return {"norm": _plain_norm, "project": _plain_project, "logits": _plain_logits}[c["kind"]](state)
    s = state["sampler"]
    if c["kind"] == "norm":
        s.rms_norm(state["x"], state["weight"], state["out"], eps=1e-6, residual=state["residual"], summed=state["summed"],
                   weight_offset=float(c["offset"]), scales=state["scales"])
        outs = dict(out=state["out"])
        if state["summed"] is not None:
            outs["summed"] = state["summed"]
        if state["scales"] is not None:
            outs["scales"] = state["scales"]
        return outs
    if c["kind"] == "project":
        s.project(state["x"], state["w"], state["out"], x_scales=state["x_scales"], weight_scales=state["w_scales"],
                  bias=state["bias"], activation=c["act"], residual=state["residual"])
        return state["out"]
    state["plan"].process_logits(state["out"], log_sum_exp=state["lse"], logprobs=bool(c["logprobs"]))
    return dict(out=state["out"], lse=state["lse"])


# ------------------------------------------------------------------ 64 bits, and the work


def _exact_norm(st):
    c = st["case"]
    h = st["x"].double()
    outs = {}
    if st["residual"] is not None:
        h = (h + st["residual"].double()).to(DTYPES[c["stream"]]).double()
        outs["summed"] = h
    ms = torch.einsum("rd,rd->r", h, h) / c["d"]
    y = h / torch.sqrt(ms + 1e-6)[:, None] * (st["weight"].double() + c["offset"])[None, :]
    if c["out"] != "e4m3":
        return {**outs, "out": y}
    scale = y.abs().max(dim=1).values / E4M3_MAX
    scale[scale * E4M3_MAX < TINY] = 0.0
    q = torch.nan_to_num(y / scale[:, None])
    # to e4m3 by its definition: steps of 2^(e - 3), e the exponent, from 2^-9 on
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3.0)
    return {**outs, "out": torch.round(q / step) * step, "scales": scale}


def _exact_project(st):
    c = st["case"]
    outs = []
    x = st["x"].double()
    for lo in range(0, c["n"], 32768):
        hi = min(lo + 32768, c["n"])
        v = x @ st["w"][lo:hi].double().T
        if st["x_scales"] is not None:
            v = v * torch.outer(st["x_scales"].double(), st["w_scales"][lo:hi].double())
        if st["bias"] is not None:
            v = v + st["bias"][lo:hi].double()
        if c["act"] == "silu":
            v = v * torch.sigmoid(v)
        elif c["act"] == "relu":
            v = v.clamp_min(0.0)
        elif c["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        elif c["act"] == "gelu_tanh":
            v = v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
        outs.append(v)
    v = torch.cat(outs, 1)
    return v if st["residual"] is None else v + st["residual"].double()


def _exact_logits(st):
    c = st["case"]
    outs, lses = [], []
    for r in range(c["rows"]):
        a = st["logits"][r].double()
        if st["bias"] is not None:
            a[st["bias"][0][r]] += st["bias"][1][r].double()
        if st["history"] is not None:
            ids, n = torch.unique(st["history"][r].long(), return_counts=True)
            l = a[ids]
            l = torch.where(l > 0, l / PENALTIES["repetition_penalty"], l * PENALTIES["repetition_penalty"])
            a[ids] = l - PENALTIES["presence_penalty"] - PENALTIES["frequency_penalty"] * n.double()
        if st["allow"] is not None:
            bits = (st["allow"][r].long()[:, None] >> torch.arange(32, device=DEVICE)[None, :]) & 1
            a[bits.reshape(-1)[: c["vocab"]] == 0] = -math.inf
        a = a / c["temperature"]
        lse = torch.logsumexp(a, 0)
        if c["logprobs"] and bool(torch.isfinite(lse)):
            a = a - lse
        outs.append(a.float() if c["out"] == "bf16" else a)
        lses.append(lse)
    return dict(out=torch.stack(outs), lse=torch.stack(lses))


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "project": _exact_project, "logits": _exact_logits}[case["kind"]](st)


def _bytes(name):
    return {"none": 0, "bf16": 2, "f32": 4, "e4m3": 1}[name]


def work(case):
    c, rows = case, case["rows"]
    if c["kind"] == "norm":
        per = _bytes(c["x"]) + 2 * _bytes(c["stream"]) + _bytes(c["out"])
        return dict(bytes=rows * c["d"] * per + 2 * c["d"] + (4 * rows if c["out"] == "e4m3" else 0), flops=6 * rows * c["d"])
    if c["kind"] == "project":
        e, o = _bytes(c["dtype"]), _bytes(c["out"])
        scales = 4 * (rows + c["n"]) if c["dtype"] == "e4m3" else 0
        return dict(bytes=(rows + c["n"]) * c["d"] * e + rows * c["n"] * o * (1 + c["residual"]) + 4 * c["n"] * c["bias"] + scales,
                    flops=2 * rows * c["n"] * c["d"])
    v = c["vocab"]
    # a bit an id for the mask and one for the history's ids, whose counts come on top
    extra = (v / 8 if c["mask"] else 0) + (v / 8 + 4 * min(c["history"], v) if c["history"] else 0) + 8 * c["bias"]
    return dict(bytes=rows * (v * (_bytes(c["x"]) + _bytes(c["out"])) + extra + 4), flops=6 * rows * v)
