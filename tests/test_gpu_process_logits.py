"""Processed logits (lily_process_logits, lily_plan_process_logits) against numpy.

Bar:
  * adjusted f32 values bit-exact against the draws' arithmetic restated in numpy f32 (biases in list
    order, mask, penalties, IEEE division by T; NaN worth -inf); bf16 output: those rounded to nearest even;
  * log_sum_exp against f64 over the reference's f32 values: a thread adds n <= max(8, V / 1024) terms
    (slices of 2 048 to 8 192 ids, 32 a thread at most, or of a 64th of a long row), each addition, each raise of its reference (one
    in four) and each term (exponent formed with three roundings of at most |x| e^-|x| <= 0.37 weight, the
    exponential 2 steps) rounded: (1.25 n + 8) 2^-24 relative to the sum, so absolute in its logarithm,
    and one rounding of the result;
  * log-probabilities: that, and the roundings of a - top, of the logarithm of the sum and of their
    difference, none of which is larger than the log-probability;
  * bf16 output half a bf16 step (2^-8 relative) more.
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


def _adjusted(x, kw, counts=None, allow=None, bias=None):
    """One row in f32, operation for operation."""
    p = ls_params(**kw)
    with np.errstate(all="ignore"):
        l = x.astype(F).copy()
        for i, delta in bias or []:
            if i < len(l):
                l[i] = F(l[i] + F(delta))
        if counts is not None:
            c = counts.astype(F)
            rep, pres, freq = F(p.repetition_penalty), F(p.presence_penalty), F(p.frequency_penalty)
            low = np.where(l > 0, l / rep, l * rep).astype(F)
            low = (low - (pres + (freq * c).astype(F)).astype(F)).astype(F)
            l = np.where(counts > 0, low, l)
        if allow is not None:
            bits = (allow[np.arange(len(l)) >> 5] >> (np.arange(len(l)) & 31)) & 1
            l = np.where(bits != 0, l, F(-np.inf))
        l = (l / F(p.effective()[0])).astype(F)
        return np.where(np.isnan(l), F(-np.inf), l)


def _lse(a):
    a = a.astype(np.float64)
    top = a.max()
    if np.isinf(top):
        return top
    return top + np.log(np.exp(a - top).sum())


def _to_f32(t):
    return t.float().cpu().numpy()


def _check(out, lse, want, logprobs, vocab):
    """out: tensor [rows, V]; want: list of f32 rows."""
    n = max(8, vocab / 1024)
    off = (1.25 * n + 8) * U
    got, got_lse = _to_f32(out), None if lse is None else lse.cpu().numpy()
    half = 2.0 ** -8 if out.dtype == torch.bfloat16 else 0.0
    for r, a in enumerate(want):
        ref = _lse(a)
        if got_lse is not None:
            if np.isinf(ref):
                assert got_lse[r] == ref, (r, got_lse[r], ref)
            else:
                assert abs(got_lse[r] - ref) <= off + abs(ref) * U, (r, got_lse[r], ref)
        if not logprobs:
            rounded = a if out.dtype == torch.float32 else W.bf16_bits_to_f32(W.to_bf16_bits(a))
            assert np.array_equal(got[r].view(np.uint32), rounded.astype(F).view(np.uint32)), r
            continue
        fin = np.isfinite(a)
        assert np.all(got[r][~fin & (a < 0)] == -np.inf), r
        if np.isfinite(ref):
            p = a[fin].astype(np.float64) - ref
            g = got[r][fin].astype(np.float64)
            if half:
                # bf16's largest value is (2 - 2^-7) 2^127; from (2 - 2^-8) 2^127 = 3.396e38 on, and the f32
                # lowest of these rows is 3.403e38, the nearest bf16 value is an infinity
                beyond = p <= -(2.0 - 2.0 ** -8) * 2.0 ** 127
                assert np.all(g[beyond] == -np.inf), r
                g, p = g[~beyond], p[~beyond]
            err = np.abs(g - p)
            assert np.all(err <= (off + 3 * U * np.abs(p)) * (1 + half) + half * np.abs(p)), (r, float(err.max()))


def _history(sampler, rng, vocab, n):
    sc = LS.SamplerScratch(sampler, vocab)
    ids = (rng.zipf(1.3, n) % vocab).astype(np.int32)
    sc.add_history(torch.from_numpy(ids).to(dev()))
    return sc, np.bincount(ids, minlength=vocab).astype(np.int64)


def _case(sampler, rng, rows, vocab, dtype, pen, mask, bias, temps):
    """Inputs of every kind a batch can mix, row by row, and the wanted rows."""
    x = rng.normal(0, 3, (rows, vocab)).astype(F)
    if vocab > 40:
        x[0, vocab // 3] = np.nan
        x[0, vocab // 2] = -np.inf
        x[-1, 5] = -3.4028234663852886e38
    if dtype == "bf16":
        x = W.bf16_bits_to_f32(W.to_bf16_bits(x))
    kws, scratch, counts = [], [], []
    for r in range(rows):
        kw = dict(temperature=temps[r % len(temps)], top_k=50, seed=r)
        sc = cnt = None
        if pen and r % 4 != 3:
            kw.update([dict(repetition_penalty=1.1, presence_penalty=0.3, frequency_penalty=0.2),
                       dict(repetition_penalty=0.8), dict(presence_penalty=-0.5, frequency_penalty=0.1)][r % 3])
            sc, cnt = _history(sampler, rng, vocab, int(rng.integers(1, 400)))
        kws.append(kw)
        scratch.append(sc)
        counts.append(cnt)
    words = (vocab + 31) // 32
    allow = None
    if mask == "rows":
        allow = rng.integers(0, 2 ** 32, (rows, words + 2), dtype=np.uint32)
        allow[rows // 2] = 0
        allow[0] = 0xFFFFFFFF
    elif mask == "one":
        allow = rng.integers(0, 2 ** 32, words, dtype=np.uint32)
    lists = None
    if bias:
        lists = [[(int(i), float(rng.normal(0, 4))) for i in rng.integers(0, vocab, bias if r % 3 else 1)]
                 for r in range(rows)]
        lists[-1] = lists[-1] + [lists[-1][0], (vocab - 1, 2.5), (vocab + 7, 9.0)]   # twice the same id, the last, one outside
        if rows > 1:
            lists[0] = []
    want = [_adjusted(x[r], kws[r], counts[r], None if allow is None else (allow[r] if allow.ndim == 2 else allow),
                      lists[r] if lists else None) for r in range(rows)]
    return x, kws, scratch, allow, lists, want


def _place(x, dtype, pad, start):
    """The rows in a wider buffer that starts anywhere."""
    rows, vocab = x.shape
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    buf = torch.full((rows * (vocab + pad) + start + 4,), 7.0, dtype=dt, device=dev())
    m = torch.as_strided(buf, (rows, vocab), (vocab + pad, 1), start)
    m.copy_(upload_logits(W.to_bf16_bits(x) if dtype == "bf16" else x))
    return buf, m


SHAPES = [(1, 1), (2, 3), (3, 31), (1, 33), (8, 1000), (9, 4097), (5, 50257), (3, 151936), (1, 151936), (64, 8200), (300, 2500)]


@pytest.mark.parametrize("rows, vocab", SHAPES)
@pytest.mark.parametrize("dtype, out_dtype", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("logprobs, with_sum", [(False, False), (False, True), (True, True), (True, False)])
@pytest.mark.parametrize("kind", ["plain", "everything"])
def test_against_numpy(sampler, rows, vocab, dtype, out_dtype, logprobs, with_sum, kind):
    rng = np.random.default_rng(rows * 7 + vocab + 2 * logprobs + with_sum)
    full = kind == "everything"
    x, kws, scratch, allow, lists, want = _case(sampler, rng, rows, vocab, dtype, full, "rows" if full else None,
                                                20 if full else 0, [1.0, 0.7, 0.0, 1.9])
    pad, start = (5, 3) if full else (0, 0)
    _, logits = _place(x, dtype, pad, start)
    buf, out = _place(np.zeros_like(x), out_dtype, 3 if full else 0, 1 if full else 0)
    before = buf.clone()
    lse = torch.full((rows,), 5.0, device=dev()) if with_sum else None
    a = None if allow is None else torch.from_numpy(allow.view(np.int32)).to(dev())
    params = [ls_params(**kw) for kw in kws]
    torch.cuda.synchronize()
    keep = sampler.process_logits(logits, params, out, log_sum_exp=lse, logprobs=logprobs, scratch=scratch, allow=a, bias=lists)
    sampler.synchronize()
    _check(out, lse, want, logprobs, vocab)
    mask = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(mask, (rows, vocab), out.stride(), out.storage_offset()).fill_(False)
    assert torch.equal(buf[mask], before[mask])
    # the same through a resident plan (which a batch of a few rows that draw differently reorders)
    ids = torch.zeros(rows, dtype=torch.int32, device=dev())
    plan = sampler.plan(logits, params, [0] * rows, ids, scratch=scratch, allow=a, bias=lists)
    again = torch.empty_like(out)
    lse2 = torch.empty_like(lse) if with_sum else None
    torch.cuda.synchronize()
    plan.process_logits(again, log_sum_exp=lse2, logprobs=logprobs)
    sampler.synchronize()
    _check(again, lse2, want, logprobs, vocab)
    plan.close()
    del keep


def test_a_plan_whose_rows_were_reordered_writes_them_in_order(sampler):
    """A batch of streamable rows and a few that need the other selects is kept in two parts."""
    rng = np.random.default_rng(3)
    rows, vocab = 80, 6000
    x = rng.normal(0, 2, (rows, vocab)).astype(F)
    kws = [dict(temperature=1.0, top_k=500 if r % 10 == 0 else 20, seed=r) for r in range(rows)]
    logits = upload_logits(x)
    ids = torch.zeros(rows, dtype=torch.int32, device=dev())
    plan = sampler.plan(logits, [ls_params(**k) for k in kws], [0] * rows, ids)
    out, lse = torch.empty_like(logits), torch.empty(rows, device=dev())
    torch.cuda.synchronize()
    plan.process_logits(out, log_sum_exp=lse)
    sampler.synchronize()
    _check(out, lse, [x[r] for r in range(rows)], False, vocab)
    plan.run(0)
    plan.process_logits(out, log_sum_exp=lse, logprobs=True)
    sampler.synchronize()
    _check(out, lse, [x[r] for r in range(rows)], True, vocab)
    plan.close()


@pytest.mark.parametrize("rows", [2, 400])
@pytest.mark.parametrize("logprobs", [False, True])
def test_in_place_and_one_mask_for_all_rows(sampler, rows, logprobs):
    rng = np.random.default_rng(11 + rows)
    vocab = 9001
    x, kws, scratch, allow, lists, want = _case(sampler, rng, rows, vocab, "f32", True, "one", 5, [0.9])
    logits = upload_logits(x)
    lse = torch.empty(rows, device=dev())
    a = torch.from_numpy(allow.view(np.int32)).to(dev())
    torch.cuda.synchronize()
    sampler.process_logits(logits, [ls_params(**k) for k in kws], logits, log_sum_exp=lse, logprobs=logprobs,
                           scratch=scratch, allow=a, bias=lists)
    sampler.synchronize()
    _check(logits, lse, want, logprobs, vocab)


@pytest.mark.parametrize("rows, vocab, pairs", [(2, 20000, 2000), (300, 4000, 700), (1, 300000, 5000)])
def test_long_bias_lists(sampler, rows, vocab, pairs):
    """More pairs in a slice than LDS keeps, the same id many times over, and a row longer than one slice's bitmap."""
    rng = np.random.default_rng(pairs)
    x = rng.normal(0, 2, (rows, vocab)).astype(F)
    lists = [[(int(i), float(v)) for i, v in zip(rng.integers(0, min(vocab, 1500), pairs), rng.normal(0, 1, pairs))]
             for _ in range(rows)]
    want = [_adjusted(x[r], {}, bias=lists[r]) for r in range(rows)]
    logits = upload_logits(x)
    for logprobs in (False, True):
        out, lse = torch.empty_like(logits), torch.empty(rows, device=dev())
        torch.cuda.synchronize()
        keep = sampler.process_logits(logits, [ls_params()] * rows, out, log_sum_exp=lse, logprobs=logprobs, bias=lists)
        sampler.synchronize()
        _check(out, lse, want, logprobs, vocab)
        del keep


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_lowest_values_of_infinities_and_of_nothing(sampler, rows, dtype):
    vocab = 3001
    low = -3.4028234663852886e38 if dtype == "f32" else -3.3895313892515355e38
    x = np.full((4, vocab), low, dtype=F)            # masked by the type's lowest value, all of it
    x[1] = -np.inf
    x[2] = 1.5
    x[2, 100] = np.inf
    x[3] = np.nan
    x[3, 7] = 2.0
    x = np.repeat(x, rows, axis=0)
    logits = upload_logits(W.to_bf16_bits(x) if dtype == "bf16" else x)
    n = x.shape[0]
    out, lse = torch.empty(n, vocab, device=dev()), torch.empty(n, device=dev())
    torch.cuda.synchronize()
    sampler.process_logits(logits, [ls_params()] * n, out, log_sum_exp=lse, logprobs=True)
    sampler.synchronize()
    p, s = out.cpu().numpy(), lse.cpu().numpy()
    lo, none, inf, one = 0, rows, 2 * rows, 3 * rows
    assert s[lo] == F(low) and np.all(np.abs(p[lo] + np.log(vocab)) < 1e-5)
    assert s[none] == -np.inf and np.all(p[none] == -np.inf)
    assert s[inf] == np.inf and np.all(p[inf][np.arange(vocab) != 100] == -np.inf) and np.isnan(p[inf][100])
    assert s[one] == 2.0 and p[one][7] == 0.0 and np.all(np.delete(p[one], 7) == -np.inf)


def test_a_draw_from_the_written_row_is_the_draw_from_the_raw_one(sampler):
    rng = np.random.default_rng(21)
    rows, vocab = 6, 50257
    x, kws, scratch, allow, lists, _ = _case(sampler, rng, rows, vocab, "f32", True, "rows", 12, [0.7, 1.3])
    allow[rows // 2] = 0xFFFFFFFF
    for r, k in enumerate(kws):
        k.update(top_k=40, top_p=0.95)
    logits, a = upload_logits(x), torch.from_numpy(allow.view(np.int32)).to(dev())
    written = torch.empty_like(logits)
    raw_ids, ids = (torch.zeros(rows, dtype=torch.int32, device=dev()) for _ in range(2))
    lp, lse = torch.zeros(rows, device=dev()), torch.zeros(rows, device=dev())
    torch.cuda.synchronize()
    params = [ls_params(**k) for k in kws]
    sampler.process_logits(logits, params, written, log_sum_exp=lse, scratch=scratch, allow=a, bias=lists)
    plain = [ls_params(temperature=1.0, top_k=40, top_p=0.95, seed=r) for r in range(rows)]
    for step in range(8):
        sampler.sample_rows(written, plain, [step] * rows, ids)
        sampler.process_logits(logits, params, written, log_sum_exp=lse, scratch=scratch, allow=a, bias=lists)
        keep = sampler.sample_rows(logits, params, [step] * rows, raw_ids, scratch=scratch, allow=a, bias=lists, out_logprobs=lp)
        sampler.synchronize()
        # (the draws above came from the row as it stood before this step's token was counted)
        got = written.gather(1, raw_ids.long()[:, None])[:, 0] - lse
        assert bool(((got - lp).abs() <= 1e-5 * lp.abs().clamp_min(1.0)).all()), (got, lp)
        assert torch.equal(ids, raw_ids), step
        sampler.process_logits(logits, params, written, log_sum_exp=lse, scratch=scratch, allow=a, bias=lists)
        del keep


@pytest.mark.parametrize("looks", ["0,0,1000000", "1,1,1000000"])
def test_slices_that_do_not_wait_for_each_other(monkeypatch, looks):
    """A slice that does not find the words of its row's other slices forms them itself: the same bits, in place of
    the logits too, and the workspace is clean for the calls that follow."""
    patient = LS.Sampler(0)
    monkeypatch.setenv("LILY_SAMPLER_WIDE_LOOKS", looks)
    hasty = LS.Sampler(0)
    monkeypatch.delenv("LILY_SAMPLER_WIDE_LOOKS")
    rng = np.random.default_rng(31)
    for rows, vocab in ((1, 151936), (7, 50257), (70, 30000)):
        x, kws, _, allow, lists, _ = _case(None, rng, rows, vocab, "f32", False, "rows", 9, [0.7, 1.0])
        logits, a = upload_logits(x), torch.from_numpy(allow.view(np.int32)).to(dev())
        params = [ls_params(**k) for k in kws]
        for logprobs in (False, True):
            outs = []
            for s, place in ((patient, False), (hasty, False), (patient, True), (hasty, True), (hasty, False)):
                out = logits.clone() if place else torch.empty_like(logits)
                lse = torch.zeros(rows, device=dev())
                torch.cuda.synchronize()
                keep = s.process_logits(out if place else logits, params, out, log_sum_exp=lse, logprobs=logprobs, allow=a, bias=lists)
                s.synchronize()
                outs.append((out.cpu().numpy().view(np.uint32), lse.cpu().numpy().view(np.uint32)))
                del keep
            for o in outs[1:]:
                assert np.array_equal(outs[0][0], o[0]) and np.array_equal(outs[0][1], o[1]), (rows, vocab, logprobs)
        # the draws of many candidates use the same workspace
        ids = [torch.zeros(rows, dtype=torch.int32, device=dev()) for _ in range(2)]
        torch.cuda.synchronize()
        for s, out in ((patient, ids[0]), (hasty, ids[1])):
            s.sample_rows(logits, [ls_params(temperature=0.9, top_k=0, seed=r) for r in range(rows)], [3] * rows, out)
            s.synchronize()
        assert torch.equal(ids[0], ids[1])
    patient.close()
    hasty.close()


def test_rows_longer_than_the_slices_that_are_held(sampler):
    rng = np.random.default_rng(77)
    rows, vocab = 2, 600001
    x, kws, scratch, allow, lists, want = _case(sampler, rng, rows, vocab, "bf16", True, "rows", 30, [0.8])
    _, logits = _place(x, "bf16", 1, 0)
    a = torch.from_numpy(allow.view(np.int32)).to(dev())
    out, lse = torch.empty(rows, vocab, device=dev()), torch.empty(rows, device=dev())
    for logprobs in (False, True, False):
        torch.cuda.synchronize()
        keep = sampler.process_logits(logits, [ls_params(**k) for k in kws], out, log_sum_exp=lse, logprobs=logprobs,
                                      scratch=scratch, allow=a, bias=lists)
        sampler.synchronize()
        _check(out, lse, want, logprobs, vocab)
        del keep
    short = torch.empty(rows, 5000, device=dev())   # the words these rows left are gone
    torch.cuda.synchronize()
    sampler.process_logits(upload_logits(x[:, :5000].astype(F)), [ls_params()] * rows, short, log_sum_exp=lse)
    sampler.synchronize()
    _check(short, lse, [_adjusted(x[r, :5000], {}) for r in range(rows)], False, 5000)


def test_rows_that_share_a_scratch_and_leave_its_counts_alone(sampler):
    rng = np.random.default_rng(8)
    vocab = 4000
    x = rng.normal(0, 2, (3, vocab)).astype(F)
    sc, counts = _history(sampler, rng, vocab, 300)
    kw = dict(temperature=0.8, top_k=20, repetition_penalty=1.2, frequency_penalty=0.1)
    logits = upload_logits(x)
    out = torch.empty_like(logits)
    torch.cuda.synchronize()
    sampler.process_logits(logits, [ls_params(**kw)] * 3, out, scratch=[sc] * 3)
    sampler.synchronize()
    _check(out, None, [_adjusted(x[r], kw, counts) for r in range(3)], False, vocab)
    assert np.array_equal(sc.read_counts().numpy(), counts)


def test_a_captured_plan_replays(sampler):
    stream = torch.cuda.Stream()
    s = LS.Sampler(0, stream)
    rng = np.random.default_rng(2)
    rows, vocab = 5, 30011
    sc = [LS.SamplerScratch(s, vocab) for _ in range(rows)]
    counts = np.zeros((rows, vocab), dtype=np.int64)
    kw = dict(temperature=0.9, top_k=20, presence_penalty=0.4)
    x = upload_logits(rng.normal(0, 2, (rows, vocab)).astype(F))
    ids = torch.zeros(rows, dtype=torch.int32, device=dev())
    plan = s.plan(x, [ls_params(seed=r, **kw) for r in range(rows)], [0] * rows, ids, scratch=sc)
    out, lse = torch.empty_like(x), torch.empty(rows, device=dev())
    torch.cuda.synchronize()
    plan.process_logits(out, log_sum_exp=lse)
    plan.process_logits(out, log_sum_exp=lse, logprobs=True)
    s.synchronize()
    graph, sums = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.process_logits(out, log_sum_exp=lse, logprobs=True)
    with torch.cuda.graph(sums, stream=stream):
        plan.process_logits(out, log_sum_exp=lse)
    for turn in range(4):
        new = rng.normal(0, 2 + turn, (rows, vocab)).astype(F)
        x.copy_(torch.from_numpy(new))
        hist = rng.integers(0, vocab, (rows, 50)).astype(np.int32)
        torch.cuda.synchronize()
        for r in range(rows):
            sc[r].add_history(torch.from_numpy(hist[r]).to(dev()))
            counts[r] += np.bincount(hist[r], minlength=vocab)
        s.synchronize()
        want = [_adjusted(new[r], kw, counts[r]) for r in range(rows)]
        for g, lp in ((graph, True), (sums, False), (graph, True)):
            out.zero_()
            lse.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            _check(out, lse, want, lp, vocab)
    plan.close()
    s.close()


def test_what_the_python_mirror_refuses(sampler):
    x = torch.zeros(2, 100, device=dev())
    out = torch.empty(2, 100, device=dev())
    p = [ls_params()] * 2
    for bad in (dict(out=out[:1]), dict(out=out.half()), dict(out=out[:, :50]), dict(log_sum_exp=torch.zeros(3, device=dev())),
                dict(out=x.view(torch.bfloat16)[:, :100]), dict(out=x.cpu()), dict(params=[ls_params(top_p=0.0)] * 2),
                dict(params=[ls_params(presence_penalty=1.0)] * 2)):
        kw = dict(logits=x, params=p, out=out)
        kw.update(bad)
        with pytest.raises(LS.SamplerError):
            sampler.process_logits(**kw)


@pytest.mark.parametrize("temperature", [0.7, 1.3, 0.1, 1.9999999, 0.50000006, 3.0, 1e-5, 9e5, 2e6, 1e-7])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_division_is_ieee_s(sampler, temperature, dtype):
    """Quotients bit for bit: ordinary values, zeros of both signs, subnormal, tiny and huge ones, values that overflow on
    either side, infinities and NaN (worth -inf), each among ordinary neighbours and by itself."""
    rng = np.random.default_rng(5)
    vocab = 40003
    x = (rng.normal(0, 4, (3, vocab)) * np.exp2(rng.integers(-3, 4, (3, vocab)))).astype(F)
    odd = np.array([0.0, -0.0, 1e-45, -1e-45, 1.1754944e-38, -3e-39, 7.9e-31, 1e-30, -1e-30, 2.0 ** -100, -(2.0 ** -101), 1.2e30, 1.3e30,
                    -1.3e30, 2.0 ** 100, -(2.0 ** 101), 3.4028235e38, -3.4028235e38, -3.3895314e38, 1e38, -1e38, np.inf, -np.inf, np.nan], F)
    x[1, 100:4100:7] = odd[rng.integers(0, len(odd), 572)]
    x[2, : 4 * len(odd)] = np.repeat(odd, 4)
    if dtype == "bf16":
        x = W.bf16_bits_to_f32(W.to_bf16_bits(x))
    logits = upload_logits(x) if dtype == "f32" else torch.from_numpy(x).to(dev()).bfloat16()
    out, lse = torch.empty(3, vocab, device=dev()), torch.empty(3, device=dev())
    kws = [dict(temperature=temperature, top_k=5, seed=r) for r in range(3)]
    params = [ls_params(**k) for k in kws]
    want = [_adjusted(x[r], kws[r]) for r in range(3)]
    assert params[0].effective()[0] == F(temperature)
    torch.cuda.synchronize()
    for sums in (None, lse):
        keep = sampler.process_logits(logits, params, out, log_sum_exp=sums)
        sampler.synchronize()
        for r in range(3):
            assert np.array_equal(out[r].cpu().numpy().view(np.uint32), want[r].view(np.uint32)), (r, sums is None)
        del keep
    ref = _lse(want[0])
    assert abs(float(lse[0]) - ref) <= (1.25 * max(8, vocab / 1024) + 8 + abs(ref)) * U
    assert float(lse[2]) == np.inf


@pytest.mark.parametrize("vocab", [4, 1029, 8200, 30001])
@pytest.mark.parametrize("what", ["counts", "biases", "both"])
@pytest.mark.parametrize("with_sum", [False, True])
def test_every_id_is_listed(sampler, vocab, what, with_sum):
    """More ids of a wave than it gathers at once: every id counted, biased, or both, under a mask that leaves three of four."""
    rng = np.random.default_rng(vocab)
    rows = 2
    x = rng.normal(0, 3, (rows, vocab)).astype(F)
    penalties = dict(repetition_penalty=1.2, presence_penalty=0.4, frequency_penalty=0.1) if what != "biases" else {}
    kws = [dict(temperature=0.9, top_k=5, seed=r, **penalties) for r in range(rows)]
    counts, scratch = None, None
    if what != "biases":
        counts = rng.integers(1, 9, (rows, vocab)).astype(np.int32)
        scratch = [LS.SamplerScratch(sampler, vocab) for _ in range(rows)]
        for r in range(rows):
            scratch[r].write_counts(torch.from_numpy(counts[r]))
    lists = None
    if what != "counts":
        n = min(vocab, 400)   # in a run, so that a lane's ids are all of them
        lists = [[(int(i), float(d)) for i, d in zip(range(r, n), rng.normal(0, 2, n - r))] for r in range(rows)]
    allow = np.zeros((rows, (vocab + 31) // 32), np.uint32)
    allow[:] = 0xEEEEEEEE
    a = torch.from_numpy(allow.view(np.int32)).to(dev())
    logits, out = upload_logits(x), torch.empty(rows, vocab, device=dev())
    lse = torch.empty(rows, device=dev()) if with_sum else None
    torch.cuda.synchronize()
    keep = sampler.process_logits(logits, [ls_params(**k) for k in kws], out, log_sum_exp=lse, scratch=scratch, allow=a, bias=lists)
    sampler.synchronize()
    want = [_adjusted(x[r], kws[r], None if counts is None else counts[r], allow[r], None if lists is None else lists[r]) for r in range(rows)]
    _check(out, lse, want, False, vocab)
    del keep
