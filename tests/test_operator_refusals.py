"""What the operators around the head refuse, told from the descriptor alone: no GPU needed (the
descriptor is looked at before the sampler, so the calls are made without one; a call with nothing wrong
answers that the sampler is missing)."""
import ctypes as C

import pytest

import lily_sampler as LS

INVALID, RANGE = -1, -6
L = LS._lib


def _said(rc):
    return rc, L.lily_last_error().decode()


def _norm(**over):
    kw = dict(rows=4, d=64, x_dev=0x10000, x_stride=64, residual_dev=0x20000, residual_stride=64, sum_dev=0x30000,
              sum_stride=64, weight_dev=0x40000, out_dev=0x50000, out_stride=64, scales_dev=None, x_dtype=LS.BF16,
              stream_dtype=LS.BF16, weight_dtype=LS.F32, out_dtype=LS.BF16, eps=1e-6, weight_offset=0.0)
    kw.update(over)
    n = LS._Norm()
    for k, v in kw.items():
        setattr(n, k, v)
    return n


@pytest.mark.parametrize("over", [
    dict(),
    dict(rows=1, x_stride=0, residual_stride=0, sum_stride=0, out_stride=0),      # one row: strides say nothing
    dict(residual_dev=None, sum_dev=None),
    dict(weight_dev=None),
    dict(weight_offset=1.0, eps=0.0),
    dict(out_dtype=LS.E4M3, scales_dev=0x60000),
    dict(sum_dev=0x20000),                                                        # in place of the residual
    dict(sum_dev=0x10000, out_dev=0x20000),                                       # in place of both inputs
    dict(d=63, x_dev=0x10002),
    dict(d=LS.NORM_MAX_D, **{k: LS.NORM_MAX_D for k in ("x_stride", "residual_stride", "sum_stride", "out_stride")},
         rows=1, weight_dtype=LS.BF16),
    # columns side by side of one wide buffer
    dict(x_dev=0x10000, residual_dev=0x10080, sum_dev=0x10100, out_dev=0x10180,
         **{k: 256 for k in ("x_stride", "residual_stride", "sum_stride", "out_stride")}),
])
def test_a_sound_norm_only_lacks_the_sampler(over):
    rc, text = _said(L.lily_rms_norm(None, C.byref(_norm(**over))))
    assert rc == INVALID and text == "sampler is null"


@pytest.mark.parametrize("over, code, word", [
    (dict(x_dev=None), INVALID, "required"),
    (dict(out_dev=None), INVALID, "required"),
    (dict(rows=0), INVALID, "positive"),
    (dict(d=0), INVALID, "positive"),
    (dict(d=LS.NORM_MAX_D + 1), RANGE, "elements"),
    (dict(rows=0x80000000), RANGE, "elements"),
    (dict(x_dtype=LS.E4M3), INVALID, "LILY_BF16"),
    (dict(stream_dtype=3), INVALID, "LILY_BF16"),
    (dict(weight_dtype=LS.E4M3), INVALID, "LILY_BF16"),
    (dict(out_dtype=3), INVALID, "out is"),
    (dict(out_dtype=LS.E4M3), INVALID, "scales"),
    (dict(scales_dev=0x60000), INVALID, "scales"),
    (dict(residual_dev=None), INVALID, "needs a residual"),
    (dict(eps=-1e-6), INVALID, "eps"),
    (dict(eps=float("nan")), INVALID, "eps"),
    (dict(eps=float("inf")), INVALID, "eps"),
    (dict(weight_offset=float("nan")), INVALID, "eps"),
    (dict(weight_dev=None, weight_offset=1.0), INVALID, "needs weights"),
    (dict(x_stride=63), INVALID, "shorter"),
    (dict(residual_stride=63), INVALID, "shorter"),
    (dict(sum_stride=0), INVALID, "shorter"),
    (dict(out_stride=63), INVALID, "shorter"),
    (dict(x_dev=0x10001), INVALID, "multiple"),
    (dict(weight_dev=0x40002), INVALID, "multiple"),
    (dict(x_stride=1 << 62), RANGE, "address"),
    (dict(x_stride=1 << 63), RANGE, "address"),
    (dict(x_dev=(1 << 63) - 64), RANGE, "address"),
    (dict(sum_dev=0x10002), INVALID, "overlaps an input"),                   # shifted by one element
    (dict(out_dev=0x10000, out_dtype=LS.F32), INVALID, "overlaps an input"),  # another type in the same place
    (dict(out_dev=0x10000, out_stride=128), INVALID, "overlaps an input"),
    (dict(out_dev=0x40000), INVALID, "weights"),
    (dict(out_dev=0x30000), INVALID, "sum and out"),
    (dict(out_dtype=LS.E4M3, scales_dev=0x50004), INVALID, "scales"),
    (dict(out_dtype=LS.E4M3, scales_dev=0x10000), INVALID, "scales"),
    (dict(x_dev=0x10000, out_dev=0x10080 - 2, x_stride=256, out_stride=256), INVALID, "overlaps an input"),
    (dict(x_dev=0x10100, out_dev=0x10000, x_stride=160, out_stride=160), INVALID, "overlaps an input"),
])
def test_what_a_norm_refuses(over, code, word):
    rc, text = _said(L.lily_rms_norm(None, C.byref(_norm(**over))))
    assert rc == code and word in text, (rc, text)


def test_a_missing_descriptor():
    assert _said(L.lily_rms_norm(None, None))[0] == INVALID


# ---- processed logits


def _process(rows_over, out_over):
    kw = dict(rows=2, vocab=100, dtype=LS.F32, logits_dev=0x10000, row_stride=100)
    kw.update(rows_over)
    b = LS._Rows()
    n = max(1, min(kw["rows"], 64))
    params = (LS.SamplingParams * n)(*[LS.SamplingParams.greedy() for _ in range(n)])
    b.params = params
    for k, v in kw.items():
        setattr(b, k, v)
    kw = dict(out_dev=0x20000, out_stride=100, out_dtype=LS.F32, logprobs=0, log_sum_exp_dev=None)
    kw.update(out_over)
    o = LS._LogitsOut()
    for k, v in kw.items():
        setattr(o, k, v)
    return _said(L.lily_process_logits(None, C.byref(b), C.byref(o)))


@pytest.mark.parametrize("rows_over, out_over", [
    ({}, {}),
    ({}, dict(log_sum_exp_dev=0x30000, logprobs=1)),
    ({}, dict(out_dev=0x10000)),                                  # in place
    (dict(rows=9, row_stride=101), dict(out_stride=103)),
    (dict(rows=1, row_stride=100), dict(out_stride=0)),
    (dict(dtype=LS.BF16), dict(out_dtype=LS.BF16)),
    (dict(row_stride=200), dict(out_dev=0x10000 + 400, out_stride=200)),   # side by side in wider rows
])
def test_a_sound_call_for_processed_logits_only_lacks_the_sampler(rows_over, out_over):
    rc, text = _process(rows_over, out_over)
    assert rc == INVALID and text == "sampler is null", text


@pytest.mark.parametrize("rows_over, out_over, code, word", [
    (dict(rows=0), {}, INVALID, "empty"),
    (dict(vocab=0), {}, INVALID, "empty"),
    (dict(dtype=LS.E4M3), {}, INVALID, "dtype"),
    (dict(logits_dev=None), {}, INVALID, "required"),
    (dict(row_stride=99), {}, INVALID, "row_stride"),
    ({}, dict(out_dev=None), INVALID, "output"),
    ({}, dict(out_dtype=LS.E4M3), INVALID, "processed logits"),
    ({}, dict(logprobs=2), INVALID, "logprobs"),
    ({}, dict(out_stride=99), INVALID, "out_stride"),
    (dict(vocab=(1 << 24) + 1, row_stride=1 << 25), dict(out_stride=1 << 25), RANGE, "vocabularies"),
    (dict(row_stride=1 << 62), {}, RANGE, "address"),
    (dict(logits_dev=0x10002), {}, INVALID, "multiple"),
    ({}, dict(out_dev=0x20001), INVALID, "multiple"),
    ({}, dict(log_sum_exp_dev=0x30001), INVALID, "multiple"),
    ({}, dict(out_dev=0x10004), INVALID, "overlaps"),
    ({}, dict(out_dev=0x10000, out_dtype=LS.BF16), INVALID, "overlaps"),
    ({}, dict(out_dev=0x10000, out_stride=120), INVALID, "overlaps"),
    ({}, dict(log_sum_exp_dev=0x10000), INVALID, "overlaps"),
    ({}, dict(log_sum_exp_dev=0x20004), INVALID, "overlaps"),
    (dict(bias_dev=0x40000), {}, INVALID, "bias_offsets"),
])
def test_what_processed_logits_refuse(rows_over, out_over, code, word):
    rc, text = _process(rows_over, out_over)
    assert rc == code and word in text, (rc, text)


def test_a_plan_that_is_missing():
    assert _said(L.lily_plan_process_logits(None, None))[0] == INVALID


# ---- the product with an epilogue


def _project(**over):
    kw = dict(rows=4, n=48, d=64, dtype=LS.BF16, x_dev=0x10000, x_stride=64, weight_dev=0x20000, weight_stride=64,
              x_scales_dev=None, weight_scales_dev=None, bias_dev=0x30000, residual_dev=0x40000, residual_stride=48,
              out_dev=0x50000, out_stride=48, bias_dtype=LS.F32, residual_dtype=LS.BF16, out_dtype=LS.BF16, activation=1)
    kw.update(over)
    p = LS._Projection()
    for k, v in kw.items():
        setattr(p, k, v)
    return _said(L.lily_project(None, C.byref(p)))


@pytest.mark.parametrize("over", [
    dict(), dict(dtype=LS.E4M3, x_scales_dev=0x60000, weight_scales_dev=0x61000), dict(bias_dev=None), dict(residual_dev=None),
    dict(rows=1, x_stride=0, residual_stride=0, out_stride=0), dict(n=1, weight_stride=0),
    dict(out_dev=0x40000), dict(residual_dev=0x50000 + 96, residual_stride=96, out_stride=96),
    dict(activation=4), dict(d=8, x_stride=8, weight_stride=8), dict(out_dev=0x50002), dict(bias_dtype=LS.BF16, bias_dev=0x30002),
])
def test_a_sound_product_only_lacks_the_sampler(over):
    rc, text = _project(**over)
    assert rc == INVALID and text == "sampler is null", text


@pytest.mark.parametrize("over, code, word", [
    (dict(x_dev=None), INVALID, "required"),
    (dict(weight_dev=None), INVALID, "required"),
    (dict(out_dev=None), INVALID, "required"),
    (dict(rows=0), INVALID, "positive"),
    (dict(n=0), INVALID, "positive"),
    (dict(d=0), INVALID, "positive"),
    (dict(dtype=LS.F32), INVALID, "x and weight are"),
    (dict(dtype=3), INVALID, "x and weight are"),
    (dict(bias_dtype=2), INVALID, "bias, residual"),
    (dict(residual_dtype=2), INVALID, "bias, residual"),
    (dict(out_dtype=2), INVALID, "bias, residual"),
    (dict(activation=5), INVALID, "activation"),
    (dict(d=60), INVALID, "16 bytes"),
    (dict(dtype=LS.E4M3, d=56), INVALID, "16 bytes"),
    (dict(d=0x80000000, x_stride=0x80000000, weight_stride=0x80000000), RANGE, "up to"),
    (dict(rows=(1 << 24) + 1), RANGE, "up to"),
    (dict(n=(1 << 30) + 1), RANGE, "up to"),
    (dict(x_stride=56), INVALID, "shorter"),
    (dict(weight_stride=56), INVALID, "shorter"),
    (dict(out_stride=47), INVALID, "shorter"),
    (dict(residual_stride=47), INVALID, "shorter"),
    (dict(x_dev=0x10008), INVALID, "16 bytes"),
    (dict(x_stride=68), INVALID, "16 bytes"),
    (dict(weight_stride=68), INVALID, "16 bytes"),
    (dict(weight_stride=(1 << 22) + 8), RANGE, "apart"),
    (dict(x_stride=(1 << 22) + 8), RANGE, "apart"),
    (dict(out_stride=1 << 62), RANGE, "address"),
    (dict(out_dev=0x50001), INVALID, "multiple"),
    (dict(bias_dev=0x30002), INVALID, "multiple"),
    (dict(x_scales_dev=0x60002), INVALID, "multiple"),
    (dict(out_dev=0x10000), INVALID, "operand"),
    (dict(out_dev=0x20000), INVALID, "operand"),
    (dict(out_dev=0x30000), INVALID, "operand"),
    (dict(x_scales_dev=0x50000), INVALID, "operand"),
    (dict(weight_scales_dev=0x50010), INVALID, "operand"),
    (dict(out_dev=0x40002), INVALID, "residual"),
    (dict(out_dev=0x40000, out_dtype=LS.F32), INVALID, "residual"),
    (dict(out_dev=0x40000, out_stride=50), INVALID, "residual"),
])
def test_what_a_product_refuses(over, code, word):
    rc, text = _project(**over)
    assert rc == code and word in text, (rc, text)


def test_a_product_without_a_descriptor():
    assert _said(L.lily_project(None, None))[0] == INVALID


# ---- more than a launch holds (2^32 - 1 threads)


@pytest.mark.parametrize("rows, d, sound", [
    ((1 << 26) - 1, 512, True), (1 << 26, 512, False), ((1 << 26) - 1, 1, True), (1 << 26, 1, False),
    ((1 << 22) - 1, 8192, True), (1 << 22, 8192, False), ((1 << 22) - 1, 32768, True), (1 << 22, 32768, False),
    ((1 << 32) - 1, 513, False),
])
def test_the_most_rows_of_a_norm(rows, d, sound):
    far = 1 << 44
    rc, text = _said(L.lily_rms_norm(None, C.byref(_norm(rows=rows, d=d, x_stride=d, residual_stride=d, sum_stride=d, out_stride=d,
                                                         x_dev=far, residual_dev=2 * far, sum_dev=3 * far, weight_dev=0x40000,
                                                         out_dev=4 * far))))
    assert (rc, text) == (INVALID, "sampler is null") if sound else rc == RANGE and "up to" in text, (rc, text)


@pytest.mark.parametrize("rows, n, sound", [
    (1, 1 << 26, True), (1, (1 << 26) + 1, False), (1 << 24, 64, True), (1 << 24, 63 * 64, True), (1 << 24, 64 * 64, False),
    (1 << 10, 1 << 26, False), (960, 1 << 26, True), (65, 1 << 26, True),
])
def test_the_most_tiles_of_a_product(rows, n, sound):
    far = 1 << 44
    rc, text = _project(rows=rows, n=n, x_dev=far, weight_dev=2 * far, residual_dev=3 * far, out_dev=4 * far, residual_stride=n,
                        out_stride=n, bias_dev=5 * far)
    assert (rc, text) == (INVALID, "sampler is null") if sound else rc == RANGE and "up to" in text, (rc, text)
