"""What the operators that train and serve a draft head refuse, told from the descriptor alone: no GPU needed (the descriptor is
looked at before the sampler; a call with nothing wrong answers that the sampler is missing)."""
import ctypes as C

import pytest

import lily_sampler as LS

INVALID, RANGE = -1, -6
L = LS._lib
NAN, INF = float("nan"), float("inf")


def _said(rc):
    return rc, L.lily_last_error().decode()


def _call(entry, struct, defaults, over):
    s = struct()
    for k, v in {**defaults, **over}.items():
        setattr(s, k, v)
    return _said(getattr(L, entry)(None, C.byref(s)))


LAYER = dict(rows=4, d=64, x_dev=0x10000, x_stride=64, residual_dev=0x20000, residual_stride=64, sum_dev=0x30000, sum_stride=64,
             weight_dev=0x40000, bias_dev=0x41000, out_dev=0x50000, out_stride=64, scales_dev=None, scales_stride=0, mean_dev=0x60000,
             rstd_dev=0x61000, x_dtype=LS.BF16, stream_dtype=LS.BF16, weight_dtype=LS.F32, out_dtype=LS.BF16, scale_block=0, eps=1e-5)
GRAD = dict(rows=4, d=64, grad_dev=0x10000, grad_stride=64, h_dev=0x20000, h_stride=64, mean_dev=0x60000, rstd_dev=0x61000, weight_dev=0x40000,
            past_dev=0x30000, past_stride=64, grad_x_dev=0x50000, grad_x_stride=64, grad_weight_dev=0x70000, grad_bias_dev=0x71000,
            grad_dtype=LS.BF16, h_dtype=LS.BF16, weight_dtype=LS.F32, grad_x_dtype=LS.BF16, accumulate=0)
BLOCKS = dict(rows=4, d=200, x_dev=0x10000, x_stride=200, out_dev=0x20000, out_stride=200, scales_dev=0x30000, scales_stride=2, x_dtype=LS.BF16,
              block_rows=1)
PRODUCT = dict(rows=4, n=200, d=272, activation=1, x_dev=0x10000, x_stride=272, x_scales_dev=0x11000, x_scales_stride=3, weight_dev=0x20000,
               weight_stride=272, weight_scales_dev=0x31000, weight_scales_stride=3, bias_dev=0x32000, residual_dev=0x40000, residual_stride=200,
               out_dev=0x50000, out_stride=200, bias_dtype=LS.F32, residual_dtype=LS.BF16, out_dtype=LS.BF16, reserved=0)
DISTILL = dict(rows=4, vocab=100, logits_dev=0x10000, logits_stride=100, ids_dev=0x20000, ids_stride=8, values_dev=0x30000, values_stride=8,
               counts_dev=0x40000, teacher_lse_dev=None, row_weights_dev=0x41000, loss_dev=0x50000, stats_dev=0x51000, grad_dev=0x60000, grad_stride=100,
               k=8, teacher=0, rest=0, logits_dtype=LS.F32, values_dtype=LS.F32, grad_dtype=LS.F32, temperature=1.0, grad_scale=1.0)
BACKWARD = dict(DISTILL, loss_dev=None)
ENTRIES = dict(layer=("lily_layer_norm", LS._Layer, LAYER), grad=("lily_layer_norm_backward", LS._LayerGrad, GRAD),
               blocks=("lily_quantize_blocks", LS._Blocks, BLOCKS), product=("lily_project_blocks", LS._BlockProjection, PRODUCT),
               distill=("lily_distill", LS._Distillation, DISTILL), backward=("lily_distill_backward", LS._Distillation, BACKWARD))

SOUND = [
    ("layer", {}), ("layer", dict(rows=1, x_stride=0, residual_stride=0, sum_stride=0, out_stride=0)),
    ("layer", dict(residual_dev=None, sum_dev=None)), ("layer", dict(weight_dev=None, bias_dev=None)), ("layer", dict(mean_dev=None, rstd_dev=None, eps=0.0)),
    ("layer", dict(out_dtype=LS.E4M3, scales_dev=0x68000)), ("layer", dict(out_dtype=LS.E4M3, scales_dev=0x68000, scale_block=128, scales_stride=1)),
    ("layer", dict(sum_dev=0x20000)), ("layer", dict(sum_dev=0x10000, out_dev=0x20000)), ("layer", dict(d=63, x_dev=0x10002)),
    ("layer", dict(x_dev=0x10000, residual_dev=0x10080, sum_dev=0x10100, out_dev=0x10180, x_stride=256, residual_stride=256, sum_stride=256, out_stride=256)),
    ("grad", {}), ("grad", dict(rows=1, grad_stride=0, h_stride=0, past_stride=0, grad_x_stride=0)), ("grad", dict(past_dev=None)),
    ("grad", dict(past_dev=None, grad_x_dev=None)), ("grad", dict(grad_weight_dev=None, grad_bias_dev=None)), ("grad", dict(weight_dev=None)),
    ("grad", dict(grad_x_dev=0x10000)), ("grad", dict(grad_x_dev=0x20000)), ("grad", dict(grad_x_dev=0x30000)), ("grad", dict(accumulate=1, grad_weight_dev=None)),
    ("blocks", {}), ("blocks", dict(block_rows=128, scales_stride=0)), ("blocks", dict(rows=1, x_stride=0, out_stride=0, scales_stride=0)),
    ("blocks", dict(x_dtype=LS.F32, x_dev=0x10004, out_dev=0x20001)),
    ("product", {}), ("product", dict(rows=1, x_stride=0, x_scales_stride=0, residual_stride=0, out_stride=0)), ("product", dict(bias_dev=None, residual_dev=None)),
    ("product", dict(out_dev=0x40000)), ("product", dict(n=1, weight_stride=0, weight_scales_stride=0)), ("product", dict(n=128, weight_scales_stride=0)),
    ("distill", {}), ("distill", dict(grad_dev=0x10000)), ("distill", dict(grad_dev=None)), ("distill", dict(loss_dev=None, stats_dev=None)),
    ("distill", dict(rest=1, teacher_lse_dev=0x42000)), ("distill", dict(rest=1, teacher=1)), ("distill", dict(counts_dev=None, row_weights_dev=None)),
    ("distill", dict(rows=1, logits_stride=0, ids_stride=0, values_stride=0, grad_stride=0)), ("distill", dict(k=1024, ids_stride=1024, values_stride=1024, ids_dev=0x100000, values_dev=0x200000)),
    ("backward", {}), ("backward", dict(grad_dev=0x10000)),
]


@pytest.mark.parametrize("which, over", SOUND)
def test_a_sound_call_only_lacks_the_sampler(which, over):
    rc, text = _call(*ENTRIES[which], over)
    assert rc == INVALID and text == "sampler is null", text


FAULTS = [
    # layer norm
    ("layer", dict(x_dev=None), INVALID, "required"), ("layer", dict(out_dev=None), INVALID, "required"), ("layer", dict(rows=0), INVALID, "positive"),
    ("layer", dict(d=0), INVALID, "positive"), ("layer", dict(d=LS.NORM_MAX_D + 1), RANGE, "elements"), ("layer", dict(rows=0x80000000), RANGE, "up to"),
    ("layer", dict(x_dtype=LS.E4M3), INVALID, "LILY_BF16"), ("layer", dict(stream_dtype=3), INVALID, "LILY_BF16"), ("layer", dict(weight_dtype=2), INVALID, "LILY_BF16"),
    ("layer", dict(out_dtype=3), INVALID, "out is"), ("layer", dict(out_dtype=LS.E4M3), INVALID, "scales"), ("layer", dict(scales_dev=0x68000), INVALID, "scales"),
    ("layer", dict(scale_block=128), INVALID, "scale_block"), ("layer", dict(out_dtype=LS.E4M3, scales_dev=0x68000, scale_block=64), INVALID, "scale_block"),
    ("layer", dict(d=200, x_stride=200, residual_stride=200, sum_stride=200, out_stride=200, out_dtype=LS.E4M3, scales_dev=0x68000, scale_block=128, scales_stride=1), INVALID, "shorter"),
    ("layer", dict(residual_dev=None), INVALID, "needs a residual"), ("layer", dict(eps=-1.0), INVALID, "eps"), ("layer", dict(eps=NAN), INVALID, "eps"), ("layer", dict(eps=INF), INVALID, "eps"),
    ("layer", dict(x_stride=63), INVALID, "shorter"), ("layer", dict(residual_stride=63), INVALID, "shorter"), ("layer", dict(sum_stride=0), INVALID, "shorter"),
    ("layer", dict(out_stride=63), INVALID, "shorter"), ("layer", dict(x_dev=0x10001), INVALID, "multiple"), ("layer", dict(bias_dev=0x41002), INVALID, "multiple"),
    ("layer", dict(mean_dev=0x60002), INVALID, "multiple"), ("layer", dict(x_stride=1 << 62), RANGE, "address"), ("layer", dict(sum_dev=0x10002), INVALID, "overlaps an input"),
    ("layer", dict(out_dev=0x10000, out_dtype=LS.F32), INVALID, "overlaps an input"), ("layer", dict(out_dev=0x40000), INVALID, "weight or bias"),
    ("layer", dict(mean_dev=0x41000), INVALID, "weight or bias"), ("layer", dict(mean_dev=0x10000), INVALID, "overlap an input"), ("layer", dict(mean_dev=0x61000), INVALID, "two outputs"),
    ("layer", dict(rstd_dev=0x50000), INVALID, "two outputs"), ("layer", dict(sum_dev=0x50000), INVALID, "two outputs"),
    ("layer", dict(out_dtype=LS.E4M3, scales_dev=0x50010), INVALID, "two outputs"),
    # its backward pass
    ("grad", dict(grad_dev=None), INVALID, "required"), ("grad", dict(h_dev=None), INVALID, "required"), ("grad", dict(mean_dev=None), INVALID, "required"),
    ("grad", dict(rstd_dev=None), INVALID, "required"), ("grad", dict(past_dev=None, grad_x_dev=None, grad_weight_dev=None, grad_bias_dev=None), INVALID, "nothing"),
    ("grad", dict(rows=0), INVALID, "positive"), ("grad", dict(d=LS.NORM_MAX_D + 1), RANGE, "elements"), ("grad", dict(rows=1 << 31), RANGE, "up to"),
    ("grad", dict(grad_dtype=2), INVALID, "LILY_BF16"), ("grad", dict(h_dtype=2), INVALID, "LILY_BF16"), ("grad", dict(weight_dtype=2), INVALID, "LILY_BF16"),
    ("grad", dict(grad_x_dtype=2), INVALID, "LILY_BF16"), ("grad", dict(grad_x_dev=None), INVALID, "past needs"), ("grad", dict(accumulate=2), INVALID, "accumulate"),
    ("grad", dict(grad_stride=63), INVALID, "shorter"), ("grad", dict(h_stride=63), INVALID, "shorter"), ("grad", dict(past_stride=63), INVALID, "shorter"),
    ("grad", dict(grad_x_stride=63), INVALID, "shorter"), ("grad", dict(grad_weight_dev=0x70002), INVALID, "multiple"), ("grad", dict(h_stride=1 << 62), RANGE, "address"),
    ("grad", dict(grad_x_dev=0x10002), INVALID, "grad_x overlaps"), ("grad", dict(grad_x_dev=0x20000, grad_x_dtype=LS.F32), INVALID, "grad_x overlaps"),
    ("grad", dict(grad_x_dev=0x40000), INVALID, "grad_x overlaps"), ("grad", dict(grad_x_dev=0x60000), INVALID, "grad_x overlaps"),
    ("grad", dict(grad_weight_dev=0x10000), INVALID, "gradient of weight"), ("grad", dict(grad_bias_dev=0x40000), INVALID, "gradient of weight"),
    ("grad", dict(grad_bias_dev=0x50000), INVALID, "gradient of weight"), ("grad", dict(grad_bias_dev=0x70010), INVALID, "weight and bias overlap"),
    # quantisation
    ("blocks", dict(x_dev=None), INVALID, "required"), ("blocks", dict(out_dev=None), INVALID, "required"), ("blocks", dict(scales_dev=None), INVALID, "required"),
    ("blocks", dict(rows=0), INVALID, "positive"), ("blocks", dict(d=0), INVALID, "positive"), ("blocks", dict(x_dtype=2), INVALID, "x is"),
    ("blocks", dict(block_rows=64), INVALID, "block_rows"), ("blocks", dict(x_stride=199), INVALID, "shorter"), ("blocks", dict(out_stride=199), INVALID, "shorter"),
    ("blocks", dict(scales_stride=1), INVALID, "shorter"), ("blocks", dict(x_dev=0x10001), INVALID, "multiple"), ("blocks", dict(scales_dev=0x30002), INVALID, "multiple"),
    ("blocks", dict(x_stride=1 << 62), RANGE, "address"), ("blocks", dict(out_dev=0x10000), INVALID, "overlap"), ("blocks", dict(scales_dev=0x20004), INVALID, "overlap"),
    ("blocks", dict(scales_dev=0x10004), INVALID, "overlap"), ("blocks", dict(rows=1 << 28, d=1, x_stride=1, out_stride=1), RANGE, "up to"),
    # the product
    ("product", dict(x_dev=None), INVALID, "required"), ("product", dict(weight_dev=None), INVALID, "required"), ("product", dict(out_dev=None), INVALID, "required"),
    ("product", dict(x_scales_dev=None), INVALID, "required"), ("product", dict(weight_scales_dev=None), INVALID, "required"), ("product", dict(rows=0), INVALID, "positive"),
    ("product", dict(n=0), INVALID, "positive"), ("product", dict(d=0), INVALID, "positive"), ("product", dict(bias_dtype=2), INVALID, "bias, residual"),
    ("product", dict(out_dtype=2), INVALID, "bias, residual"), ("product", dict(residual_dtype=2), INVALID, "bias, residual"), ("product", dict(activation=5), INVALID, "activation"),
    ("product", dict(reserved=1), INVALID, "reserved"), ("product", dict(d=264), INVALID, "16"), ("product", dict(rows=(1 << 24) + 1), RANGE, "up to"),
    ("product", dict(n=(1 << 26) + 1), RANGE, "up to"), ("product", dict(x_stride=256), INVALID, "shorter"), ("product", dict(weight_stride=256), INVALID, "shorter"),
    ("product", dict(x_scales_stride=2), INVALID, "shorter"), ("product", dict(weight_scales_stride=2), INVALID, "shorter"), ("product", dict(out_stride=199), INVALID, "shorter"),
    ("product", dict(residual_stride=199), INVALID, "shorter"), ("product", dict(x_dev=0x10008), INVALID, "16 bytes"), ("product", dict(weight_stride=280), INVALID, "16 bytes"),
    ("product", dict(weight_stride=(1 << 23) + 16), RANGE, "apart"), ("product", dict(x_scales_stride=(1 << 21) + 1), RANGE, "apart"),
    ("product", dict(weight_scales_stride=1 << 30), RANGE, "apart"), ("product", dict(x_scales_dev=0x11002), INVALID, "multiple"), ("product", dict(out_dev=0x50001), INVALID, "multiple"),
    ("product", dict(out_dev=0x10000), INVALID, "operand"), ("product", dict(out_dev=0x11000), INVALID, "operand"), ("product", dict(out_dev=0x31000), INVALID, "operand"),
    ("product", dict(out_dev=0x32000), INVALID, "operand"), ("product", dict(out_dev=0x40002), INVALID, "residual"), ("product", dict(out_stride=1 << 62), RANGE, "address"),
    # distillation
    ("distill", dict(logits_dev=None), INVALID, "required"), ("distill", dict(ids_dev=None), INVALID, "required"), ("distill", dict(values_dev=None), INVALID, "required"),
    ("distill", dict(loss_dev=None, stats_dev=None, grad_dev=None), INVALID, "nothing"), ("distill", dict(rows=0), INVALID, "positive"), ("distill", dict(vocab=0), INVALID, "positive"),
    ("distill", dict(k=0), INVALID, "positive"), ("distill", dict(vocab=(1 << 24) + 1, logits_stride=1 << 25, grad_stride=1 << 25), RANGE, "vocabularies"),
    ("distill", dict(k=1025, ids_stride=2000, values_stride=2000), RANGE, "entries"), 
    ("distill", dict(logits_dtype=2), INVALID, "logits, values"), ("distill", dict(values_dtype=2), INVALID, "logits, values"), ("distill", dict(grad_dtype=2), INVALID, "logits, values"),
    ("distill", dict(teacher=2), INVALID, "teacher is"), ("distill", dict(rest=2), INVALID, "rest 0 or 1"), ("distill", dict(rest=1), INVALID, "teacher_lse"),
    ("distill", dict(teacher_lse_dev=0x42000), INVALID, "teacher_lse"), ("distill", dict(rest=1, teacher=1, teacher_lse_dev=0x42000), INVALID, "teacher_lse"),
    ("distill", dict(temperature=0.0), INVALID, "temperature"), ("distill", dict(temperature=-1.0), INVALID, "temperature"), ("distill", dict(temperature=NAN), INVALID, "temperature"),
    ("distill", dict(temperature=1e-38), INVALID, "temperature"), ("distill", dict(temperature=1e-40), INVALID, "temperature"),
    ("distill", dict(temperature=INF), INVALID, "temperature"), ("distill", dict(grad_scale=INF), INVALID, "grad_scale"), ("distill", dict(logits_stride=99), INVALID, "shorter"),
    ("distill", dict(ids_stride=7), INVALID, "shorter"), ("distill", dict(values_stride=7), INVALID, "shorter"), ("distill", dict(grad_stride=99), INVALID, "shorter"),
    ("distill", dict(ids_dev=0x20002), INVALID, "multiple"), ("distill", dict(stats_dev=0x51002), INVALID, "multiple"), ("distill", dict(logits_stride=1 << 62), RANGE, "address"),
    ("distill", dict(grad_dev=0x10004), INVALID, "without being them"), ("distill", dict(grad_dev=0x10000, grad_dtype=LS.BF16), INVALID, "without being them"),
    ("distill", dict(grad_dev=0x10000, grad_stride=128), INVALID, "without being them"), ("distill", dict(grad_dev=0x20000), INVALID, "overlaps an input"),
    ("distill", dict(loss_dev=0x41000), INVALID, "overlaps an input"), ("distill", dict(stats_dev=0x30000), INVALID, "overlaps an input"), ("distill", dict(loss_dev=0x10000), INVALID, "overlap"),
    ("distill", dict(loss_dev=0x51000), INVALID, "overlap"), ("distill", dict(stats_dev=0x60000), INVALID, "overlap"),
    ("backward", dict(stats_dev=None), INVALID, "requires"), ("backward", dict(grad_dev=None), INVALID, "requires"), ("backward", dict(loss_dev=0x50000), INVALID, "no loss"),
    ("backward", dict(grad_dev=0x51000), INVALID, "overlap"),
]


@pytest.mark.parametrize("which, over, code, word", FAULTS)
def test_what_is_refused(which, over, code, word):
    rc, text = _call(*ENTRIES[which], over)
    assert rc == code and word in text, (rc, text)


@pytest.mark.parametrize("which", list(ENTRIES))
def test_a_missing_descriptor(which):
    assert _said(getattr(L, ENTRIES[which][0])(None, None))[0] == INVALID


@pytest.mark.parametrize("rows, d, block_rows, sound", [
    ((1 << 28) - 1, 1, 1, True), (1 << 28, 1, 1, False), ((1 << 27) - 1, 200, 1, True), (1 << 27, 200, 1, False), ((1 << 31) - 128, 128, 128, True),
    (1 << 31, 128, 128, False),
])
def test_the_most_blocks(rows, d, block_rows, sound):
    far = 1 << 48
    rc, text = _call(*ENTRIES["blocks"], dict(rows=rows, d=d, block_rows=block_rows, x_dev=far, out_dev=2 * far, scales_dev=3 * far, x_stride=d, out_stride=d))
    assert (rc, text) == (INVALID, "sampler is null") if sound else rc == RANGE and "up to" in text, (rc, text)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("d, sound", [(0xffffff80, True), (0xffffff81, False), (0xffffff82, False), (0xffffffff, False)])
def test_the_longest_rows_of_blocks(d, sound, block_rows):
    """Blocks of a row are counted, and its pieces of eight looked at, in 32 bits.  (2^25 blocks of rows are more than a call takes.)"""
    far = 1 << 48
    rc, text = _call(*ENTRIES["blocks"], dict(rows=1, d=d, block_rows=block_rows, x_dev=far, out_dev=2 * far, scales_dev=3 * far))
    assert (rc, text) == (INVALID, "sampler is null") if sound and block_rows == 1 else rc == RANGE and "up to" in text, (rc, text)
