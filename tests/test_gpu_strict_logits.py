"""Processed logits of rows in slices under LILY_SAMPLER_HANDOVER=strict, a launch for the sums and one that writes, and under
relaxed, one launch.
The bar is test_gpu_process_logits.py's; calls of every form follow each other, so that a word left behind would be found."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev, ls_params, upload_logits
from test_gpu_process_logits import _case, _check


@pytest.mark.parametrize("form", ["strict", "relaxed"])
@pytest.mark.parametrize("looks", ["", "0,0,1000000"])
@pytest.mark.parametrize("rows, vocab, dtype", [(1, 151936, "f32"), (7, 50257, "bf16"), (70, 30000, "f32"), (300, 9001, "bf16")])
def test_forms_in_turn(monkeypatch, form, looks, rows, vocab, dtype):
    monkeypatch.setenv("LILY_SAMPLER_HANDOVER", form)
    if looks:
        monkeypatch.setenv("LILY_SAMPLER_WIDE_LOOKS", looks)
    s = LS.Sampler(0)
    rng = np.random.default_rng(rows)
    x, kws, scratch, allow, lists, want = _case(s, rng, rows, vocab, dtype, True, "rows", 9, [0.7, 1.0])
    raw = upload_logits(x) if dtype == "f32" else torch.from_numpy(x).to(dev()).bfloat16()
    a = torch.from_numpy(allow.view(np.int32)).to(dev())
    params = [ls_params(**k) for k in kws]
    first = {}
    for turn in range(2):
        for logprobs in (True, False):
            for place in (True, False):
                logits = raw.clone()
                out = logits if place else torch.empty(rows, vocab, device=dev())
                lse = torch.zeros(rows, device=dev())
                torch.cuda.synchronize()
                keep = s.process_logits(logits, params, out, log_sum_exp=lse, logprobs=logprobs, scratch=scratch, allow=a, bias=lists)
                s.synchronize()
                _check(out, lse, want, logprobs, vocab)
                bits = (out.float().cpu().numpy().view(np.uint32), lse.cpu().numpy().view(np.uint32))
                before = first.setdefault((logprobs, place), bits)
                assert np.array_equal(bits[0], before[0]) and np.array_equal(bits[1], before[1])
                del keep
    # the draws of many candidates use the same workspace
    ids = torch.zeros(rows, dtype=torch.int32, device=dev())
    torch.cuda.synchronize()
    for _ in range(2):
        s.sample_rows(raw, [ls_params(temperature=0.9, top_k=0, seed=r) for r in range(rows)], [3] * rows, ids)
        s.synchronize()
        assert np.array_equal(first.setdefault("ids", ids.cpu().numpy()), ids.cpu().numpy())
    s.close()
