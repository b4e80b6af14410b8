import json
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle"),
          os.path.join(ROOT, "lily-qwen3.8-flash-next_amd", "python")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests that hold a wrong value: they run, are meant to fail, and are reported if they ever pass.
WRONG_VALUES = {
    # Nineteen of its 900 lists come to more than 1 (up to 1.16: at T = 1e-6 the teacher's sums lie at some 5e6, where f32 rounds them by up to
    # 1 / 4, and exp(1 / 4) of a share of 0.95 is 1.22).  P is 0 there, so loss / T^2 = sum p_j (log p_j - z_j / T) + (sum p) log(sum exp(z / T)), whose
    # derivative is ((sum p) q_v - p_v) / T.  The test expects (q_v - p_v) / T: off by w T (sum p - 1) q_v, 7.4e-8 where its bar is 9e-12.  The same lists
    # are held to the derivative by test_gpu_distill_gradient.py::test_lists_that_a_small_temperature_brings_beyond_all.
    "test_gpu_distill.py::test_temperatures_that_leave_one_outcome_or_all_alike[900-logits-True-1e-06]":
        "expects q - p of lists with sum p > 1, whose loss has the derivative (sum p) q - p",
}


def pytest_collection_modifyitems(items):
    for item in items:
        why = WRONG_VALUES.get(item.nodeid.split("/")[-1])
        if why is not None:
            item.add_marker(pytest.mark.xfail(reason=why, strict=True))


@pytest.fixture(scope="session")
def kat():
    with open(os.path.join(ROOT, "tests", "golden", "kat.json")) as f:
        return json.load(f)
