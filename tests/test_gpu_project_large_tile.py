"""The matrix product's tile of 256 x 256 (lily_project), at sizes that get it, against the formula in 64 bits; the bar is
test_gpu_project.py's.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

import lily_sampler as LS
from gpu_util import dev
from test_gpu_project import _check, _formula, _rows, _run


@pytest.fixture(scope="module")
def sampler():
    s = LS.Sampler(0)
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
