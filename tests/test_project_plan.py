"""Which kernel a matrix product gets (csrc/project_plan.h, built for the host; no GPU needed): the sizes that the tests
of the large tile and the benchmark rely on, and what every choice must keep to."""
import os
import random
import subprocess
import sys

import pytest

from project_sizes import LARGE_TILE

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "perf"))
PART_FLOATS = 1 << 23
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1, None: 0}

PROGRAM = r"""
#include <cstdio>
#include "project_plan.h"
// a line: rows n d e4m3 out_bf16 residual (0, 2, 4 bytes an element) pad (of x and weight, elements) part_floats tile
int main() {
    unsigned rows, n, d, e4m3, out_bf16, residual, pad, tile;
    unsigned long long floats;
    while (std::scanf("%u %u %u %u %u %u %u %llu %u", &rows, &n, &d, &e4m3, &out_bf16, &residual, &pad, &floats, &tile) == 9) {
        lily_projection p = {};
        p.rows = rows, p.n = n, p.d = d;
        p.dtype = e4m3 ? LILY_E4M3 : LILY_BF16;
        p.x_stride = p.weight_stride = (unsigned long long)d + pad;
        p.out_stride = p.residual_stride = n;
        p.out_dtype = out_bf16 ? LILY_BF16 : LILY_F32;
        p.residual_dtype = residual == 2 ? LILY_BF16 : LILY_F32;
        p.residual_dev = residual ? reinterpret_cast<const void*>(1ull << 40) : nullptr;
        lily::ProjectWorkspace ws;
        ws.part = nullptr;
        ws.part_floats = floats;
        ws.tile = tile;
        const lily::ProjectPlan plan = lily::project_plan(lily::project_args(p, ws), ws);
        std::printf("%u %u\n", plan.tile, plan.splits);
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    where = tmp_path_factory.mktemp("plan")
    src, exe = where / "plan.cpp", where / "plan"
    src.write_text(PROGRAM)
    csrc = os.path.join(ROOT, "lily-qwen3.8-flash-next_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", csrc, "-I", "/opt/rocm/include", str(src), "-o", str(exe)],
                   check=True)

    def ask(products):
        """[(rows, n, d, dtype, out, residual, pad, part_floats, tile)] -> [(tile, parts of d)]"""
        lines = "".join(f"{r} {n} {d} {int(t == 'e4m3')} {int(o == 'bf16')} {SIZE[res]} {pad} {floats} {tile}\n"
                        for r, n, d, t, o, res, pad, floats, tile in products)
        out = subprocess.run([str(exe)], input=lines, capture_output=True, text=True, check=True, timeout=60).stdout
        answers = [tuple(int(v) for v in line.split()) for line in out.splitlines()]
        assert len(answers) == len(products)
        return answers

    return ask


def test_the_large_tile_s_tests_get_it(plan):
    for size, answer in zip(LARGE_TILE, plan([s[:6] + (0, PART_FLOATS, 0) for s in LARGE_TILE])):
        assert answer == (256, 1), (size, answer)


def test_the_benchmark_s_prefill_gets_the_large_tile(plan):
    import operators
    cases = [c for c in operators.listed() if c["kind"] == "project"]
    asked = [(c["rows"], c["n"], c["d"], c["dtype"], c["out"], c["out"] if c["residual"] else None, c["pad"], PART_FLOATS, 0) for c in cases]
    got = {c["name"]: a[0] for c, a in zip(cases, plan(asked))}
    assert got["prefill_bf16_b8192"] == 256 and got["prefill_e4m3_b8192"] == 256
    assert got["draft_block_b1"] == 0 and got["draft_block_b12"] == 0 and got["head_e4m3_b4"] == 0
    assert got["layer_e4m3_b100"] in (64, 128)


def test_every_choice_keeps_to_the_kernels_limits(plan):
    """Parts of d fit the workspace and have four lines of 128 bytes each; up to 16 rows one kernel takes all; the tile
    that is asked for is the one that comes; launches stay within 2^32 - 1 threads."""
    rng = random.Random(1)
    products = []
    while len(products) < 20000:
        rows, n = int(2 ** rng.uniform(0, 24)), int(2 ** rng.uniform(0, 26))
        dtype = rng.choice(["bf16", "e4m3"])
        d = 16 * int(2 ** rng.uniform(0, 18))
        if ((rows + 63) // 64) * ((n + 63) // 64) >= 1 << 24 or d * SIZE[dtype] > 1 << 23:
            continue
        products.append((rows, n, d, dtype, rng.choice(["f32", "bf16"]), rng.choice([None, "f32", "bf16"]), rng.choice([0, 16, 24]),
                         rng.choice([PART_FLOATS, 1 << 16, 0]), rng.choice([0, 0, 64, 128, 256])))
    for (rows, n, d, dtype, _, _, _, floats, forced), (tile, parts) in zip(products, plan(products)):
        case = (rows, n, d, dtype, floats, forced, tile, parts)
        lines = (d * SIZE[dtype] + 127) // 128
        assert tile in (0, 64, 128, 256) and 1 <= parts <= 16, case
        assert tile != 0 or rows <= 64, case
        assert rows > 16 or tile == 0, case
        assert rows <= 16 or forced in (0, tile), case
        if parts > 1:
            assert tile in (64, 128) and lines >= 4 * parts and parts * rows * ((n + 3) // 4 * 4) <= floats, case
        groups = (n + 15) // 16 * 2 if tile == 0 else ((rows + tile - 1) // tile) * ((n + tile - 1) // tile) * parts
        assert groups * 256 < 1 << 32, case
