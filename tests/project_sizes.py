"""Products that get the tile of 256 x 256 by the plan's own choice: (rows, n, d, type of x and weight, out, residual or
None, elements behind a row of out and residual)."""
LARGE_TILE = [
    (4090, 4090, 4112, "bf16", "bf16", "bf16", 3), (4090, 4090, 4112, "bf16", "f32", "f32", 3),
    (4096, 4096, 4096, "bf16", "bf16", "bf16", 1), (4090, 4090, 4112, "bf16", "f32", "bf16", 1),
    (1020, 16380, 8208, "e4m3", "bf16", "bf16", 1), (1020, 16380, 8208, "e4m3", "bf16", "f32", 5),
    (4090, 4090, 4112, "bf16", "f32", None, 0), (1020, 16380, 8208, "e4m3", "f32", "f32", 0),
    (1020, 16380, 8208, "e4m3", "bf16", None, 0), (4096, 4096, 4096, "bf16", "bf16", "bf16", 0),
    (4096, 4096, 4096, "bf16", "f32", "f32", 0),
]
