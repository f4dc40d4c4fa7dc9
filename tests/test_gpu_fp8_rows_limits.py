"""8-bit rows at the ends of what their calls take: sizes that pass a launch's threads.
Tolerances as in test_gpu_fp8_rows."""
import pytest
import torch

from test_gpu_fp8_rows import gpu_near, ordered_ctx  # noqa: F401
from test_gpu_fp8_rows_tiles import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("special", [False, True])
def test_products_of_more_outputs_than_a_launch_has_threads(ctx, special):
    """65600 x 65552 outputs.  With a code of +-480 in the weight the vector kernel does
    them, 16 x 16 a workgroup: more than 2^24 of them."""
    n, rows, cols = 65600, 65552, 128
    c = Case(ctx, 1, n, rows, cols)
    if special:
        ctx.release(c.h)
        c.codes[rows - 1, 5], c.codes[40000, 127] = 0x7F, 0xFF
        torch.cuda.synchronize()
        c.h = ctx.store_fp8_device(c.codes.data_ptr(), rows, cols, c.scales.data_ptr(), *c.scales.shape)
    y = torch.full((n + 1, rows), 5.0, dtype=torch.bfloat16, device="cuda")
    ctx.fp8_rows_mm_async(c.h, 0, rows, c.rows.c, n, y.data_ptr(), rows, True)
    ctx.synchronize()
    assert bool((y[n] == 5.0).all())
    x, w = c.x(), c.w(0, rows)
    for a, b in ((0, 300), (n // 2, n // 2 + 17), (n - 1000, n)):
        gpu_near(y[a:b], x[a:b], w, True, cols)
    for a, b in ((0, 20), (40000, 40001), (rows - 17, rows)):
        gpu_near(y[:n, a:b], x, w[a:b], True, cols)
    c.close()
