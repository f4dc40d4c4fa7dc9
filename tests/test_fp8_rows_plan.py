"""CPU checks of how products of 8-bit rows are done: the rule that picks a kernel
needs no device.  Also the sizes that calls on rows are refused from on."""
import ctypes

import pytest

import wohper_amd as wa
from test_fp8_rows_host import every_row_call, lib_and_ctx, rows  # noqa: F401

EMPTY, SHAPE, ARGUMENT, UNSUPPORTED = 1, 2, 13, 15
VECTOR, THIN, TILE, HALF, TALL = range(5)


def plan(n, rows, cols, groups=0, f32=False, special=False, bf16=True):
    """Status, then kernel, ranges of columns, workgroups of each and most tiles (groups 0: without lists)."""
    p = (ctypes.c_uint64 * 4)()
    status = wa.load_library().wh_debug_fp8_rows_plan(n, max(groups, 1), int(groups > 0), rows, cols, int(f32), int(special),
                                                      int(bf16), p)
    return (status, *p)


@pytest.mark.parametrize("call,kind", [
    (dict(n=1, rows=4096, cols=4096), THIN), (dict(n=84, rows=4096, cols=4096, groups=64, bf16=False), THIN),
    (dict(n=333, rows=32768, cols=1024, f32=True, bf16=False), TILE), (dict(n=128, rows=4096, cols=4096), TILE),
    (dict(n=2048, rows=4096, cols=4096), HALF), (dict(n=4096, rows=4096, cols=8192), TALL),
    (dict(n=24000, rows=4096, cols=4096, groups=64), TALL), (dict(n=4096, rows=4096, cols=8192, f32=True), TILE),
    (dict(n=4096, rows=4096, cols=8192, special=True), VECTOR)])
def test_kernels_of_sizes(call, kind):
    status, got, splits, grid, tiles = plan(**call)
    assert status == 0 and got == kind and splits >= 1 and 1 <= grid <= tiles + 7


def test_refusals():
    lib, p = wa.load_library(), (ctypes.c_uint64 * 4)()
    assert lib.wh_debug_fp8_rows_plan(1, 1, 0, 16, 128, 0, 0, 0, None) == ARGUMENT
    for zero in range(4):
        sizes = [4, 1, 16, 128]
        sizes[zero] = 0
        assert lib.wh_debug_fp8_rows_plan(sizes[0], sizes[1], 0, sizes[2], sizes[3], 0, 0, 0, p) == EMPTY
    assert plan(1, 16, 192)[0] == SHAPE
    assert plan(1 << 31, 16, 128)[0] == plan(1, 1 << 23, 128, groups=1024)[0] == plan(1, 16, 128, groups=1025)[0] == UNSUPPORTED


@pytest.mark.parametrize("n,rows,cols,groups", [(65600, 65552, 128, 0), (1 << 21, 1 << 16, 128, 0), (3, 1 << 30, 128, 0),
                                                ((1 << 31) - 1, 16, 256, 0), (1 << 24, 1 << 13, 128, 1024), (1 << 20, 1 << 18, 640, 64)])
@pytest.mark.parametrize("bf16", [False, True])
def test_sizes_that_are_taken_do_not_depend_on_codes(n, rows, cols, groups, bf16):
    """Above 2^32 outputs too, a thread each in the vector kernel."""
    for special in (False, True):
        status, kind, splits, grid, tiles = plan(n, rows, cols, groups, special=special, bf16=bf16)
        assert status == 0 and grid * splits * (512 if kind == THIN else 256) < 1 << 32
        assert kind == VECTOR if special else grid >= tiles or kind in (VECTOR, HALF, TALL)


def test_blocks_of_a_call_are_counted(lib_and_ctx):  # noqa: F811
    """268435440 blocks, as the header says: one more is refused before the context is touched."""
    cols = 128 * 268435441
    wide = rows(stride=cols, scale_stride=268435444)
    assert every_row_call(*lib_and_ctx, r=wide, n=1, cols=cols, stride=cols) == [UNSUPPORTED] * 3
    assert every_row_call(*lib_and_ctx, n=134217721) == [UNSUPPORTED] * 3
