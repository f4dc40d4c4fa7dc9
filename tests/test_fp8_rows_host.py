"""CPU checks of the 8-bit rows' entry points: every refusal that needs no tensor.
A refused call returns before it touches the context, so a block of zeros stands
in for one."""
import ctypes

import pytest

import wohper_amd as wa

EMPTY, SHAPE, SMALL, ARGUMENT, UNSUPPORTED = 1, 2, 5, 13, 15
DEV = 0x10000  # an aligned address that a refused call never reads


@pytest.fixture
def lib_and_ctx():
    return wa.load_library(), ctypes.cast(ctypes.create_string_buffer(1 << 16), ctypes.c_void_p)


def rows(**kw):
    d = dict(codes=DEV, stride=256, scales=DEV, scale_stride=4)
    d.update(kw)
    return wa.WhFp8Rows(d["codes"], d["stride"], d["scales"], d["scale_stride"])


ROWS = [
    (dict(codes=None), ARGUMENT), (dict(scales=None), ARGUMENT), (dict(codes=DEV + 8), ARGUMENT),
    (dict(scales=DEV + 2), ARGUMENT), (dict(stride=264), ARGUMENT), (dict(scale_stride=6), ARGUMENT),
    (dict(stride=240), SHAPE), (dict(scale_stride=0), SHAPE), (dict(stride=1 << 41), UNSUPPORTED),
    (dict(scale_stride=1 << 41), UNSUPPORTED),
]
CALLS = [
    (dict(x=None), ARGUMENT), (dict(x=DEV + 2), ARGUMENT), (dict(x=DEV + 1, bf16=1), ARGUMENT), (dict(stride=255), SHAPE),
    (dict(stride=1 << 41), UNSUPPORTED), (dict(cols=0), EMPTY), (dict(cols=192), SHAPE), (dict(n=1 << 31), UNSUPPORTED),
    (dict(n=1 << 28), UNSUPPORTED), (dict(r=None), ARGUMENT),
]


def every_row_call(lib, ctx, x=DEV, stride=256, bf16=0, n=3, cols=256, r="rows"):
    r = rows() if r == "rows" else r
    p = ctypes.byref(r) if r is not None else None
    return [lib.wh_fp8_quant_rows_async(ctx, x, stride, bf16, n, cols, p),
            lib.wh_fp8_swiglu_rows_async(ctx, x, DEV, stride, bf16, n, cols, 10.0, p),
            lib.wh_fp8_read_rows_async(ctx, p, n, cols, x, stride, bf16)]


@pytest.mark.parametrize("change,status", ROWS)
def test_descriptors_refused(lib_and_ctx, change, status):
    assert every_row_call(*lib_and_ctx, r=rows(**change)) == [status] * 3


@pytest.mark.parametrize("change,status", CALLS)
def test_row_calls_refused(lib_and_ctx, change, status):
    assert every_row_call(*lib_and_ctx, **change) == [status] * 3


def test_no_rows_are_no_work(lib_and_ctx):
    assert every_row_call(*lib_and_ctx, n=0, x=None, r=rows(codes=None, scales=None)) == [0] * 3
    assert every_row_call(lib_and_ctx[0], None) == [ARGUMENT] * 3


@pytest.mark.parametrize("limit", [0.0, -1.0, float("nan")])
def test_limits_refused(lib_and_ctx, limit):
    lib, ctx = lib_and_ctx
    r = rows()
    assert lib.wh_fp8_swiglu_rows_async(ctx, DEV, DEV, 256, 0, 3, 256, limit, ctypes.byref(r)) == ARGUMENT
    assert lib.wh_fp8_swiglu_rows_async(ctx, DEV, None, 256, 0, 3, 256, 10.0, ctypes.byref(r)) == ARGUMENT
    assert lib.wh_fp8_swiglu_rows_async(ctx, DEV, DEV + 2, 256, 0, 3, 256, 10.0, ctypes.byref(r)) == ARGUMENT


def test_products_refused(lib_and_ctx):
    lib, ctx = lib_and_ctx
    r = rows()
    p = ctypes.byref(r)
    assert lib.wh_fp8_rows_mm_async(None, 1, 0, 16, p, 1, DEV, 16, 0) == ARGUMENT
    assert lib.wh_fp8_rows_mm_async(ctx, 1, 0, 16, None, 1, DEV, 16, 0) == ARGUMENT
    assert lib.wh_fp8_rows_mm_async(ctx, 1, 16, 16, p, 1, DEV, 16, 0) == SHAPE

    def groups(gr=16, ng=2, rp=p, n_x=4, rows_ptr=None, starts=DEV, n=4):
        return lib.wh_fp8_rows_mm_groups_async(ctx, 1, 0, gr, ng, rp, n_x, rows_ptr, starts, n, DEV, 16, 0)

    assert groups(rp=None) == groups(starts=None) == groups(starts=DEV + 2) == groups(rows_ptr=DEV + 1) == ARGUMENT
    assert groups(gr=0) == groups(ng=0) == EMPTY
    assert groups(ng=1025) == groups(n=1 << 31) == UNSUPPORTED
    assert groups(n_x=3) == groups(rows_ptr=DEV, n_x=0) == SMALL


def test_plans_refused(lib_and_ctx):
    lib, ctx = lib_and_ctx

    def plan(ids=DEV, npos=4, topk=2, n=8, starts=DEV, rows_=DEV, slots=DEV, c=ctx):
        return lib.wh_expert_plan_async(c, ids, npos, topk, n, starts, rows_, slots)

    assert plan(c=None) == plan(ids=None) == plan(starts=None) == plan(rows_=None) == plan(slots=None) == ARGUMENT
    assert plan(ids=DEV + 1) == plan(starts=DEV + 2) == plan(rows_=DEV + 3) == plan(slots=DEV + 2) == ARGUMENT
    assert plan(topk=0) == plan(n=0) == EMPTY
    assert plan(n=1025) == plan(topk=65537) == plan(npos=1 << 30, topk=2) == plan(npos=1 << 62) == UNSUPPORTED


def test_combines_refused(lib_and_ctx):
    lib, ctx = lib_and_ctx

    def combine(y=DEV, ys=128, bf16=0, n=4, slots=DEV, w=DEV, npos=3, topk=2, hidden=128, add=None, adds=0, out=DEV, outs=128,
                c=ctx):
        return lib.wh_expert_combine_async(c, y, ys, bf16, n, slots, w, npos, topk, hidden, add, adds, out, outs)

    for kw in (dict(c=None), dict(y=None), dict(slots=None), dict(w=None), dict(out=None), dict(y=DEV + 8), dict(ys=130),
               dict(y=DEV + 4, bf16=1), dict(add=DEV + 4, adds=128), dict(add=DEV, adds=130), dict(out=DEV + 4),
               dict(outs=130), dict(slots=DEV + 2), dict(w=DEV + 1)):
        assert combine(**kw) == ARGUMENT, kw
    assert combine(hidden=0) == combine(topk=0) == EMPTY
    assert combine(hidden=126) == combine(ys=124) == combine(outs=124) == combine(add=DEV, adds=124) == SHAPE
    assert combine(npos=1 << 31) == combine(n=1 << 31) == combine(hidden=1 << 31) == UNSUPPORTED
    assert combine(npos=1 << 26, hidden=4096, ys=4096, outs=4096) == UNSUPPORTED
    assert combine(npos=0, y=None, out=None) == 0
