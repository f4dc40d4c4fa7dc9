"""CPU checks of the paged 4-bit cache: the address arithmetic that its
kernels run on (garbage lengths, starts, pages and slots included) and every
refusal of its entry points.  A refused call returns before it touches the
context, so a block of zeros stands in for one."""
import ctypes
import subprocess
from pathlib import Path

import pytest

import wohper_amd as wa

ROOT = Path(__file__).resolve().parents[1]
EMPTY, SHAPE, ARGUMENT, UNSUPPORTED = 1, 2, 13, 15
DEV = 0x10000  # an aligned address that a refused call never reads


def test_index_arithmetic(tmp_path):
    exe = tmp_path / "kv4_index"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", str(ROOT / "wohper_amd" / "csrc"), str(ROOT / "tests" / "kv4_index.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe), "4000"], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr


@pytest.fixture
def lib_and_ctx():
    return wa.load_library(), ctypes.cast(ctypes.create_string_buffer(1 << 16), ctypes.c_void_p)


def cache(**kw):
    d = dict(k_codes=DEV, k_scales=DEV, v_codes=None, v_scales=None, n_pages=4, page_size=16, kv_heads=2, head_dim=128)
    d.update(kw)
    return wa.WhKv4Cache(**d)


CACHES = [
    (dict(k_codes=None), ARGUMENT), (dict(k_scales=None), ARGUMENT), (dict(v_codes=DEV), ARGUMENT),
    (dict(v_scales=DEV), ARGUMENT), (dict(k_codes=DEV + 8), ARGUMENT), (dict(k_scales=DEV + 4), ARGUMENT),
    (dict(v_codes=DEV + 4, v_scales=DEV), ARGUMENT), (dict(v_codes=DEV, v_scales=DEV + 2), ARGUMENT),
    (dict(n_pages=0), EMPTY), (dict(page_size=0), EMPTY), (dict(kv_heads=0), EMPTY), (dict(head_dim=0), EMPTY),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=32), UNSUPPORTED), (dict(head_dim=1024), UNSUPPORTED),
    (dict(page_size=12), UNSUPPORTED), (dict(page_size=1 << 17), UNSUPPORTED), (dict(kv_heads=70000), UNSUPPORTED),
    (dict(n_pages=1 << 28), UNSUPPORTED), (dict(n_pages=1 << 61), UNSUPPORTED),
]


@pytest.mark.parametrize("change,status", CACHES)
def test_caches_refused(lib_and_ctx, change, status):
    lib, ctx = lib_and_ctx
    c = ctypes.byref(cache(**change))
    vp = DEV if change.get("v_codes") and change.get("v_scales") else None
    assert lib.wh_kv4_write_async(ctx, c, DEV, 256, vp, 256, 0, DEV, 1) == status
    assert lib.wh_kv4_read_async(ctx, c, DEV, 1, DEV, 256, None, 0, 0) == status
    a = attention()
    assert lib.wh_kv4_attention_async(ctx, c, ctypes.byref(a)) == status


ROWS = [
    (dict(cache=None), ARGUMENT), (dict(k=None), ARGUMENT), (dict(slots=None), ARGUMENT), (dict(v=DEV), ARGUMENT),
    (dict(k=DEV + 4), ARGUMENT), (dict(ks=258), ARGUMENT), (dict(ks=260, bf16=1), ARGUMENT), (dict(ks=252), SHAPE),
    (dict(n=1 << 31), UNSUPPORTED),
    (dict(own=True), ARGUMENT),  # values of their own, none given
    (dict(own=True, v=DEV + 8), ARGUMENT), (dict(own=True, v=DEV, vs=250), ARGUMENT),
    (dict(own=True, v=DEV, vs=128), SHAPE),
]


@pytest.mark.parametrize("change,status", ROWS)
def test_rows_refused(lib_and_ctx, change, status):
    lib, ctx = lib_and_ctx
    d = dict(cache=cache(), k=DEV, ks=256, v=None, vs=256, bf16=0, slots=DEV, n=3)
    if change.get("own"):
        d["cache"] = cache(v_codes=DEV, v_scales=DEV)
    d.update({k: v for k, v in change.items() if k != "own"})
    c = ctypes.byref(d["cache"]) if d["cache"] is not None else None
    assert lib.wh_kv4_write_async(ctx, c, d["k"], d["ks"], d["v"], d["vs"], d["bf16"], d["slots"], d["n"]) == status
    if change != dict(own=True):  # keys may be read alone
        got = lib.wh_kv4_read_async(ctx, c, d["slots"], d["n"], d["k"], d["ks"], d["v"], d["vs"], d["bf16"])
        assert got == status
    assert lib.wh_kv4_write_async(None, c, d["k"], d["ks"], d["v"], d["vs"], d["bf16"], d["slots"], d["n"]) == ARGUMENT


def test_no_rows_are_no_call(lib_and_ctx):
    lib, ctx = lib_and_ctx
    c = ctypes.byref(cache())
    assert lib.wh_kv4_write_async(ctx, c, DEV, 256, None, 0, 0, None, 0) == 0
    assert lib.wh_kv4_read_async(ctx, c, None, 0, DEV, 256, None, 0, 0) == 0
    assert lib.wh_kv4_attention_async(ctx, c, ctypes.byref(attention(n_tokens=0))) == 0
    assert lib.wh_kv4_attention_async(ctx, c, ctypes.byref(attention(n_requests=0))) == 0


def attention(**kw):
    d = dict(q_dev=DEV, q_stride=512, out_dev=2 * DEV, out_stride=512, is_bf16=0, n_tokens=2, n_requests=1,
             starts_dev=DEV, lens_dev=DEV, tables_dev=DEV, table_stride=4, max_len=64, heads=4, scale=0.1, window=0,
             first=0, sink=None)
    d.update(kw)
    return wa.WhKv4Attention(**d)


ATTENTION = [
    (dict(q_dev=None), ARGUMENT), (dict(out_dev=None), ARGUMENT), (dict(starts_dev=None), ARGUMENT),
    (dict(lens_dev=None), ARGUMENT), (dict(tables_dev=None), ARGUMENT), (dict(q_dev=DEV + 4), ARGUMENT),
    (dict(out_dev=DEV + 8), ARGUMENT), (dict(q_stride=514), ARGUMENT), (dict(out_stride=516, is_bf16=1), ARGUMENT),
    (dict(q_stride=508), SHAPE), (dict(out_stride=256), SHAPE), (dict(heads=0), EMPTY), (dict(heads=5), SHAPE),
    (dict(n_tokens=1 << 30), UNSUPPORTED), (dict(n_requests=1 << 30), UNSUPPORTED),
    (dict(heads=1 << 20, q_stride=1 << 27, out_stride=1 << 27), UNSUPPORTED), (dict(table_stride=1 << 32), UNSUPPORTED),
]


@pytest.mark.parametrize("change,status", ATTENTION)
def test_attention_refused(lib_and_ctx, change, status):
    lib, ctx = lib_and_ctx
    assert lib.wh_kv4_attention_async(ctx, ctypes.byref(cache()), ctypes.byref(attention(**change))) == status


def test_attention_without_descriptors(lib_and_ctx):
    lib, ctx = lib_and_ctx
    assert lib.wh_kv4_attention_async(None, ctypes.byref(cache()), ctypes.byref(attention())) == ARGUMENT
    assert lib.wh_kv4_attention_async(ctx, None, ctypes.byref(attention())) == ARGUMENT
    assert lib.wh_kv4_attention_async(ctx, ctypes.byref(cache()), None) == ARGUMENT


PLANS = [
    (dict(starts_dev=None), ARGUMENT), (dict(free_dev=None), ARGUMENT), (dict(free_count_dev=None), ARGUMENT),
    (dict(free_out_dev=None), ARGUMENT), (dict(free_count_out_dev=None), ARGUMENT), (dict(old_lens_dev=None), ARGUMENT),
    (dict(new_lens_dev=None), ARGUMENT), (dict(tables_dev=None), ARGUMENT), (dict(slots_dev=None), ARGUMENT),
    (dict(positions_dev=None), ARGUMENT), (dict(page_size=0), EMPTY), (dict(n_pages=0), EMPTY),
    (dict(page_size=24), UNSUPPORTED), (dict(page_size=1 << 17), UNSUPPORTED), (dict(n_requests=4097), UNSUPPORTED),
    (dict(max_tokens=1 << 31), UNSUPPORTED), (dict(n_pages=1 << 28), UNSUPPORTED),
]


@pytest.mark.parametrize("change,status", PLANS)
def test_plans_refused(lib_and_ctx, change, status):
    lib, ctx = lib_and_ctx
    d = dict(n_requests=3, old_lens_dev=DEV, new_lens_dev=DEV, tables_dev=DEV, table_stride=4, page_size=16, n_pages=8,
             free_dev=DEV, free_count_dev=DEV, free_out_dev=DEV, free_count_out_dev=DEV, max_tokens=9, starts_dev=DEV,
             slots_dev=DEV, positions_dev=DEV)
    d.update(change)
    assert lib.wh_kv_plan_async(ctx, ctypes.byref(wa.WhKvPlan(**d))) == status
    assert lib.wh_kv_plan_async(None, ctypes.byref(wa.WhKvPlan(**d))) == ARGUMENT
    assert lib.wh_kv_plan_async(ctx, None) == ARGUMENT
