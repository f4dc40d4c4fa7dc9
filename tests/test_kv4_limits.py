"""CPU checks of how large a call of the paged 4-bit cache may be (a grid
dimension times its workgroup's threads stays below 2^32), and of its scale."""
import ctypes
import subprocess
from pathlib import Path

import pytest

import wohper_amd as wa
from test_kv4_host import ARGUMENT, UNSUPPORTED, attention, cache, lib_and_ctx  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]


def build_and_run(tmp_path, source):
    (tmp_path / "t.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    str(ROOT / "wohper_amd" / "csrc"), str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    return subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("n_tokens,n_requests,kv_heads,group,head_dim", [
    (1 << 20, 1 << 29, 64, 3, 64),     # 2^35 workgroups, of which 32 bits keep 2^26
    (1 << 24, 1, 64, 64, 128), (1 << 22, 1 << 26, 1, 1, 512), (1 << 26, 1, 1, 16, 64), (1 << 14, 1, 65535, 1, 64)])
def test_too_many_workgroups_are_refused(lib_and_ctx, n_tokens, n_requests, kv_heads, group, head_dim, bf16):  # noqa: F811
    lib, ctx = lib_and_ctx
    width = kv_heads * group * head_dim
    c = cache(kv_heads=kv_heads, head_dim=head_dim)
    a = attention(n_tokens=n_tokens, n_requests=n_requests, heads=kv_heads * group, q_stride=width, out_stride=width,
                  is_bf16=bf16, max_len=1 << 20)
    assert lib.wh_kv4_attention_async(ctx, ctypes.byref(c), ctypes.byref(a)) == UNSUPPORTED


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3.4e38])
def test_scales_that_are_not_finite_are_refused(lib_and_ctx, scale, bf16):  # noqa: F811
    lib, ctx = lib_and_ctx
    a = attention(scale=scale, is_bf16=bf16)
    assert lib.wh_kv4_attention_async(ctx, ctypes.byref(cache()), ctypes.byref(a)) == ARGUMENT


SOURCE = r"""
#include <cstdio>
#include <initializer_list>
#include "kv4_index.h"
int main() {
    for (uint64_t heads : {1u, 3u, 64u, 4097u, 65535u})
        for (uint64_t d : {64u, 128u, 256u, 512u})
            for (uint64_t n : {1ull, 2ull, 511ull, 1000003ull, 33554431ull, 33554432ull, 536870911ull, 536870912ull, 2147483647ull}) {
                const uint64_t pieces = heads * (d / 8);
                uint64_t at = 0, launches = 0;
                while (at < n) {
                    const uint64_t k = wh_kv4_rows_of_launch(n - at, pieces);
                    const uint64_t groups = (k * pieces + 255) / 256;
                    if (k == 0 || k > n - at || groups * 256 >= (1ull << 32)) {
                        std::printf("%llu heads of %llu, %llu rows: %llu\n", (unsigned long long)heads, (unsigned long long)d,
                                    (unsigned long long)n, (unsigned long long)k);
                        return 1;
                    }
                    at += k;
                    if (++launches > 3 && n * pieces < (1ull << 32)) return 2;
                }
                if (at != n) return 3;
            }
    return 0;
}
"""


def test_rows_are_cut_into_launches(tmp_path):
    res = build_and_run(tmp_path, SOURCE)
    assert res.returncode == 0, res.stdout


SHARE = r"""
#include <initializer_list>
#include "kv4_index.h"
int main() {
    // a cache of pages of one row may have 2^32 - 2 of them; a 32-bit counter that
    // steps past the last one would start over
    for (uint64_t n : {0ull, 1ull, 1025ull, 0xfffffffeull, 0xffffffffull})
        for (uint64_t step : {1ull << 18, 0x7fffff00ull}) {
            uint64_t calls = 0, last = 0;
            for (uint64_t first : {(uint64_t)0, (uint64_t)5, step - 1})
                wh_kv_share(first, step, n, [&](uint32_t i) { ++calls, last = i > last ? i : last; });
            uint64_t want = 0;
            for (uint64_t first : {(uint64_t)0, (uint64_t)5, step - 1}) want += first < n ? (n - first + step - 1) / step : 0;
            if (calls != want || (n && last >= n)) return 1;
        }
    return 0;
}
"""


def test_a_workgroups_share_comes_to_an_end(tmp_path):
    assert build_and_run(tmp_path, SHARE).returncode == 0
