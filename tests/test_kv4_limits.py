"""CPU checks of how large a call of the paged 4-bit cache may be: a grid
dimension times its workgroup's threads stays below 2^32."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def build_and_run(tmp_path, source):
    (tmp_path / "t.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    str(ROOT / "wohper_amd" / "csrc"), str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    return subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)


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
