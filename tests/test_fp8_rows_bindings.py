"""CPU check of the comments at the Rust structs of device buffers."""
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("struct,says", [("WhFp8Rows", "8-bit rows"), ("WhKv4Attention", "Attention of new tokens"),
                                         ("WhKv4Cache", "4-bit"), ("WhKvPlan", "page")])
def test_rust_structs_have_their_own_comments(struct, says):
    text = (ROOT / "ffi" / "rust" / "src" / "sys.rs").read_text()
    found = re.search(r"((?:^///[^\n]*\n)+)(?:#\[[^\n]*\n)+pub struct " + struct + r"\b", text, flags=re.M)
    assert found and says.lower() in found.group(1).lower()
