"""Bounded waits of the product kernels, without a GPU: what their source says
of them."""
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parent.parent / "sym_b200" / "csrc" / "cuda" / "mx_product.cu"


def test_every_wait_is_decided_by_the_whole_warp():
    """Behind these waits stand instructions that need all lanes of a warp, so
    no lane may run out of time alone: waits are those of ``warp_wait``, which
    votes."""
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    calls = re.findall(r"\b(mbar_\w+|warp_wait)\s*\(", text)
    assert calls.count("warp_wait") > 8
    assert "__all_sync(~0u, mbar_wait_often(" in text
    assert {c for c in calls if "wait" in c or "try" in c} == {"warp_wait", "mbar_wait_often"}
    assert calls.count("mbar_wait_often") == 1
