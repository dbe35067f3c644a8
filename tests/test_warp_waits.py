"""Waits that run out: what follows a wait of a whole warp (matrix loads and products, shuffles, votes) needs all its lanes, so the lanes agree on
how the wait ended.  A wait gives up by each lane's own clock, and a run-out cannot be brought about by a call: the source is read instead."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "flashck_b200", "csrc")


def _unvoted(text):
    """Lines with a bounded wait that neither a vote nor a single lane (whose result is then handed round) takes."""
    code = re.sub(r"//[^\n]*", lambda m: " " * len(m.group()), text)
    bad = []
    for m in re.finditer(r"mbar_wait_bounded\(", code):
        before = code[:m.start()]
        depth, alone = 0, False
        for c in before[before.rfind("if (lane == 0) {") + 15:] if "if (lane == 0) {" in before else "":
            depth += (c == "{") - (c == "}")
            alone = depth > 0
            if not alone:
                break
        if not alone and not before.endswith("__all_sync(0xffffffffu, "):
            bad.append(before.count("\n") + 1)
    return bad


@pytest.mark.parametrize("name", ["splitkv_int4.cu", "splitkv_decode.cu"])
def test_warps_leave_a_wait_together(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    assert "mbar_wait_bounded(" in text and _unvoted(text) == []


def test_what_counts_as_together():
    assert _unvoted("ok = __all_sync(0xffffffffu, mbar_wait_bounded(a));") == []
    assert _unvoted("if (lane == 0) {\n  ok = mbar_wait_bounded(a);\n}\nok = __shfl_sync(0xffffffffu, ok, 0);") == []
    assert _unvoted("x;\nif (!mbar_wait_bounded(a)) return;") == [2]
    assert _unvoted("if (lane == 0) {\n}\nfor (;;) { if (failed || !mbar_wait_bounded(a)) failed = true; }") == [3]
