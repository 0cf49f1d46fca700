"""Bounded waits by whole warps: their result has to be the same in every lane.

A lane may find its time up while another sees the copy land.  Lanes that then go different ways meet full-mask shuffles
and barriers with lanes missing, which may hang, so a wait's result goes through a vote before anything depends on it.
No wait is made to run out in the kernels themselves, so this reads the source."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "sonata_b200" / "csrc"


def _code(name):
    text = (CSRC / name).read_text()
    return re.sub(r"//[^\n]*", "", text)


def _waits(code):
    """The text before each bounded wait, from the start of its statement."""
    for m in re.finditer(r"\bmbar_wait_bounded\(", code):
        start = max(code.rfind(c, 0, m.start()) for c in ";{}")
        yield code[start + 1:m.start()]


def test_paged_attention_waits_by_vote():
    code = _code("paged_kv.cu")
    waits = list(_waits(code))
    assert waits, "paged_kv.cu has no bounded wait: this test looks at nothing"
    for before in waits:
        assert "__all_sync(0xffffffffu, " in before, before


def test_paged_attention_waits_again_before_the_ring_is_reused():
    """A tile whose wait ran out is waited for once more, and is not counted as there."""
    code = _code("paged_kv.cu")
    m = re.search(r"there = wait_tile\((?P<args>.*?)\);\s*if \(!there\) \{(?P<body>.*?)\n        \}", code, re.S)
    assert m, "the tile's wait has another form"
    assert "record_status(SN_ERR_TIMEOUT)" in m["body"] and "dead = true" in m["body"]
    assert f"wait_tile({m['args']})" in m["body"]


@pytest.mark.parametrize("name", ["paged_kv.cu", "mamba_prompt.cu"])
def test_whole_warp_waits_do_not_branch_on_a_lane(name):
    """`if (!mbar_wait_bounded(...))` is for code of one thread only: it is inside a lambda or block that lane 0 alone enters."""
    code = _code(name)
    for m in re.finditer(r"if \([^;{]*!mbar_wait_bounded\(", code):
        scope = code[max(0, m.start() - 400):m.start()]
        assert "lane == 0" in scope, code[m.start():m.start() + 80]
