"""Named barriers of the device code: every thread that one counts has to reach it, also after a bounded wait has run out."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "simple_vsa_b200", "csrc")
SOURCES = sorted(f for f in glob.glob(os.path.join(CSRC, "*")) if "named_barrier(" in open(f).read())


def _under_a_wait(text):
    """Lines with a named barrier inside a block, or behind a condition, that depends on ``ok``: the result of a warp's own wait, which
    another warp of the same barrier may see differently."""
    text = re.sub(r"//[^\n]*", "", text)
    blocks, last, found = [], 0, []
    for m in re.finditer(r"[{};]|named_barrier\(", text):
        head = text[last:m.start()]
        if m.group() == "{":
            blocks.append(head)
        elif m.group() == "}":
            blocks.pop()
        elif m.group() == "named_barrier(":
            if any(re.search(r"\b(if|for|while)\s*\(.*\bok\b", h, re.S) for h in blocks + [head]):
                found.append(text[:m.start()].count("\n") + 1)
        last = m.end()
    return found


def test_the_search_finds_a_barrier_that_some_warps_may_miss():
    assert _under_a_wait("{\nif (ok) {\n x;\n named_barrier(1, 256);\n}\n}") == [4]
    assert _under_a_wait("{ if (ok && part) named_barrier(1, 256); }") == [1]
    assert _under_a_wait("{ if (ok) { x; }\n named_barrier(1, 256); // if (ok)\n }") == []


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_no_named_barrier_depends_on_a_warps_own_wait(path):
    assert _under_a_wait(open(path).read()) == []


def test_memory_in_flight_settles_before_a_cross_attention_cta_ends():
    """Every CTA gives its tensor memory back behind ``settle``, which waits for what is in flight after a wait that ran out."""
    text = open(os.path.join(CSRC, "cross_umma.cu")).read()
    ends = re.findall(r"([^;]*);\s*if \(warp == \d\) tmem_dealloc", text)
    assert len(ends) == len(re.findall(r"tmem_alloc\(", text)) == 3 and all(e.strip() == "settle(ok)" for e in ends)
