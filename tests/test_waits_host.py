"""Bounded waits on the device, read from the sources: a warp that gives one up leaves as a whole.  Lanes count their polls each for itself; a lane
that left alone would be missing from the shuffles and barriers of the others, and a wait that ran out for lanes other than 0 only would
not be reported (lane 0 writes the error word)."""
import os
import re

import pytest

from tests.util import ROOT

CSRC = os.path.join(ROOT, "shadow-engine_b200", "csrc")
#: files whose kernels leave a loop or return where a wait of a whole warp ran out
FILES = ["sz_session_rows.cuh"]


def leaving_waits(text):
    """Statements `if (.. wait ..) {.. return / break ..}` -> the waits they call."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"if \(([^;{}]*\bsz_mbar_wait\w*\([^;{}]*)\) *(\{[^{}]*\}|[^;{}]*;)", text):
        if re.search(r"\b(return|break)\b", m.group(2)):
            yield from re.findall(r"\bsz_mbar_wait\w*", m.group(1))


@pytest.mark.parametrize("name", FILES)
def test_a_warp_leaves_a_wait_as_a_whole(name):
    waits = list(leaving_waits(open(os.path.join(CSRC, name)).read()))
    assert waits and set(waits) == {"sz_mbar_wait_warp"}


def test_the_warps_wait_is_a_vote():
    text = open(os.path.join(CSRC, "sz_common.cuh")).read()
    assert re.search(r"bool sz_mbar_wait_warp\([^)]*\) \{ return __all_sync\(0xffffffffu, sz_mbar_wait\(bar, phase\)\); \}", text)


def body(text, begin, end):
    at = text.index(begin)
    return text[at:text.index(end, at)]


def test_the_tcgen05_attention_ends_with_nothing_under_way():
    """Whichever role gives up a wait, the others' copies and products are seen to their end, within a limit, before the block frees its tensor memory and leaves."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "sz_paged_tc.cu")).read())
    roles = body(text, "if (warp == TMA_WARP", "sz_pdl_trigger();")
    tma, s, pv = body(roles, "if (warp == TMA_WARP", "warp == S_WARP"), body(roles, "warp == S_WARP", "warp == PV_WARP"), body(roles, "warp == PV_WARP", "pt_stored();\n    }")
    after = tma[tma.rindex("u += T;"):]
    assert re.search(r"for \(u32 n = fills > C::SLOTS \? fills - C::SLOTS : 0; n < fills; n\+\+\) if \(!pt_wait_warp\(&S\.full\[kind\]\[n % C::SLOTS\], n / C::SLOTS\)\)", after)
    for i, role in enumerate((s, pv)):
        after = role[role.index("done += T;"):]
        assert re.search(r"pt_commit\(&S\.last\[%d\], one\);\s*if \(!pt_wait_warp\(&S\.last\[%d\], 0\)\) failed" % (i, i), after)
    assert roles.rstrip().endswith("pt_stored();\n    }")
    assert text.index("__syncthreads();", text.index("sz_pdl_trigger();")) < text.index("tcgen05.dealloc")


def test_the_paged_attention_waits_for_its_copies_after_one_was_given_up():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "sz_paged.cuh")).read())
    given_up = body(text, "if (!dead && !sz_mbar_wait_warp(", "if (NQT > 1) __syncthreads();")
    assert "steps_left = -1 - steps_left;" in given_up       # .. asked for: below 0 from here on
    end = body(text, "if (dead) {", "sz_pdl_trigger();")
    assert "n = (int)(2 * (u1 - u0)) + 1 + steps_left;" in end and re.search(r"for \(int i = max\(0, n - C::NR\); i < n; i\+\+\) sz_mbar_wait_warp\(", end)
    assert re.search(r"auto issue = \[&\]\(int which\) \{\s*if \(steps_left <= 0\) return;", text)
