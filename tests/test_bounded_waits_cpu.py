"""Kernel sources: what a bounded wait that gives up may lead to.

Every wait on an mbarrier ends, after two seconds at most.  That must not turn
into another wait that does not: warps that meet at a named barrier all have to
get there, so none of them may leave its loop when a wait gives up; and the
lanes of a warp that acts as one have to agree on it.
"""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blockfp8_b200", "csrc")
FILES = ["mx_gemm.cuh", "moe.cuh", "gemm_kernel.cuh", "stream_gemm.cuh"]


def _statements(path):
    """(line, text, [headers of the enclosing blocks], [their ids]) of every statement or header, comments taken out."""
    text = open(path).read()
    text = re.sub(r"//[^\n]*", "", text)
    stack, out, start, line, serial = [], [], 0, 1, 0
    at, depth = 1, 0
    for k, c in enumerate(text):
        depth += (c == "(") - (c == ")")
        if c == "\n":
            line += 1
        if c in "{}" or (c == ";" and depth == 0):
            piece = " ".join(text[start:k].split())
            if piece:
                out.append((at, piece, [h for h, _ in stack], [n for _, n in stack]))
            if c == "{":
                serial += 1
                stack.append((piece, serial))
            elif c == "}":
                stack.pop()
            start, at = k + 1, line
    return out


def _one_thread(headers):
    return any(re.search(r"\blane == 0\b|threadIdx\.x == 0|\btid == 0\b", h) for h in headers)


@pytest.mark.parametrize("name", FILES)
def test_a_wait_that_gives_up_strands_no_other_warp(name):
    statements = _statements(os.path.join(CSRC, name))
    # blocks (roles) whose warps meet at a named barrier
    meeting = set()
    for _, piece, headers, ids in statements:
        if "named_bar_sync(" in piece:
            meeting.update(n for h, n in zip(headers, ids) if re.match(r"(\} )?(else )?(if|else|for)\b", h))
    bad = []
    for line, piece, headers, ids in statements:
        leaves = re.search(r"\bmbar_wait(_warp)?\(.*\)\)*\s*(break|return|goto)\b", piece)
        if not leaves or _one_thread(headers + [piece]):
            continue
        if not leaves.group(1):
            bad.append((line, "lanes may disagree", piece))
        elif any(n in meeting for n in ids):
            bad.append((line, "other warps wait at a named barrier", piece))
    assert not bad


@pytest.mark.parametrize("name", FILES[:2])
def test_waits_of_a_whole_warp_are_found(name):
    """The test above sees the roles that it is about."""
    statements = _statements(os.path.join(CSRC, name))
    assert any("mbar_wait" in p and not _one_thread(h + [p]) for _, p, h, _ in statements)
    assert any("mbar_wait" in p and _one_thread(h + [p]) for _, p, h, _ in statements)


TMEM_ACCESS = re.compile(r"\b(tmem_st16|tmem_ld16|tmem_ld32|mma_mxf4(<\w+>)?|tmem_cp_scales_pair)\(")


def test_tensor_memory_is_touched_behind_a_fence():
    """An mbarrier orders nothing in tensor memory by itself: between a wait and the next tcgen05 access of the
    same thread stands tcgen05.fence::after_thread_sync."""
    seen, bad = 0, []
    waited = None
    for line, piece, _, _ in _statements(os.path.join(CSRC, "mx_gemm.cuh")):
        if "__global__" in piece:
            waited = None
        if "tc_fence_after()" in piece:
            waited = None
        if TMEM_ACCESS.search(piece):
            seen += 1
            if waited:
                bad.append((line, f"wait in line {waited}", piece))
        if re.search(r"\bmbar_wait(_warp)?\(", piece):
            waited = line
    assert seen >= 5 and not bad
