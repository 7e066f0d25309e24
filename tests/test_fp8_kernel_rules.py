"""What the e4m3 product's exchange over a cluster must keep, read from the sources: a barrier that some threads do not reach, or a store into a CTA that has not
started, would hang or corrupt a GPU and shows in no result."""
import os
import re

import pytest

import test_kernel_waits as W

KERNELS = {"fp8_gemm_kernel": os.path.join(W.CSRC, "fp8", "k_fp8_gemm.cuh"), "blockwise_smallm_kernel": os.path.join(W.CSRC, "k_blockwise_smallm.cuh")}


def _body(name):
    with open(KERNELS[name]) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    at = text.index("\n%s(const __grid_constant__" % name)
    return text[at:text.index("\n}\n", at)]


def _block(text, at):
    """The braces that open at or behind `at`, with what they hold."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError("braces")


# Where each kernel's two sides of the exchange are: the promotion warps', and everybody else's.
SIDES = {
    "fp8_gemm_kernel": (r"if constexpr \(SPLITK\) \{\s*const int share_cols", r"if constexpr \(SPLITK\) \{\s*__syncwarp\(\);\s*cluster_sync_all"),
    "blockwise_smallm_kernel": (r"if \(p\.splits > 1\) \{", r"if \(p\.splits > 1 && !\(\(warp & 3\) < 2\)\) \{"),
}


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_both_sides_of_the_exchange_meet_as_often(name):
    body = _body(name)
    counts = []
    for pattern in SIDES[name]:
        found = re.findall(pattern, body)
        assert len(found) == 1, pattern
        side = _block(body, re.search(pattern, body).start())
        counts.append(side.count("cluster_sync_all()"))
        # nothing leaves between the barriers, and none of them stands in a branch or a loop of its own
        outer = side[1:-1]
        while True:
            inner = re.search(r"\{[^{}]*\}", outer)
            if not inner:
                break
            assert "cluster_sync_all" not in inner.group(0) and "return" not in inner.group(0), inner.group(0)
            outer = outer[:inner.start()] + outer[inner.end():]
        assert not re.search(r"\b(return|break|continue)\b", re.sub(r"(for|if) \([^;{]*(;[^;{]*){0,2}\) (break|continue);", "", outer))
    assert counts == [2, 2]
    # all other barriers of the cluster are the pair form's, which every thread reaches
    pair = len(re.findall(r"if constexpr \(PAIR\) cluster_sync_all\(\);", body))
    assert body.count("cluster_sync_all()") == sum(counts) + pair


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_remote_stores_stand_between_the_two_barriers(name):
    body = _body(name)
    stores = [m.start() for m in re.finditer(r"st\.shared::cluster", body)]
    side = _block(body, re.search(SIDES[name][0], body).start())
    first, second = (m.start() for m in re.finditer(r"cluster_sync_all\(\)", side))
    at = [m.start() for m in re.finditer(r"st\.shared::cluster", side)]
    assert len(stores) == len(at) >= 1
    assert all(first < a < second for a in at)


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_no_thread_leaves_early(name):
    """Only lambdas return: a thread that left the kernel would be missed at its barriers."""
    body = _body(name)
    depth_free = body
    for m in re.finditer(r"\[[&=\w]*\](?:\((?:[^()]|\([^()]*\))*\))? \{", body):
        depth_free = depth_free.replace(_block(body, m.start()), "{}")
    assert not re.search(r"\breturn\b", depth_free)


def test_a_split_tile_ends_for_nobody_alone():
    """A failed wait ends the tiles of the other forms; a split one's promotion warps go on to the exchange."""
    body = _body("fp8_gemm_kernel")
    assert "if (!SPLITK && !ok) break;" in body
    tail = body[body.index("if (!SPLITK && !ok) break;"):]
    assert "if (!ok) break" not in tail.replace("if (!SPLITK && !ok) break;", "")
