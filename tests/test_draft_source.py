"""Properties of the tree attention kernels' source that no call can show without making a kernel give up."""
import re

import pytest

from lumenllm_b200.csrc.build import CSRC


def conditions_around(text, at):
    """The conditions of all `if (...)` whose braces or single statement hold the text at `at`."""
    found, stack, i = [], [], 0
    while i < at:
        if text.startswith("//", i):
            i = text.index("\n", i)
        elif text[i] == "{":
            stack.append(text[max(text.rfind(c, 0, i) for c in ";{}") + 1:i])
            i += 1
        elif text[i] == "}":
            stack.pop()
            i += 1
        else:
            i += 1
    for head in stack + [text[max(text.rfind(c, 0, at) for c in ";{}") + 1:at]]:
        found += re.findall(r"\bif\s*\((.*)", head, re.S)
    return found


def test_conditions_around():
    text = "a; if (x) { b; for (;;) { if (y) c(); } d(); }"
    assert [c.split(")")[0] for c in conditions_around(text, text.index("c()"))] == ["x", "y"]
    assert [c.split(")")[0] for c in conditions_around(text, text.index("d()"))] == ["x"]


@pytest.mark.parametrize("wait", ["mbar_wait(&k_full[", "mbar_wait(&v_full[", "mbar_wait(&s_full[(cs - 1)", "mbar_wait(&pv_done[(cv - 1)",
                                  'asm volatile("cp.async.wait_all;" ::: "memory");\n        if'])
def test_a_block_waits_for_its_copies_and_products_whichever_role_gives_up(wait):
    """The role that asked for a copy or a product may have left in good order when another gives up waiting for it: its
    waits at the end hang on no `ok` of its own."""
    text = (CSRC / "attn_tree_tc.cuh").read_text()
    text = text[text.index("attn_tree_tc_kernel(const TreeTc t) {"):text.index("tcgen05.dealloc")]
    places = [m.start() for m in re.finditer(re.escape(wait), text)]
    assert len(places) == 1
    for cond in conditions_around(text, places[0]):
        assert not re.search(r"\bok\b", cond.split("{")[0]), cond


def test_a_block_that_leaves_at_once_leaves_nothing_to_join():
    """The joining kernel takes its places from every block's record: no way out of the first kernel leaves one unwritten."""
    text = (CSRC / "attn_tree_tc.cuh").read_text()
    text = text[text.index("attn_tree_tc_kernel(const TreeTc t) {"):]
    before = text[:text.index("TreeJoin join = {")]
    for way_out in [m.start() for m in re.finditer(r"\breturn;", before)]:
        assert "t.joins[blockIdx.x] =" in before[before.rfind("if (smem_u32", 0, way_out):way_out]


def test_a_warp_whose_first_lane_waits_is_ordered_behind_it():
    """What one lane has waited for is read by all: a shuffle hands them the answer but orders no memory, a warp barrier does."""
    text = (CSRC / "attn_tree_tc.cuh").read_text()
    body = text[text.index("bool tt_warp_wait("):]
    body = body[:body.index("\n}")]
    assert body.index("mbar_wait(") < body.index("__syncwarp()") < body.rindex("return")
