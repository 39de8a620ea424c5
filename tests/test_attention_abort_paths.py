"""What the attention kernels leave behind when a bounded wait has run out, as far as their source shows it: copies in flight get time to land, and what the
next kernel follows (where the pieces of cut units lie) is written on every path."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "warpforge_b200", "csrc")


def body(name, start):
    code = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    at = code.index("{", re.search(start, code).end())
    depth, end = 1, at + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(code[end], 0)
        end += 1
    return code[at + 1:end - 1]


def test_kernels_with_copies_in_flight_drain():
    for name, kernel in (("wf_attention_tree.cuh", r"void __launch_bounds__\([^)]*\) tree_tiles_kernel\([^{]*"), ("wf_attention_prompt.cuh", r"prompt_tiles_kernel\([^{]*")):
        assert "drain_after_abort()" in body(name, kernel)


def test_every_cta_says_whether_a_cut_unit_begins_in_it():
    """tree_join_kernel follows cuts[..] of every CTA: no path may leave the entry of an earlier launch, or of none."""
    for name, walker in (("wf_attention_tree.cuh", r"bool tree_load\([^{]*"), ("wf_attention_prompt.cuh", r"bool tree_items\([^{]*")):
        code = body(name, walker)
        walk = code.index("walk_line<")
        depth, end = 0, code.index("(", code.index(">(", walk))
        while True:
            depth += {"(": 1, ")": -1}.get(code[end], 0)
            end += 1
            if depth == 0:
                break
        assert "return" not in code[:walk]
        behind = code[end:]
        assert 0 <= behind.find("first_cta = -1") < behind.index("return"), name
