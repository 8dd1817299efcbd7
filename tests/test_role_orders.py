"""What the prompts' kernels of linear attention wait for before one thread reads what another wrote: read in their source, since an
order that is missing shows on a GPU once in a great while or never."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "biv_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def between(text, start, end):
    at = text.index(start)
    return text[at:text.index(end, at)]


def test_values_that_a_lane_takes_out_are_seen_by_the_lanes_that_load_them():
    """A vote and a fence between proxies order nothing among a warp's threads."""
    w = between(code("linear_chunks.cu"), "for (int again = 0;", "arrive_warp(&H.w_full")
    assert "ldmatrix" in w
    assert "__syncwarp()" in w[w.index("st.shared.u16"):w.index("wait_st()")]
