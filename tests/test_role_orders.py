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


TOLD = r"wait_told(?:_here)?\(&H\.%s, %s & 1, &H\.%s, %s, &H\)"


def test_roles_wait_for_those_whose_words_they_read():
    """Where a chunk's values are not finite comes from the weights' warps, its decays from the copying one, which those have waited for: a
    product's end, told by the issuing thread, puts neither before a read of them.  The word is asked for behind the end: a role that sits out
    the first pass has not followed the ring, and a wait for odd parity returns at once while a barrier is in its first phase."""
    ready = between(code("linear_tc.cuh"), "struct WaitTold", "};")
    assert re.search(r"ended = pf_bar_try\(this->bar, this->parity\), told = pf_bar_try\(word, word_parity\);\s+return ended && told;", ready)
    text = code("linear_chunks.cu")
    for start, end, product, turn, word in (("for (int k = 0;; k++)", "arrive_warp(&H.u_free)", "u_full", "k", "w_full"),
                                            ("for (int j = 0; j < own; j++, out +=", "write_out(", "n_full", "j", "w_full"),
                                            ("const int r = tid - 384", "weights_row(", "qk_full", "j", "known")):
        role = between(text, start, end)
        wait = re.search(TOLD.replace("%s, %s, &H", r"%s\[k %% kRing\], \(k / kRing\) & 1, &H") % (product, turn, word), role)
        assert wait and (wait.end() < role.index("dec = H.ring") if "dec = H.ring" in role else role.count("wait_") == 1)
    weights = between(text, "for (int k = 0; k < twice + own; k++)", "arrive_warp(&H.w_full")
    assert weights.index("wait_warp(&H.known[k % kRing]") < weights.index("dec = H.ring")


def test_no_place_of_the_ring_is_told_twice_while_a_role_looks():
    """The parity of a phase says which of two it is.  The roles of a block as the waits between them order them, in many orders: behind the
    product that a role waits for, the last phase that ended in chunk k's place is chunk k's."""
    import random
    ring, stages = 8, 3
    for seed in range(60):
        rng = random.Random(seed)
        twice, own = rng.randint(0, 40), rng.randint(1, 40)
        n = twice + own
        second = ("qk", "p", "n", "out")                     # roles of the second pass alone
        done = {name: 0 for name in ("copy", "w", "u", "state") + second}        # chunks that a role has ended
        speed = {name: rng.random() ** 3 + 1e-3 for name in done}
        may = dict(
            copy=lambda k: k < stages or (done["u"] > k - stages and (k - stages < twice or done["n"] > k - stages - twice)),
            w=lambda k: done["copy"] > k and (k < 2 or done["u"] > k - 2),
            # products in the issuing thread's order: U of a chunk behind N of the one before
            u=lambda k: done["w"] > k and done["state"] >= k and (k <= twice or done["n"] >= k - twice),
            state=lambda k: done["u"] > k,
            qk=lambda j: done["copy"] > twice + j and done["p"] >= j and (j == 0 or done["u"] >= twice + j),
            p=lambda j: done["qk"] > j,
            n=lambda j: done["u"] > twice + j and done["p"] > j and done["state"] >= twice + j and (j == 0 or done["out"] >= j),
            out=lambda j: done["n"] > j)
        total = {name: own if name in second else n for name in done}
        while any(done[r] < total[r] for r in done):
            for r, tellers in (("state", ("copy", "w")), ("out", ("copy", "w")), ("p", ("copy",))):
                if done[r] == total[r]:
                    continue
                j, k = done[r], done[r] + (twice if r in second else 0)
                if not may[r](j):                            # the product that the role waits for has not ended
                    continue
                for teller in tellers:
                    phases = len([c for c in range(done[teller]) if c % ring == k % ring])
                    assert phases - k // ring == 1, (r, k, teller, done)
            ready = [r for r in done if done[r] < total[r] and may[r](done[r])]
            assert ready, (twice, own, done)
            r = rng.choices(ready, [speed[x] for x in ready])[0]
            done[r] += 1


def test_the_chain_waits_for_the_warp_that_has_the_other_half_of_its_rows():
    """With the delta rule two warps take places of a row out of rhs and u, by halves of the chunk's tokens; each then reads whether the row
    has any.  (The next w_full wants these warps' own arrivals, so that the phase seen is this chunk's.)"""
    chain = between(code("linear_delta.cu"), "for (int k = 0; k < chunks && ok; k++)", "store_state(")
    wait = re.search(TOLD % ("u_full", "k", "w_full", "k & 1"), chain)
    assert wait and chain.index("arrive_warp(&H.w_full)") < wait.start() < chain.index("dec.bad[row]")


def test_the_state_leaves_behind_the_outputs_word():
    """The state's warps have not followed the last product's barrier: behind the outputs' last word the phase that ended last is the last one."""
    way_out = between(code("linear_chunks.cu"), "if (ok && rank + 1 == blocks && seq.to", "store_state(")
    assert 0 < way_out.index("wait_here(&H.out_done, 0") < way_out.index("wait_here(&H.n_full, (own - 1) & 1")
