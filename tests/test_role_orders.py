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


def test_roles_wait_for_those_whose_words_they_read():
    """A chunk's decays come from the copying warp (`known`), where its values are not finite from the weights' warps (`w_full`): a product's
    end, told by the issuing thread, puts neither before a read of them."""
    text = code("linear_chunks.cu")
    told = between(text, "auto told", "};")
    assert "wait_here(&H.known[k % kRing], parity" in told and "wait_here(&H.w_full[k % kRing], parity" in told
    for start, end, product in (("for (int k = 0;; k++)", "arrive_warp(&H.u_free)", "u_full"),
                                ("for (int j = 0; j < own; j++, out +=", "write_out(", "n_full")):
        role = between(text, start, end)
        wait = re.search(r"if \(!wait_\w+\(&H\.%s, \w & 1, &H\) \|\| !told\(k\)\)" % product, role)
        assert wait and wait.end() < role.index("dec = H.ring")


def test_no_place_of_the_ring_is_told_twice_while_a_role_looks():
    """The parity of a phase says which of two it is: a role that looks at chunk k's must not be eight chunks behind.  The roles of a
    block as the waits between them order them, in many orders: whoever looks finds chunk k's phase the last one that ended."""
    import random
    ring, stages = 8, 3
    for seed in range(60):
        rng = random.Random(seed)
        twice, own = rng.randint(0, 40), rng.randint(1, 40)
        n = twice + own
        done = {name: 0 for name in ("copy", "w", "u", "state", "n", "out")}     # chunks (n, out: of the second pass) that a role has ended
        speed = {name: rng.random() ** 3 + 1e-3 for name in done}
        may = dict(
            copy=lambda k: k < stages or (done["u"] > k - stages and (k - stages < twice or done["n"] > k - stages - twice)),
            w=lambda k: done["copy"] > k and (k < 2 or done["u"] > k - 2),
            # products in the issuing thread's order: U of a chunk behind N of the one before
            u=lambda k: done["w"] > k and done["state"] >= k and (k <= twice or done["n"] >= k - twice),
            state=lambda k: done["u"] > k,
            n=lambda j: done["u"] > twice + j and done["state"] >= twice + j and (j == 0 or done["out"] >= j),
            out=lambda j: done["n"] > j)
        total = {name: own if name in ("n", "out") else n for name in done}
        while any(done[r] < total[r] for r in done):
            ready = [r for r in done if done[r] < total[r] and may[r](done[r])]
            assert ready, (twice, own, done)
            r = rng.choices(ready, [speed[x] for x in ready])[0]
            if r in ("state", "out"):
                k = done[r] + (twice if r == "out" else 0)
                for teller in ("copy", "w"):
                    told = [c for c in range(done[teller]) if c % ring == k % ring]
                    assert told and told[-1] == k, (r, k, done)
            done[r] += 1


def test_warps_that_sit_out_the_first_pass_look_at_its_ring_behind_a_product():
    """A wait for odd parity returns at once while a barrier is in its first phase: with eight to fifteen chunks gone through twice a wait
    for `known` by warps that have not followed the ring would prove nothing if it came first."""
    text = code("linear_chunks.cu")
    for product, role in (("qk_full", between(text, "const int r = tid - 384", "weights_row(")), ("n_full", between(text, "j < own; j++, out +=", "write_out("))):
        waits = [m.group(1) for m in re.finditer(r"wait_\w+\(&H\.(\w+)|!told\(k\)", role)]
        assert waits[0] == product and len(waits) == 2, waits


def test_the_chain_waits_for_the_warp_that_has_the_other_half_of_its_rows():
    """With the delta rule two warps take places of a row out of rhs and u, by halves of the chunk's tokens; each then reads whether the row
    has any.  (The next w_full wants these warps' own arrivals, so that the phase seen is this chunk's.)"""
    chain = between(code("linear_delta.cu"), "for (int k = 0; k < chunks && ok; k++)", "store_state(")
    wait = re.search(r"wait_here\(&H\.u_full, k & 1, &H\) \|\| !wait_here\(&H\.w_full, k & 1, &H\)", chain)
    assert wait and chain.index("arrive_warp(&H.w_full)") < wait.start() < chain.index("dec.bad[row]")
