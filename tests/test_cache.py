"""The paged key/value cache against plain statements in 64 bits: tables and slots, the rotary store,
attention over the pages, at the sizes and masks where they can go wrong; and what is refused."""
import ctypes as C
import math
import os
import random
import subprocess

import pytest
import torch

from biv_b200 import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# half the distance of two neighbours of a type, relative
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def cache(heads=4, heads_kv=2, dim=64, page=16, seqs=64, tokens=8192, dtype=BF16, **kw):
    from biv_b200.cache import PagedCache
    return PagedCache(heads, heads_kv, dim, page, seqs, tokens, dtype, **kw)


# ---- without a GPU ---------------------------------------------------------------------------------
def test_argument_structs_have_the_header_s_sizes(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "bivmoe.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", sizeof(bivmoe_cache_desc), '
                   "sizeof(bivmoe_extend_args), sizeof(bivmoe_store_args), sizeof(bivmoe_attend_args)); return 0; }\n")
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(t) for t in (capi.CacheDesc, capi.ExtendArgs, capi.StoreArgs, capi.AttendArgs)]


def test_null_arguments_are_refused():
    L = capi.lib()
    assert L.bivmoe_cache_create(None, None) == capi.ERR_ARGUMENT
    for call in (L.bivmoe_cache_extend, L.bivmoe_cache_store, L.bivmoe_cache_attend):
        assert call(None, None, None) == capi.ERR_ARGUMENT
    assert L.bivmoe_cache_status(None, None) == capi.ERR_ARGUMENT
    L.bivmoe_cache_destroy(None)


def desc(**kw):
    d = capi.CacheDesc()
    for k, v in dict(ggml_type=30, n_head=4, n_head_kv=2, head_dim=64, page_size=16, max_seqs=8, max_tokens=64, rope_base=10000.0).items():
        setattr(d, k, v)
    for k, v in kw.items():
        if k == "rope_sections":
            for i, s in enumerate(v):
                d.rope_sections[i] = s
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("code, bad", [
    (capi.ERR_UNSUPPORTED, dict(ggml_type=0)), (capi.ERR_UNSUPPORTED, dict(head_dim=96)), (capi.ERR_ARGUMENT, dict(n_head=5)),
    (capi.ERR_ARGUMENT, dict(n_head_kv=0)), (capi.ERR_ARGUMENT, dict(page_size=0)), (capi.ERR_ARGUMENT, dict(max_seqs=1025)),
    (capi.ERR_ARGUMENT, dict(max_tokens=0)), (capi.ERR_ARGUMENT, dict(n_rot=80)), (capi.ERR_UNSUPPORTED, dict(n_rot=24)),
    (capi.ERR_ARGUMENT, dict(n_rot=64, rope_axes=5)), (capi.ERR_ARGUMENT, dict(n_rot=64, rope_axes=2, rope_sections=[16, 8])),
    (capi.ERR_ARGUMENT, dict(n_rot=64, rope_axes=1, rope_sections=[32], rope_base=0.0)),
    (capi.ERR_ARGUMENT, dict(n_rot=64, rope_axes=3, rope_interleaved=1, rope_sections=[4, 24, 4])),
])
def test_descriptors_that_are_refused(code, bad):
    h = C.c_void_p()
    assert capi.lib().bivmoe_cache_create(C.byref(desc(**bad)), C.byref(h)) == code
    assert not h.value and capi.lib().bivmoe_global_error()


# ---- extend ----------------------------------------------------------------------------------------
def extend_by_hand(page, past, added, held, free, count, table, width, n):
    """One request after another, one token after another."""
    length, first, slots, positions, kept, taken = [], [0], [], [], [], 0
    table = [list(r) for r in table]
    count = max(0, min(count, len(free)))
    for b, (p, a) in enumerate(zip(past, added)):
        have = held[b] if held is not None else -(-p // page)
        need = max(0, -(-(p + a) // page) - have)
        beyond = {}
        for j in range(have, have + need):
            got = free[count - 1 - taken] if taken < count else -1
            taken += 1
            if j < width:
                table[b][j] = got
            beyond[j] = got
        for t in range(p, p + a):
            pg = table[b][t // page] if t // page < width else -1
            slots.append(pg * page + t % page if pg >= 0 else -1)
            positions.append(t)
        length.append(p + a)
        first.append(first[-1] + a)
        kept.append(have + need)
    slots, positions = (slots + [-1] * n)[:n], (positions + [0] * n)[:n]
    return length, first, slots, positions, [max(0, count - taken), max(0, taken - count)], kept, table


@pytest.mark.gpu
@pytest.mark.parametrize("seqs, page, most, spare, pad, use_held", [
    (1, 16, 1, 4, 0, False), (3, 1, 5, 0, 7, False), (64, 16, 3, 2, 0, False), (257, 48, 40, 9, 3, True),
    (1000, 16, 70, -20, 0, False), (1024, 7, 9, 1, -11, True), (5, 64, 0, 3, 2, False), (2, 256, 5000, 1, 0, False)])
def test_extend(seqs, page, most, spare, pad, use_held):
    r = random.Random(seqs * 31 + page)
    past = [r.choice([0, 1, page - 1, page, page + 1, r.randint(0, 900)]) for _ in range(seqs)]
    added = [r.choice([0, 1, r.randint(0, most)]) if most else 0 for _ in range(seqs)]
    held = [-(-p // page) + r.choice([0, 0, 1, 3]) for p in past] if use_held else None
    width = max(-(-(p + a) // page) for p, a in zip(past, added)) + 4 - (3 if seqs == 1024 else 0)
    need = sum(max(0, -(-(p + a) // page) - (held[b] if held else -(-p // page))) for b, (p, a) in enumerate(zip(past, added)))
    numbers = list(range(need + max(spare, 0) + 3 + seqs * width))
    r.shuffle(numbers)
    free = numbers[:need + max(spare, 0) + 3]
    count = need + spare
    rest = iter(numbers[len(free):])
    table = [[next(rest) if j < (held[b] if held else -(-past[b] // page)) else -9 for j in range(width)] for b in range(seqs)]
    n = max(0, sum(added) + pad)
    c = cache(page=page, seqs=seqs, tokens=max(n, 1))
    wide = torch.full((seqs, width + 3), -7, dtype=torch.int32, device=DEV)     # rows that are not neighbours
    wide[:, :width] = ints(table)
    t = wide[:, :width]
    want = extend_by_hand(page, past, added, held, free, count, table, width, n)
    for _ in range(2):        # the lists are not changed: the same call gives the same again
        s = c.extend(ints(past), ints(added), ints(free), ints([count]), t, n, held=None if held is None else ints(held))
        got = [x.tolist() for x in (s.length, s.first, s.slots, s.positions, s.left, s.held, t)]
        assert got == [list(x) for x in want]
    assert bool((wide[:, width:] == -7).all())


@pytest.mark.gpu
def test_extend_into_its_own_lists_is_refused():
    c = cache(page=4, seqs=2, tokens=4)
    table, past, count = torch.full((2, 2), -1, dtype=torch.int32, device=DEV), ints([0, 0]), ints([3])
    s = c.extend(past, ints([1, 1]), ints([7, 8, 9]), count, table, 2)
    cases = [(count, s._replace(length=past)), (count, s._replace(held=past)), (count, s._replace(first=table.view(-1))), (s.left[1:], s)]
    for free_count, bad in cases:
        with pytest.raises(capi.BivMoeError) as e:
            c.extend(past, ints([1, 1]), ints([7, 8, 9]), free_count, table, 2, out=bad)
        assert e.value.code == capi.ERR_ARGUMENT


@pytest.mark.gpu
def test_extend_of_lists_that_do_not_fit():
    c = cache(page=4, seqs=4, tokens=16)
    table = torch.full((3, 2), -1, dtype=torch.int32, device=DEV)
    s = c.extend(ints([-5, 100, 2]), ints([-1, 3, 2]), ints([7, 8]), ints([99]), table, 8)
    big = 2 ** 31 - 1
    t = c.extend(ints([big, big, 5]), ints([big, 1, 1]), ints([7, 8]), ints([2]), table.clone(), 8, held=ints([0, 0, 2]))
    assert t.slots.tolist() == [-1] * 8 and t.left.tolist()[0] == 0      # the first request takes what there is, past its table
    # request 1 has no place for its page in the table, and the free list holds two whatever the count says
    assert s.first.tolist() == [0, 0, 3, 5] and s.length.tolist() == [0, 103, 4]
    assert s.slots.tolist() == [-1] * 8      # request 2's page was never given (the table says -1)
    assert s.left.tolist() == [1, 0]


# ---- store -----------------------------------------------------------------------------------------
def turned64(x, pos, rope, n_rot):
    x = x.double().clone()
    pairs = n_rot // 2
    sec = rope.sections
    for i in range(pairs):
        if rope.interleaved:
            a = i % len(sec)
            a = a if i < len(sec) * sec[a] else 0
        else:
            a = next(k for k in range(len(sec)) if i < sum(sec[:k + 1]))
        t = pos[a].double() * rope.base ** (-2.0 * i / n_rot)
        u, v = (2 * i, 2 * i + 1) if rope.adjacent else (i, i + pairs)
        p, q = x[..., u].clone(), x[..., v].clone()
        co, si = torch.cos(t)[:, None], torch.sin(t)[:, None]
        x[..., u], x[..., v] = p * co - q * si, p * si + q * co
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("n, heads, heads_kv, dim, n_rot, sections, inter, adj, rows, dtype, page, order, skew", [
    (1, 16, 2, 256, 64, [12, 10, 10], True, False, F32, BF16, 16, "token", 0),
    (1, 1, 1, 64, 16, [8], False, True, F16, F16, 1, "head", 0),
    (77, 14, 2, 64, 64, [32], False, False, BF16, BF16, 48, "head", 0),
    (130, 4, 4, 128, 128, [16, 24, 24], False, False, F32, F16, 16, "token", 1),
    (33, 6, 3, 128, 96, [12, 12, 12, 12], True, True, BF16, F16, 7, "token", 1),
    (5, 8, 1, 256, 256, [50, 0, 78], False, True, F16, BF16, 64, "head", 3),
    (40, 2, 2, 64, 0, None, False, False, F32, BF16, 16, "token", 0)])
def test_store(n, heads, heads_kv, dim, n_rot, sections, inter, adj, rows, dtype, page, order, skew):
    from biv_b200.cache import Rope
    g = torch.Generator(device=DEV).manual_seed(n + dim)
    rope = Rope(n_rot, 1e6, sections, inter, adj) if n_rot else None
    c = cache(heads, heads_kv, dim, page, 1, n, dtype, rope=rope)
    # q, k and v side by side in rows that begin `skew` values off an aligned place
    total = (heads + 2 * heads_kv) * dim
    flat = torch.randn(n * (total + skew) + skew, generator=g, device=DEV, dtype=torch.float32).to(rows)
    x = flat[skew:].view(n, total + skew)[:, :total].unflatten(1, (-1, dim))
    q, k, v = x[:, :heads], x[:, heads:heads + heads_kv], x[:, heads + heads_kv:]
    pages = -(-n // page) + 2
    shape = (pages, heads_kv, page, dim) if order == "head" else (pages, page, heads_kv, dim)
    pools = [torch.full(shape, -3.0, dtype=dtype, device=DEV) for _ in range(2)]
    kp, vp = [p.transpose(1, 2) if order == "head" else p for p in pools]
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n]
    if n > 4:
        slots[1], slots[3] = -1, pages * page + 5      # without a page, and past the pool
    axes = len(sections) if sections else 1
    pos = torch.randint(0, 1 << 20, (axes, n), generator=g, device=DEV, dtype=torch.int32)
    got = c.store(q, k, v, kp, vp, slots, pos if rope else None)
    wq, wk = [turned64(t, pos, rope, n_rot) if rope else t.double() for t in (q, k)]
    want_k, want_v = torch.full_like(kp, -3.0).double(), torch.full_like(vp, -3.0).double()
    for t in range(n):
        s = int(slots[t])
        if 0 <= s < pages * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = wk[t], v[t].double()
    # one rounding to the cache's type, and before it a turn in f32: the sine and cosine of an angle of at
    # most half a turn in f32 (2^-24 of pi, and two units of theirs), two products and a sum: 2^-21 |(x, y)|
    for a, w in ((got, wq), (kp, want_k), (vp, want_v)):
        far = (a.double() - w).abs()
        assert bool((far <= UNIT[dtype] * w.abs() + 2.0 ** -21 * 8 + (2.0 ** -25 if dtype == F16 else 0)).all()), far.max()


# ---- attend ----------------------------------------------------------------------------------------
class Batch:
    """Requests with `past` tokens and `new` ones on shuffled pages; what no token owns is NaN."""

    def __init__(self, new, past, heads, heads_kv, dim, dtype, page, order="token", seed=1, junk=float("nan"), peaked=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.past, self.page, self.g = new, past, page, heads // heads_kv
        counts = [-(-(a + b) // page) for a, b in zip(new, past)]
        self.pages = sum(counts) + 3
        order_of = torch.randperm(self.pages, generator=g, device=DEV).tolist()
        width = max(counts + [1]) + 1
        rows, at = [], 0
        for k in counts:
            rows.append(order_of[at:at + k] + [-1] * (width - k))
            at += k
        self.table = ints(rows)
        shape = (self.pages, heads_kv, page, dim) if order == "head" else (self.pages, page, heads_kv, dim)
        self.k, self.v = [torch.full(shape, junk, dtype=dtype, device=DEV) for _ in range(2)]
        if order == "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for b, (a, p) in enumerate(zip(new, past)):
            t = torch.arange(a + p, device=DEV)
            pg = self.table[b].long()[t // page]
            for x in (self.k, self.v):
                x[pg, t % page] = torch.randn((a + p, heads_kv, dim), generator=g, device=DEV).to(dtype)
        self.q = (torch.randn((sum(new), heads, dim), generator=g, device=DEV) * peaked).to(dtype)
        first = [0]
        for a in new:
            first.append(first[-1] + a)
        self.first, self.length = ints(first), ints([a + b for a, b in zip(new, past)])

    def want(self, window=0, sinks=0, scale=None, drop=()):
        """(o, sum of the weights' |v|) in 64 bits; keys of `drop` ((request, position)) are absent."""
        d = self.q.shape[2]
        scale = 1 / math.sqrt(d) if scale is None else scale
        o, mag = torch.zeros(self.q.shape, dtype=torch.float64, device=DEV), torch.zeros(self.q.shape, dtype=torch.float64, device=DEV)
        at = 0
        for b, (a, p) in enumerate(zip(self.new, self.past)):
            if a and a + p > 0:
                t = torch.arange(a + p, device=DEV)
                pg = self.table[b].long()[t // self.page]
                i = torch.arange(p, p + a, device=DEV)[:, None]
                see = t[None] <= i
                if window:
                    see &= (t[None] > i - window) | (t[None] < sinks)
                for r, j in drop:
                    if r == b:
                        see[:, j] = False
                for h in range(self.q.shape[1]):
                    k, v = [x[pg, t % self.page, h // self.g].double() for x in (self.k, self.v)]
                    s = (self.q[at:at + a, h].double() @ k.T * scale).masked_fill(~see, -math.inf)
                    w = torch.softmax(s, -1).masked_fill(~see, 0.0)      # a row that sees nothing: zeros, not NaN
                    # a weight of zero takes nothing, whatever lies there; a row that sees a score that is
                    # not finite has no weights that are numbers
                    v = v.nan_to_num(0.0, 0.0, 0.0)
                    o[at:at + a, h], mag[at:at + a, h] = w @ v, w @ v.abs()
            at += a
        return o, mag

    def run(self, c, **kw):
        return c.attend(self.q, self.k, self.v, self.table, self.first, self.length, **kw)


def near(got, want, dtype):
    """The weights are rounded to the type (each by at most UNIT of itself), the result once more; the
    scores, sums of up to 256 products in f32, and the power of two of them move a weight by less than
    2^-13 of itself."""
    o, mag = want
    far = (got.double() - o).abs()
    most = UNIT[dtype] * o.abs() + (UNIT[dtype] + 2.0 ** -13) * mag + 1e-7
    assert bool((far <= most).all()), float((far / most).nan_to_num(nan=1e30).max())


SHAPES = [
    # new, past, heads, heads_kv, dim, type, page, order, window, sinks
    ([1], [0], 1, 1, 64, BF16, 16, "token", 0, 0),
    ([1], [1000], 16, 2, 256, BF16, 16, "token", 0, 0),
    ([1, 1, 1], [0, 63, 64], 8, 8, 128, F16, 16, "head", 0, 0),
    ([1] * 40, list(range(0, 4000, 100)), 32, 8, 128, BF16, 16, "token", 0, 0),
    ([1, 0, 3, 0, 17], [5, 9, 0, 0, 300], 14, 2, 64, F16, 1, "token", 0, 0),
    ([5] * 7, [130, 0, 1, 127, 128, 129, 3000], 16, 2, 256, F16, 64, "head", 0, 0),
    ([300], [0], 4, 4, 128, BF16, 48, "token", 0, 0),
    ([513, 1, 129], [0, 20000, 255], 16, 2, 128, BF16, 32, "token", 0, 0),
    ([257], [1100], 6, 2, 256, BF16, 256, "head", 0, 0),
    ([400, 33], [77, 0], 7, 1, 64, BF16, 8, "head", 0, 0),
    ([1, 1], [3000, 12], 64, 8, 64, BF16, 16, "token", 128, 4),
    ([1, 1], [3000, 12], 8, 8, 128, F16, 16, "token", 1, 0),
    ([900, 5], [0, 2000], 8, 2, 64, F16, 16, "token", 100, 130),
    ([600], [1500], 4, 1, 256, BF16, 32, "token", 257, 1),
    ([700], [10], 4, 2, 128, BF16, 16, "head", 1000, 4),
    ([129], [0], 130, 1, 64, BF16, 16, "token", 3, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("new, past, heads, heads_kv, dim, dtype, page, order, window, sinks", SHAPES)
def test_attend(new, past, heads, heads_kv, dim, dtype, page, order, window, sinks, known):
    b = Batch(new, past, heads, heads_kv, dim, dtype, page, order)
    c = cache(heads, heads_kv, dim, page, len(new), sum(new), dtype)
    kw = dict(window=window, sinks=sinks, max_new=max(new) if known else 0)
    got = b.run(c, **kw)
    near(got, b.want(window, sinks), dtype)
    again = b.run(c, **kw)
    c.status()
    assert torch.equal(got, again)      # the pieces of a long axis are joined in their own order


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new, past", [([1, 1], [700, 90]), ([200, 40], [100, 0])])
def test_attend_scores_far_apart(dim, new, past):
    # scores of some hundreds either way: the running maximum moves again and again
    b = Batch(new, past, 4, 2, dim, BF16, 16, peaked=30.0)
    near(b.run(cache(4, 2, dim, 16, 2, 512, BF16)), b.want(), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new, past", [([1] * 40, [3000] * 40), ([140] * 6, [2000] * 6)])
def test_many_small_weights_beside_a_large_one(new, past, dim, dtype):
    # four keys hold all but 2^-18.73 of a weight each and have values of zero: the result is what the others
    # come to, weights that f16 has 6 bits for if the largest is 1
    b = Batch(new, past, 8, 4, dim, dtype, 16, seed=17)
    b.q.fill_(1.0)
    b.k.fill_(0.0)
    b.v.fill_(1.0)
    for j in (0, 16, 32, 48):
        at = b.table[:, j // 16].long()
        b.k[at, 0] = 18.73 * math.log(2.0) / math.sqrt(dim)
        b.v[at, 0] = 0.0
    near(b.run(cache(8, 4, dim, 16, len(new), sum(new), dtype)), b.want(), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new, past", [([3, 2], [100, 0]), ([300, 150], [20, 700])])
def test_values_a_row_does_not_see_do_not_reach_it(dim, new, past):
    # the last token of each request, and one that only the window's rows before it see, are not finite
    b = Batch(new, past, 4, 2, dim, BF16, 16)
    for r, (a, p) in enumerate(zip(new, past)):
        for j, bad in ((a + p - 1, float("nan")), (a + p - 2, float("inf"))):
            b.v[int(b.table[r, j // 16]), j % 16] = bad
            b.k[int(b.table[r, j // 16]), j % 16] = bad
    got = b.run(cache(4, 2, dim, 16, 2, 512, BF16))
    o, mag = b.want()
    at = 0
    for a in new:
        rows = slice(at, at + a - 2)
        near(got[rows], (o[rows], mag[rows]), BF16)
        assert bool(got[at + a - 2:at + a].isnan().all())     # those that see them
        at += a


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 4], [200, 70]])
def test_pages_that_are_not_there(new):
    b = Batch(new, [100, 60], 4, 2, 64, BF16, 16)
    b.table[0, 2], b.table[1, 0] = -1, b.pages + 7
    drop = [(0, j) for j in range(32, 48)] + [(1, j) for j in range(16)]
    t = b.table.clone()
    got = b.run(cache(4, 2, 64, 16, 2, 512, BF16))
    b.table[0, 2], b.table[1, 0] = 0, 0        # for the statement: any page, its keys are dropped
    b.k.nan_to_num_(0), b.v.nan_to_num_(0)
    near(got, b.want(drop=drop), BF16)
    # a table too narrow for the lengths: what lies past it is not there
    b.table = t
    narrow = t[:, :3]
    got = b.q.new_full(b.q.shape, 9.0)
    cache(4, 2, 64, 16, 2, 512, BF16).attend(b.q, b.k, b.v, narrow, b.first, b.length, out=got)
    b.table[0, 2], b.table[1, 0] = 0, 0
    near(got, b.want(drop=drop + [(r, j) for r in (0, 1) for j in range(48, new[r] + (100, 60)[r])]), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 150])
def test_rows_that_see_nothing_are_zeros_and_others_are_left(rows):
    b = Batch([rows, 1], [0, 40], 4, 2, 64, BF16, 16)
    out = torch.full((rows + 4, 4, 64), 7.0, dtype=BF16, device=DEV)
    q = torch.cat([b.q, b.q.new_full((3, 4, 64), float("nan"))])
    # request 0 says it has one token fewer than rows: its first row lies before the beginning
    b.length[0] -= 1
    cache(4, 2, 64, 16, 2, 512, BF16).attend(q, b.k, b.v, b.table, b.first, b.length, out=out)
    assert bool((out[0] == 0).all()) and bool((out[rows + 1:] == 7.0).all())
    o = torch.softmax(torch.zeros(1), 0)      # the second row sees the first key alone
    assert o.item() == 1.0
    want = b.v[int(b.table[0, 0]), 0].repeat_interleave(2, 0)
    assert torch.equal(out[1], want)
    b.length[:] = 0
    cache(4, 2, 64, 16, 2, 512, BF16).attend(q, b.k, b.v, b.table, b.first, b.length, out=out)
    assert bool((out[:rows + 1] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[2, 1], [90, 140]])
def test_lists_that_do_not_fit_the_rows(new):
    # `first` runs past the rows, backwards, or below zero: rows are cut, nothing is read or written outside
    b = Batch(new, [30, 50], 4, 2, 64, BF16, 16)
    c = cache(4, 2, 64, 16, 2, 512, BF16)
    n = sum(new)
    right = b.run(c)
    b.first[2] += 1000
    b.length[1] += 1000
    got = b.run(c)
    assert torch.equal(got[:new[0]], right[:new[0]])
    near(got[new[0]:], tuple(x[new[0]:] for x in b.want()), BF16)
    out = torch.full_like(b.q, 5.0)
    for first in ([0, -4, -9], [n + 7, n + 9, n + 20], [5, 2, 1]):
        c.attend(b.q, b.k, b.v, b.table, ints(first), b.length, out=out)
    torch.cuda.synchronize()
    assert bool((out == 5.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new, past, dim", [([1, 3], [200, 0], 128), ([130, 60], [0, 500], 64), ([140, 60], [0, 500], 256)])
def test_attend_strided_rows_on_another_stream(new, past, dim):
    b = Batch(new, past, 8, 2, dim, F16, 16)
    n = sum(new)
    wide = torch.randn((n, 13, dim), device=DEV).to(F16)
    wide[:, 2:10] = b.q
    c = cache(8, 2, dim, 16, 2, 512, F16)
    out = torch.full((8, n, dim + 8), 3.0, dtype=F16, device=DEV)      # heads first
    view = out[:, :, :dim].transpose(0, 1)
    near(b.run(c), b.want(), F16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attend(wide[:, 2:10], b.k, b.v, b.table, b.first, b.length, out=view)
    torch.cuda.current_stream().wait_stream(side)
    near(view, b.want(), F16)
    assert bool((out[:, :, dim:] == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 140])
def test_offsets_past_32_bits(rows):
    # 2^31 and more values between the pages: 5 GB to a pool
    d, page, pages = 64, 16, 2_600_000
    pool = torch.empty((2, pages, page, 1, d), dtype=BF16, device=DEV)
    b = Batch([rows], [100], 2, 1, d, BF16, page)
    used = -(-(rows + 100) // page)
    far = torch.arange(pages - used, pages, device=DEV, dtype=torch.int32)
    for x, y in ((pool[0], b.k), (pool[1], b.v)):
        x[far.long()] = y[b.table[0, :used].long()]
    got = cache(2, 1, d, page, 1, 512, BF16).attend(b.q, pool[0], pool[1], far[None], b.first, b.length)
    near(got, b.want(), BF16)


@pytest.mark.gpu
def test_a_step_in_a_graph_follows_its_lists():
    from biv_b200.cache import Rope
    c = cache(4, 2, 64, 16, 2, 8, BF16, rope=Rope(64))
    k, v = c.pools(20)
    k.fill_(float("nan")), v.fill_(float("nan"))
    table = torch.full((2, 8), -1, dtype=torch.int32, device=DEV)
    past, added, free, count = ints([0, 0]), ints([1, 1]), torch.arange(20, dtype=torch.int32, device=DEV), ints([20])
    x = torch.randn((40, 2, 8, 64), device=DEV)
    row = torch.empty((2, 8, 64), device=DEV)

    def step(out=None):
        s = c.extend(past, added, free, count, table, 2, out=out)
        q = c.store(row[:, :4], row[:, 4:6], row[:, 6:], k, v, s.slots, s.positions)
        return s, c.attend(q, k, v, table, s.first, s.length, max_new=1)

    keep, _ = step()
    table.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s, out = step(keep)
        past.copy_(s.length)
        count.copy_(s.left[:1])
    outs = []
    for i in range(40):
        row.copy_(x[i])
        graph.replay()
        outs.append(out.clone())
    assert past.tolist() == [40, 40] and count.tolist() == [20 - 2 * 3]
    # the same forty tokens at once
    table2 = torch.full((2, 8), -1, dtype=torch.int32, device=DEV)
    c2 = cache(4, 2, 64, 16, 2, 80, BF16, rope=Rope(64))
    k2, v2 = c2.pools(20)
    s2 = c2.extend(ints([0, 0]), ints([40, 40]), free, ints([20]), table2, 80)
    y = x.transpose(0, 1).reshape(80, 8, 64)
    q2 = c2.store(y[:, :4], y[:, 4:6], y[:, 6:], k2, v2, s2.slots, s2.positions)
    whole = c2.attend(q2, k2, v2, table2, s2.first, s2.length, max_new=40)
    apart = torch.stack(outs).transpose(0, 1).reshape(80, 4, 64)
    # two results within the bound of `near` of the same: weights of at most one on values of some units
    assert float((whole.float() - apart.float()).abs().max()) <= 4 * 2.0 ** -8 * float(v2[table2[table2 >= 0].long()].nan_to_num().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 3], [150, 40]])
def test_out_may_be_q_and_windows_may_be_as_wide_as_an_int(new):
    b = Batch(new, [300, 20], 4, 2, 64, BF16, 16)
    b.v[int(b.table[0, 3]), 5, 1, 7] = float("inf")        # rows that are made again read their q again
    c = cache(4, 2, 64, 16, 2, 512, BF16)
    want = b.run(c)
    assert bool(want.isinf().any())
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1)):
        assert torch.equal(b.run(c, window=window, sinks=sinks), want)
    b.length[0] = new[0] - 1        # a first row before the beginning, beside a window that reaches back further than an int
    near(b.run(c, window=2 ** 31 - 1)[new[0]:], tuple(x[new[0]:] for x in b.want()), BF16)
    b.length[0] = new[0] + 300
    assert b.run(c, out=b.q) is b.q and torch.equal(b.q, want)


@pytest.mark.gpu
def test_calls_that_are_refused():
    b = Batch([1, 2], [30, 50], 4, 2, 64, BF16, 16)
    c = cache(4, 2, 64, 16, 2, 4, BF16)

    def code(**kw):
        a = dict(q=b.q, k=b.k, v=b.v, table=b.table, first=b.first, length=b.length, more={})
        a.update(kw)
        with pytest.raises((capi.BivMoeError, ValueError)) as e:
            c.attend(a["q"], a["k"], a["v"], a["table"], a["first"], a["length"], **a["more"])
        return getattr(e.value, "code", "value")

    odd = torch.zeros(3 * 4 * 64 + 8, dtype=BF16, device=DEV)
    assert code(q=odd[1:1 + 3 * 256].view(3, 4, 64)) == capi.ERR_ARGUMENT                       # not on 16 bytes
    assert code(q=torch.zeros((5, 4, 64), dtype=BF16, device=DEV)) == capi.ERR_ARGUMENT         # more than max_tokens
    assert code(more=dict(window=-1)) == capi.ERR_ARGUMENT
    assert code(more=dict(scale=float("nan"))) == capi.ERR_ARGUMENT
    assert code(k=b.k[:2]) == capi.ERR_ARGUMENT                                                 # pools of different sizes
    assert code(q=b.q.half()) == "value" and code(k=b.k[:, :8]) == "value" and code(table=b.table.long()) == "value"
    assert code(length=ints([1, 2, 3]), table=torch.zeros((3, 2), dtype=torch.int32, device=DEV), first=ints([0] * 4)) == capi.ERR_ARGUMENT
    assert code(first=b.first.cpu()) == "value"
    with pytest.raises(ValueError):
        c.store(b.q, b.q[:, :2].float(), b.q[:, :2], b.k, b.v, torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(capi.BivMoeError):
        c.extend(ints([0]), ints([1]), ints([]), ints([0]), torch.zeros((1, 1), dtype=torch.int32, device=DEV), 5)
    # nothing to do is not an error
    assert c.attend(b.q[:0], b.k, b.v, b.table, ints([0, 0, 0]), b.length).shape[0] == 0
    near(b.run(c), b.want(), BF16)


@pytest.mark.gpu
def test_no_rows_and_no_requests():
    c = cache(4, 2, 64, 16, 2, 4, BF16)
    none = ints([])
    s = c.extend(none, none, ints([3]), ints([1]), torch.zeros((0, 4), dtype=torch.int32, device=DEV), 2)
    assert s.first.tolist() == [0] and s.slots.tolist() == [-1, -1] and s.left.tolist() == [1, 0]
    k, v = c.pools(2)
    z = torch.zeros((0, 4, 64), dtype=BF16, device=DEV)
    assert c.store(z, z[:, :2], z[:, :2], k, v, torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (0, 4, 64)


# ---- the operators together ---------------------------------------------------------------------------
def shares_by_hand(units, extra, snap, least, grid):
    """The blocks' pieces of tiles of `units` each, as (tile, part, parts, first unit, end, place)."""
    total = sum(units)
    first = [0]
    for u in units:
        first.append(first[-1] + u)
    g = min(-(-total // least), grid)
    each, more = divmod(total, g)
    longer = more * (each + 1)

    def owner(u):
        return u // (each + 1) if u < longer else longer // (each + 1) + (u - longer) // each

    got = []
    for c in range(g):
        lo = each * c + min(c, more)
        hi = lo + each + (c < more)
        t = next(i for i in range(len(units)) if lo < first[i + 1])
        at, off = lo, lo - first[t]
        if off <= snap:
            at, off = at - off, 0
        elif units[t] - off <= snap:
            at, off, t = at + units[t] - off, 0, t + 1
        while at < hi:
            u0, end = at - off, units[t]
            if hi - u0 < units[t]:
                if hi - u0 <= snap:
                    break
                if units[t] - (hi - u0) > snap:
                    end = hi - u0
            c0, part, parts, place = c, 0, 1, None
            if off or end < units[t]:
                c0 = owner(u0 + snap)
                parts, part = owner(u0 + units[t] - snap - 1) - c0 + 1, c - c0
                place = 2 * c0 + 1 if part == 0 else 2 * c
            got.append((t, part, parts, off, end, place))
            at, off = u0 + end, end
            if end == units[t]:
                t, off = t + 1, 0
    return got


def test_every_unit_is_in_one_piece_and_every_piece_has_a_place():
    # the arithmetic of the blocks' shares, as the kernels do it (cache.cuh), over random batches
    r = random.Random(5)
    for _ in range(300):
        snap = r.randint(1, 6)
        extra = r.randint(0, snap)
        units = [extra + 1 + (r.randint(0, 5) if r.random() < 0.6 else r.randint(0, 120)) for _ in range(r.randint(1, 40))]
        got = shares_by_hand(units, extra, snap, r.randint(1, 4), r.randint(1, 150))
        places = [p[5] for p in got if p[5] is not None]
        assert len(set(places)) == len(places)
        for t, u in enumerate(units):
            mine = sorted(p for p in got if p[0] == t)
            assert [p[1] for p in mine] == list(range(mine[0][2]))          # parts 0, 1, ... of the number they say
            assert [p[3] for p in mine] == [0] + [p[4] for p in mine[:-1]] and mine[-1][4] == u
            assert all(p[4] > extra for p in mine)                          # none without a key


@pytest.mark.gpu
def test_both_kernels_take_any_number_of_rows():
    b = Batch([1, 4, 2], [500, 70, 3000], 8, 2, 128, BF16, 16)
    c = cache(8, 2, 128, 16, 3, 512, BF16)
    one, other = b.run(c, max_new=4), b.run(c, max_new=0)      # 16 rows a request; not known: 28
    wide = Batch([9, 12, 40], [500, 70, 3000], 8, 2, 128, BF16, 16)
    o = wide.want()
    near(wide.run(c, max_new=8), o, BF16)                      # fewer than there are: the speed's matter alone
    near(wide.run(c, max_new=40), o, BF16)
    near(one, b.want(), BF16)
    near(other, b.want(), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
@pytest.mark.parametrize("new", [[1, 2], [150, 40]])
def test_attend_scales(scale, new):
    b = Batch(new, [300, 20], 4, 2, 64, F16, 16)
    near(b.run(cache(4, 2, 64, 16, 2, 512, F16), scale=scale), b.want(scale=scale), F16)


@pytest.mark.gpu
def test_a_prompt_in_chunks_and_token_by_token_is_the_prompt_at_once():
    import sys
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decoder
    x = torch.randn((3 * 150, 512), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).view(3, 150, 512)

    def outs(cuts):
        d = decoder.Decoder(layers=1, requests=3, n_pages=96)
        got = []
        for lo, hi in zip(cuts, cuts[1:]):
            n = hi - lo
            s = d.cache.extend(d.past, ints([n] * 3), d.free, d.free_count, d.table, 3 * n)
            got.append(d.layers[0].attention(x[:, lo:hi].reshape(-1, 512), s, d.table, n).view(3, n, 512))
            d.past.copy_(s.length), d.free_count.copy_(s.left[:1])
        d.close()
        return torch.cat(got, 1)

    whole, apart = outs([0, 150]), outs([0, 64, 65, 100] + list(range(101, 151)))
    # the same keys and weights; the sums' order and the roundings of weights, o and the product's rows differ
    assert float((whole - apart).norm() / whole.norm()) < 4 * UNIT[BF16]
    d = decoder.Decoder(layers=2, requests=3, n_pages=96)
    y = x[:, :40].reshape(-1, 512).contiguous()
    d.step(y, ints([40] * 3), 40)
    d.cache.status()
    assert bool(y.isfinite().all()) and d.past.tolist() == [40] * 3
    d.close()
