"""The paged cache at its edges: values that are not finite or near that, lists that run out, views, streams and
waits that meet, the shares of the work, the build."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from biv_b200 import capi
from test_cache import BF16, DEV, F16, F32, ROOT, UNIT, Batch, cache, ints, near, turned64


# ---- values that are not finite ----------------------------------------------------------------------
def peaked_batch(new, past, dim, dtype, low):
    """All scores 0, those of the keys `low(j)` 300 powers of two below: their weights are zero in 32 bits."""
    b = Batch(new, past, 8, 2, dim, dtype, 16, seed=5)
    b.q.fill_(1.0)
    for r, (a, p) in enumerate(zip(new, past)):
        t = torch.arange(a + p, device=DEV)
        k = torch.where(low(t), -300.0 * math.log(2.0) / math.sqrt(dim), 0.0)
        b.k[b.table[r].long()[t // 16], t % 16] = k[:, None, None].expand(-1, 2, dim).to(dtype)
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("what, bad", [("k", "nan"), ("k", "inf"), ("v", "nan"), ("v", "inf")])
def test_a_value_a_row_sees_reaches_it_whatever_its_weight(what, bad, new, dim, dtype):
    # 4 rows a kv head, and 160: both kernels; keys far below the best ones in pieces of their own (the first
    # ones, and the first half of the request), and within a tile (sixteen of 64, what one warp takes)
    for low, at in ((lambda t: t < 192, 100), (lambda t: t < 2500, 100), (lambda t: (t // 16) % 4 == 1, 4949)):
        b = peaked_batch([new, new], [5000, 5000], dim, dtype, low)
        clean = b.run(cache(8, 2, dim, 16, 2, 512, dtype), max_new=new)
        near(clean, b.want(), dtype)
        getattr(b, what)[int(b.table[0, at // 16]), at % 16] = float(bad)
        c = cache(8, 2, dim, 16, 2, 512, dtype)
        got = b.run(c, max_new=new)
        c.status()
        assert not bool(got[:new].isfinite().any())
        assert torch.equal(got[new:], clean[new:])      # the request that does not see it


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_score_of_minus_infinity_is_a_weight_of_zero(dim, new):
    b = Batch([new, new], [900, 30], 8, 2, dim, BF16, 16)
    b.q.abs_()
    b.k[int(b.table[0, 50]), 3] = -math.inf
    b.k[b.table[1][b.table[1] >= 0].long()] = -math.inf   # no key of the second request has a weight: zeros
    got = b.run(cache(8, 2, dim, 16, 2, 512, BF16), max_new=new)
    b.k.nan_to_num_(0, 0, 0)
    want = b.want(drop=[(0, 803)])
    near(got[:new], tuple(x[:new] for x in want), BF16)
    assert bool((got[new:] == 0).all())


def sees(p, j, window, sinks):
    return j <= p and (not window or p - j < window or j < sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dim, dtype", [(64, BF16), (128, F16), (256, BF16)])
@pytest.mark.parametrize("new, past", [([4, 2], [700, 90]), ([300, 150], [50, 700])])
@pytest.mark.parametrize("window, sinks", [(0, 0), (100, 0), (100, 70), (257, 3)])
def test_values_at_the_edges_of_what_a_row_sees(window, sinks, new, past, dim, dtype):
    # one value that is not finite, in places that some of the rows see: by their window's lower end, by the
    # end of the first tokens that stay visible, by their own position
    edges = {j + d for n, p in zip(new, past) for j in (p + n - 1, p + n // 2, p + n // 2 - window, p - window, sinks) for d in (-1, 0, 1)}
    c = cache(8, 2, dim, 16, 2, 512, dtype)
    b = Batch(new, past, 8, 2, dim, dtype, 16, seed=9)
    want = b.want(window, sinks)
    for j in sorted(edges):
        kept = b.v.clone()
        hit = [0 <= j < n + p for n, p in zip(new, past)]
        for r in range(2):
            if hit[r]:
                b.v[int(b.table[r, j // 16]), j % 16, 1, 5] = (math.inf, math.nan)[j % 2]
        got = b.run(c, window=window, sinks=sinks, max_new=max(new))
        at = 0
        for r, (n, p) in enumerate(zip(new, past)):
            see = torch.tensor([hit[r] and sees(p + i, j, window, sinks) for i in range(n)], device=DEV)
            rows = got[at:at + n]
            odd = torch.zeros_like(rows, dtype=torch.bool)
            odd[:, 4:, 5] = see[:, None]          # the heads of kv head 1, the value's place
            assert torch.equal(~rows.isfinite(), odd), (j, r)
            near(torch.where(odd, want[0][at:at + n].to(dtype), rows), tuple(x[at:at + n] for x in want), dtype)
            at += n
        b.v.copy_(kept)
    c.status()


@pytest.mark.gpu
@pytest.mark.parametrize("new, heads", [(256, 16), (4, 16)])
def test_a_long_past_with_a_value_that_is_not_finite(new, heads):
    # eight requests of 10^5 tokens: what one of them holds does not cost the others their results
    seqs, past, dim = 8, 100_000, 128
    b = Batch([new] * seqs, [past] * seqs, heads, 4, dim, BF16, 64, seed=3, junk=0.0)
    c = cache(heads, 4, dim, 64, seqs, new * seqs, BF16)
    clean = b.run(c, max_new=new)
    # an early value that all rows of request 3 see: its place in them, and nothing else
    at = (int(b.table[3, 1]), 7, 1, 9)
    was = b.v[at].clone()
    b.v[at] = math.inf
    got = b.run(c, max_new=new)
    c.status()
    odd = torch.zeros_like(got, dtype=torch.bool)
    odd[3 * new:4 * new, heads // 4:heads // 2, 9] = True
    assert torch.equal(~got.isfinite(), odd) and torch.equal(got[~odd], clean[~odd])
    b.v[at] = was
    # each request's last token holds values that none of its other rows sees
    last = past + new - 1
    for r in range(seqs):
        b.v[int(b.table[r, last // 64]), last % 64] = math.nan
    got = b.run(c, max_new=new).view(seqs, new, heads, dim)
    c.status()
    assert bool(got[:, -1].isnan().all()) and bool(got[:, :-1].isfinite().all())
    # against the run before: each is within `near`'s bound of the same, on values whose weights sum to one
    far = (got[:, :-1].double() - clean.view(got.shape)[:, :-1].double()).abs()
    o, mag = [x.view(got.shape)[:, :-1] for x in one_head(b, heads)]
    at = [0, heads // 4 * 2]                      # the heads that one_head states
    assert bool((far[:, :, at] <= 2 * (2.0 ** -8 * o[:, :, at].abs() + (2.0 ** -8 + 2.0 ** -13) * mag[:, :, at] + 1e-7)).all())


def one_head(b, heads):
    """`Batch.want` for the first head, and the first of kv head 2, alone."""
    o, mag = torch.zeros(b.q.shape, dtype=torch.float64, device=DEV), torch.zeros(b.q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for r, (n, p) in enumerate(zip(b.new, b.past)):
        t = torch.arange(n + p, device=DEV)
        pg = b.table[r].long()[t // b.page]
        see = t[None] <= torch.arange(p, p + n, device=DEV)[:, None]
        for h in (0, heads // 4 * 2):
            k, v = [x[pg, t % b.page, h // b.g].double() for x in (b.k, b.v)]
            w = torch.softmax((b.q[at:at + n, h].double() @ k.T / math.sqrt(k.shape[1])).masked_fill(~see, -math.inf), -1)
            v = v.nan_to_num(0.0, 0.0, 0.0)
            o[at:at + n, h], mag[at:at + n, h] = w @ v, w @ v.abs()
        at += n
    return o, mag


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 140])
def test_values_near_the_largest_there_are(dim, new):
    # all values 2^124 or minus that, where f32 ends at 2^128; one key's weight is 2^7 times any other's and comes
    # after many of them
    b = Batch([new, new], [900, 60], 8, 2, dim, BF16, 16, seed=21)
    b.q.fill_(1.0)
    b.k.copy_(torch.where(b.k.isnan(), b.k, 0.0))
    b.k[int(b.table[0, 200 // 16]), 200 % 16] = 7.0 * math.log(2.0) / math.sqrt(dim)
    b.v.copy_(torch.where(b.v.isnan(), b.v, b.v.sign() * 2.0 ** 124))
    c = cache(8, 2, dim, 16, 2, 512, BF16)
    near(b.run(c, max_new=new), b.want(), BF16)


def test_the_clock_of_a_wait_stands_while_another_role_is_at_work(tmp_path):
    src, exe = tmp_path / "clock.cpp", str(tmp_path / "clock")
    src.write_text(r"""
#include <cstdio>
#include <initializer_list>
#include "bounded_wait.h"
using namespace bivmoe;
static uint64_t now;
static int tries;
struct Wait {                     // ready never; a look every 1000 ns; another role at work until `until`
    uint64_t until; WaitClock clock{};
    bool ready() { tries++; return false; }
    bool late(uint32_t look) { return clock.late(look, now, now < until); }
    void pause() { now += 1000; }
};
int main() {
    for (uint64_t until : {0ull, 5ull * kWaitNs, 5ull * kWaitNs + 123456789}) {
        now = 77;
        tries = 0;
        if (bounded_wait<1>(Wait{until})) return 1;
        // gives up kWaitNs after the other role's end, and not without it
        const uint64_t from = until > 77 ? until : 77;
        if (now < from + kWaitNs - 2000 || now > from + kWaitNs + 2000) { printf("%llu\n", (unsigned long long)now); return 2; }
    }
    return 0;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "biv_b200", "csrc"), "-o", exe, str(src)], check=True)
    assert subprocess.run([exe], timeout=60).returncode == 0


def test_a_copying_warp_stays_until_its_last_fills_have_landed(tmp_path):
    # four warps fill a ring of eight; fills land late, by themselves; the consumer stops anywhere
    src, exe = tmp_path / "fills.cpp", str(tmp_path / "fills")
    src.write_text(r"""
#include <atomic>
#include <cstdio>
#include <mutex>
#include <random>
#include <thread>
#include <vector>
#include "bounded_wait.h"
using namespace bivmoe;
constexpr int SLOTS = 8, WARPS = 4;
struct Bar {                            // an mbarrier of one arrival
    std::mutex m; unsigned phase = 0;
    void arrive() { std::lock_guard<std::mutex> l(m); phase++; }
    bool test(unsigned parity) { std::lock_guard<std::mutex> l(m); return (phase & 1) != parity; }
};
int main() {
    std::mt19937 rng(2);
    for (int run = 0; run < 200; run++) {
        const int total = rng() % 50, used = rng() % (total + 1);
        Bar full[SLOTS], empty[SLOTS];
        std::atomic<bool> stop{false};
        std::atomic<int> bad{0};
        std::vector<std::thread> roles;
        for (int w = 0; w < WARPS; w++) {
            const unsigned seed = rng();
            roles.emplace_back([&, w, seed] {
                std::mt19937 r(seed);
                std::atomic<int> under_way{0};
                std::vector<std::thread> copies;
                uint32_t last = 0, fills = 0;
                for (int gs = w; gs < total; gs += WARPS) {
                    bool ok = true;
                    while (!empty[gs % SLOTS].test(((gs / SLOTS) & 1) ^ 1) && (ok = !stop)) std::this_thread::yield();
                    if (!ok) break;
                    last = gs;
                    fills++;
                    under_way++;
                    copies.emplace_back([&, gs, late = r() % 300] {
                        std::this_thread::sleep_for(std::chrono::microseconds(late));
                        under_way--;
                        full[gs % SLOTS].arrive();
                    });
                }
                wait_for_last_fills<SLOTS, WARPS>(last, fills, [&](uint32_t slot, uint32_t parity) {
                    while (!full[slot].test(parity)) std::this_thread::yield();
                });
                if (under_way) bad = 1;                     // it would land in memory that is another block's
                for (auto& c : copies) c.join();
            });
        }
        for (int gs = 0; gs < used; gs++) {                 // the consumer, until it gives up
            while (!full[gs % SLOTS].test((gs / SLOTS) & 1)) std::this_thread::yield();
            empty[gs % SLOTS].arrive();
        }
        stop = true;
        for (auto& r : roles) r.join();
        if (bad) { printf("run %d\n", run); return 1; }
    }
    return 0;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-Wall", "-I", os.path.join(ROOT, "biv_b200", "csrc"), "-o", exe, str(src)],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
    # and the kernel's copying warps end with it
    with open(os.path.join(ROOT, "biv_b200", "csrc", "attend_tc.cu")) as f:
        code = f.read()
    role = code[code.index("// ---- copies"):code.index("// ---- products")]
    assert "wait_for_last_fills<AT_SLOTS, AT_COPY_WARPS>(last, fills" in role[role.index("cp.async.wait_all"):]


@pytest.mark.gpu
def test_the_c_abi_s_argument_structs():
    # the calls by the structs that a ctypes caller fills, against the ones that take tensors
    from biv_b200.cache import Rope
    L, b = capi.lib(), Batch([3, 2], [0, 0], 4, 2, 64, BF16, 16, junk=0.0)
    c = cache(4, 2, 64, 16, 2, 8, BF16, rope=Rope(64))
    s = c.extend(ints([0, 0]), ints([3, 2]), ints([5, 6]), ints([2]), b.table, 5)
    x = torch.randn((5, 8, 64), device=DEV)
    k, v = [torch.zeros((8, 16, 2, 64), dtype=BF16, device=DEV) for _ in range(2)]
    q = c.store(x[:, :4], x[:, 4:6], x[:, 6:], k, v, s.slots, s.positions)
    want = c.attend(q, k, v, b.table, s.first, s.length)

    def rows(t):
        return (t.data_ptr(), t.stride(0), t.stride(1), {F32: 0, BF16: 30}[t.dtype], 0)

    def pool(t):
        return (t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), t.shape[0])

    table, k2, v2, q2, o2 = b.table.clone().fill_(-1), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(q)
    lists = [torch.zeros(n, dtype=torch.int32, device=DEV) for n in (2, 3, 5, 2, 2)]
    length, first, positions, left, held = lists
    slots = torch.zeros(5, dtype=torch.int64, device=DEV)
    ins = [ints([0, 0]), ints([3, 2]), ints([5, 6]), ints([2])]
    e = capi.ExtendArgs(ins[0].data_ptr(), ins[1].data_ptr(), None, ins[2].data_ptr(), ins[3].data_ptr(), table.data_ptr(), table.stride(0),
                        table.shape[1], 2, 2, 5, *[t.data_ptr() for t in lists], slots.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    capi.check(L.bivmoe_cache_extend(c._h, C.byref(e), stream))
    assert [t.tolist() for t in (length, first, slots, positions, left, held)] == [t.tolist() for t in s]
    a = capi.StoreArgs(*rows(x[:, :4]), *rows(x[:, 4:6]), *rows(x[:, 6:]), *rows(q2), *pool(k2), *pool(v2), slots.data_ptr(),
                       positions.data_ptr(), 5, 5, 0)
    capi.check(L.bivmoe_cache_store(c._h, C.byref(a), stream))
    assert torch.equal(q2, q) and torch.equal(k2, k) and torch.equal(v2, v)
    t = capi.AttendArgs(*rows(q2), *rows(o2), *pool(k2), *pool(v2), table.data_ptr(), table.stride(0), table.shape[1], 2, 5, 0,
                        first.data_ptr(), length.data_ptr(), 64 ** -0.5, 0, 0, 0)
    capi.check(L.bivmoe_cache_attend(c._h, C.byref(t), stream))
    assert torch.equal(o2, want)


# ---- streams -----------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_call_waits_for_all_before_it_after_a_capture():
    # a call on A; while A is captured a call on B; after it one on C, which uses the workspace of both
    b = Batch([1, 2], [300, 20], 4, 2, 64, BF16, 16)
    c = cache(4, 2, 64, 16, 2, 8, BF16)
    want = b.run(c)
    outs = [torch.zeros_like(b.q) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    ends = [torch.cuda.Event() for _ in range(3)]
    torch.cuda.synchronize()

    def call(i, wait):
        with torch.cuda.stream(streams[i]):
            if wait:
                torch.cuda._sleep(wait)
            b.run(c, out=outs[i])
            ends[i].record()

    graph = torch.cuda.CUDAGraph()
    call(0, 50_000_000)                     # some 25 ms
    with torch.cuda.stream(streams[0]):
        graph.capture_begin(capture_error_mode="relaxed")
        x = torch.zeros(1, device=DEV)
        call(1, 400_000_000)                # ends long after A's
        x += 1
        graph.capture_end()
    call(2, 0)
    ends[2].synchronize()
    assert ends[0].query() and ends[1].query()
    for o in outs:
        assert torch.equal(o, want)
    call(0, 400_000_000)                    # and once more without a capture
    call(1, 0)
    ends[1].synchronize()
    assert ends[0].query()


# ---- lists that run out ------------------------------------------------------------------------------
@pytest.mark.gpu
def test_tokens_without_a_page_are_counted_and_the_step_can_be_made_again():
    # three requests of pages of 4: 6, 1 and 5 new tokens on 0, 4 and 3; four pages are needed, two are there
    c = cache(4, 2, 64, 4, 3, 16, BF16)
    past, added, free = ints([0, 4, 3]), ints([6, 1, 5]), ints([9, 8, 7])
    table = torch.full((3, 3), -1, dtype=torch.int32, device=DEV)
    table[1, 0], table[2, 0] = 5, 6
    s = c.extend(past, added, free[:2], ints([2]), table, 13)
    assert s.left.tolist() == [0, 2] and s.slots.tolist() == [32, 33, 34, 35, 36, 37, -1, 27] + [-1] * 5
    assert c.unstored() == 1 + 4 and c.unstored() == 0
    # going on all the same: nothing new is needed, and the rows are lost without a missing page
    t = c.extend(s.length, ints([0, 2, 0]), free, ints([1]), table, 2, held=s.held)
    assert t.left.tolist() == [1, 0] and t.slots.tolist() == [-1, -1] and c.unstored() == 2
    # made again, with pages added at the end: what it needs is what it gets
    free = ints([9, 8, 7, 3])
    s = c.extend(past, added, free, ints([4]), table, 13)
    assert s.left.tolist() == [0, 0] and s.held.tolist() == [2, 2, 2] and c.unstored() == 0
    assert table.tolist() == [[3, 7, -1], [5, 8, -1], [6, 9, -1]]
    assert s.slots.tolist() == [12, 13, 14, 15, 28, 29, 32, 27, 36, 37, 38, 39, -1]


@pytest.mark.gpu
def test_tokens_past_the_table_or_the_rows_are_counted():
    c = cache(1, 1, 64, 4, 2, 16, BF16)
    past, added, free, count = ints([4, 0]), ints([5, 3]), ints([1, 2, 3]), ints([3])
    narrow = torch.full((2, 2), -1, dtype=torch.int32, device=DEV)
    narrow[0, 0] = 0
    s = c.extend(past, added, free, count, narrow, 8)
    assert s.slots.tolist() == [12, 13, 14, 15, -1, 4, 5, 6] and c.unstored() == 1
    wide = torch.full((2, 3), -1, dtype=torch.int32, device=DEV)
    wide[0, 0] = 0
    s = c.extend(past, added, free, count, wide, 8)      # again, with room: the same pages, none lost
    assert s.slots.tolist() == [12, 13, 14, 15, 8, 4, 5, 6] and s.left.tolist() == [0, 0] and c.unstored() == 0
    c.extend(past, added, free, count, wide, 6)          # two of eight tokens have no rows
    assert c.unstored() == 2
    graph = torch.cuda.CUDAGraph()
    c.extend(past, added, free, count, narrow, 8, out=s)
    with torch.cuda.graph(graph):
        c.extend(past, added, free, count, narrow, 8, out=s)
    for _ in range(5):
        graph.replay()
    assert c.unstored() == 6                             # every replay's


# ---- rows that are views -----------------------------------------------------------------------------
@pytest.mark.gpu
def test_positions_may_be_expanded_over_the_axes():
    # text tokens: the same position on every axis, one row of memory
    from biv_b200.cache import Rope
    rope, n = Rope(64, 1e6, [12, 10, 10], True), 33
    c = cache(4, 2, 64, 16, 1, n, BF16, rope=rope)
    x = torch.randn((n, 8, 64), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    k, v = [p.zero_() for p in c.pools(3)]
    pos = torch.arange(1000, 1000 + n, device=DEV, dtype=torch.int32)
    slots = torch.arange(n, device=DEV)
    got = c.store(x[:, :4], x[:, 4:6], x[:, 6:], k, v, slots, pos.expand(3, n))
    want = turned64(x[:, :4], pos.expand(3, n), rope, 64)
    # one rounding, and a turn in f32 before it (2^-21 of values of at most 8)
    assert bool(((got.double() - want).abs() <= UNIT[BF16] * want.abs() + 2.0 ** -21 * 8).all())
    again = c.store(x[:, :4], x[:, 4:6], x[:, 6:], k, v, slots, pos.expand(3, n).contiguous())
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_strides_of_a_single_token_head_or_page_do_not_count(new):
    # where there is one of something, its stride says nothing, and torch leaves it at anything
    def odd(t):      # the same memory; strides of 1 and 3 where a dimension has one place
        return t.as_strided(t.shape, [s if n > 1 else 1 + 2 * (i & 1) for i, (n, s) in enumerate(zip(t.shape, t.stride()))])

    b = Batch([new], [0], 1, 1, 64, BF16, 64)
    c = cache(1, 1, 64, 64, 1, 64, BF16)
    want = b.run(c)
    out = torch.zeros_like(b.q)
    k, v = [x[b.table[0, :1].long()].contiguous() for x in (b.k, b.v)]
    got = c.attend(odd(b.q), odd(k), odd(v), ints([[0]]), b.first, b.length, out=odd(out))
    assert torch.equal(got, want) and torch.equal(out, want)
    rows = torch.randn((new, 1, 64), device=DEV)
    slots = torch.arange(new, device=DEV)
    q = c.store(odd(rows), odd(rows), odd(rows), odd(k), odd(v), slots, out=odd(out))
    assert torch.equal(q, rows.to(BF16)) and torch.equal(k[0, :new], rows.to(BF16))


# ---- the build ---------------------------------------------------------------------------------------
def test_the_library_is_built_without_python():
    # the default target is what a caller of the C ABI needs: no interpreter is asked for anything
    make = ["make", "-n", "-B", "-C", os.path.join(ROOT, "biv_b200", "csrc"), "PYTHON=/nowhere/python"]
    r = subprocess.run(make, capture_output=True, text=True)
    assert r.returncode == 0 and "libbivmoe.so" in r.stdout and "_cache_calls" not in r.stdout and "nowhere" not in r.stderr
    r = subprocess.run(make[:-1] + ["all"], capture_output=True, text=True)
    assert r.returncode == 0 and "libbivmoe.so" in r.stdout and "_cache_calls.so" in r.stdout


# ---- the shares of the work --------------------------------------------------------------------------
SHARES = r"""
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "cache.cuh"
using namespace bivmoe;
static int bad;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s (batch %d)\n", __LINE__, #x, batch); if (++bad > 5) return; } } while (0)

// The pieces that the blocks take of random batches, by the kernels' own code.
template <int KT, int TR, int EXTRA, int SNAP, int LEAST> void check(int blocks, unsigned seed) {
    std::mt19937 rng(seed);
    auto up_to = [&](int n) { return (int)(rng() % (n + 1)); };
    for (int batch = 0; batch < 120; batch++) {
        AttendCall a{};
        a.n_seq = 1 + up_to(batch % 3 ? 30 : 3);
        a.heads_kv = 1 + up_to(7);
        a.group = FastDiv(1 + up_to(16));
        a.window = up_to(2) ? 0 : 1 + up_to(3000);
        a.sinks = up_to(300);
        std::vector<int32_t> first(1, 0), length;
        for (int b = 0; b < a.n_seq; b++) {
            const int rows = up_to(2) ? up_to(3) : up_to(400), past = up_to(3) ? up_to(5000) : up_to(60000);
            first.push_back(first.back() + rows);
            length.push_back(past + rows - (up_to(9) ? 0 : 1 + up_to(past + rows)));     // rows before the beginning
        }
        a.n_tokens = first.back() - (up_to(9) ? 0 : up_to(first.back()));               // fewer rows than the lists say
        a.first = first.data();
        a.length = length.data();
        std::vector<int64_t> before(1, 0);
        std::set<std::tuple<int, int, int>> tiles;
        for (int b = 0; b < a.n_seq; b++) {
            const Request r = request_of(a, b);
            int64_t units = 0;
            for (int t = 0; t * TR < r.rows; t++) {
                units += tile_units<KT, TR, EXTRA>(a, r, t);
                for (int h = 0; h < a.heads_kv; h++) tiles.insert({b, h, t});
            }
            before.push_back(before.back() + units * a.heads_kv);
        }
        std::map<std::tuple<int, int, int>, std::vector<Piece>> found;
        std::set<int> places, counts;
        int64_t most = 0, total = 0;
        for (int block = 0; block < blocks; block++) {
            Share s{};
            host_block() = block;
            s.before = before.data();
            s.take(before.back(), LEAST, blocks);
            CHECK(s.lo == total || s.lo == s.hi);
            total += s.hi - s.lo;
            for (int64_t u = s.lo; u < s.hi; u += 1 + up_to(5)) CHECK(s.owner(u) == block);
            Walk<KT, TR, EXTRA, SNAP> walk(a, s);
            int64_t mine = 0;
            for (Piece x; walk.next(x);) {
                found[{x.b, x.head, x.row0 / TR}].push_back(x);
                mine += EXTRA + x.n;
                CHECK(x.row0 % TR == 0 && x.part == block - x.c0);
                CHECK(x.rows == std::min(TR, x.r.rows - x.row0) && x.rows > 0);
                if (x.parts == 1) continue;
                CHECK(x.slot(x.part) >= 0 && x.slot(x.part) < 2 * blocks);              // the workspace: two to a block
                CHECK(places.insert(x.slot(x.part)).second);
                if (x.part == 0) CHECK(counts.insert(x.c0).second && x.c0 < blocks);    // a tile's count of arrivals is its own
            }
            most = std::max(most, mine);
        }
        CHECK(total == before.back());
        CHECK(found.size() == tiles.size());
        for (auto& f : found) {                       // every key tile of every tile is in one piece
            std::vector<Piece>& p = f.second;
            CHECK(tiles.count(f.first) && (int)p.size() == p[0].parts);
            int next = 0;
            for (size_t i = 0; i < p.size(); i++) {   // (the blocks were gone through in order)
                CHECK(p[i].part == (int)i && p[i].parts == p[0].parts && p[i].c0 == p[0].c0 && p[i].tiles.n == p[0].tiles.n);
                CHECK(p[i].i0 == next && (p[i].n > 0 || (p.size() == 1 && p[0].tiles.n == 0)));
                next += p[i].n;
            }
            CHECK(next == p[0].tiles.n);
            // and no key that a row sees is in another tile
            const Piece& x = p[0];
            const int p0 = x.r.past + (int)a.group.div(x.row0), p1 = x.r.past + (int)a.group.div(x.row0 + x.rows - 1);
            std::set<int> list;
            for (int i = 0; i < x.tiles.n; i++) CHECK(list.insert(x.tiles.tile(i)).second);
            for (int k = 0; k < 20; k++) {
                const int row = p0 + up_to(p1 - p0), j = row < 0 ? 0 : up_to(row);
                const bool sees = j <= row && (a.window <= 0 || row - j < a.window || j < a.sinks);
                if (sees) CHECK(list.count(j / KT));
            }
        }
        // a block's pieces are its share, apart from ends that were moved and what a tile costs besides
        CHECK(most <= (before.back() + blocks - 1) / blocks + LEAST + 2 * SNAP + EXTRA);
    }
}
int main() {
    check<64, 16, 1, 1, 2>(148, 1);       // tiles of 16 rows, one to three blocks a multiprocessor
    check<64, 16, 1, 1, 2>(444, 2);
    check<128, 256, 3, 5, 1>(148, 3);     // tcgen05, heads of up to 128 and of 256
    check<128, 128, 4, 6, 1>(148, 4);
    check<128, 128, 0, 1, 1>(7, 5);
    check<64, 16, 2, 6, 4>(33, 6);
    printf("done\n");
    return bad;
}
"""


def test_the_kernels_own_shares_cover_every_tile_once(tmp_path):
    src, exe = tmp_path / "shares.cu", str(tmp_path / "shares")
    src.write_text(SHARES)
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I",
                    os.path.join(ROOT, "biv_b200", "csrc"), "-o", exe, str(src)], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr
