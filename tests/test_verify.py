"""Drafted tokens against the target's probabilities (``biv_b200.verify``): whole numbers, equal to the definition in 64 bits.

Where a drawn weight lies so near a border of the running sum that the order of f64 sums could decide (2^-40 of the sum: a sum of
2^18 values in any order is within 2^18 * 2^-53 of it), the neighbour is right, too; the inputs of these tests, made from their
seeds, have no such row apart from those that say so."""
import importlib.util
import math

import pytest
import torch

from biv_b200 import capi

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(lengths, vocab, dtype, drafted, seed, accept=0.6, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    t = sum(lengths)
    logits = 2 * torch.randn((t, vocab), generator=g)
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits + torch.randn((t, vocab), generator=g), -1).to(dtype) if drafted else None
    first = [0]
    for n in lengths:
        first.append(first[-1] + n)
    tokens = torch.randint(0, vocab, (t,), generator=g)
    likely = p.float().argmax(-1)                            # drafts that pass often: the target's best token
    use = torch.rand((t,), generator=g) < accept
    tokens[1:] = torch.where(use[:-1], likely[:-1], tokens[1:])
    x = dict(p=p, q=q, tokens=tokens.to(torch.int32), uniform=torch.rand((t,), generator=g), sample=torch.rand((len(lengths),), generator=g),
             first=torch.tensor(first, dtype=torch.int32), length=torch.tensor([40 + 7 * i + n for i, n in enumerate(lengths)], dtype=torch.int32))
    if drafted is False:
        x["uniform"] *= 0.02
    return {k: v.to(device) if v is not None else None for k, v in x.items()}


def reference(x):
    p, tokens, first = x["p"].cpu(), x["tokens"].tolist(), x["first"].tolist()
    q = None if x["q"] is None else x["q"].cpu()
    vocab = p.shape[1]
    uniform, sample = x["uniform"].double().cpu(), x["sample"].double().cpu()
    accepted, token, kept = [], [], []
    for b in range(len(first) - 1):
        n = first[b + 1] - first[b]
        k = 0
        while k < n - 1:
            r, d = first[b] + k, tokens[first[b] + k + 1]
            if not 0 <= d < vocab or not uniform[r] * (q[r, d].double() if q is not None else 1.0) < p[r, d].double():
                break
            k += 1
        accepted.append(k)
        kept.append(int(x["length"][b]) - max(n - 1 - k, 0) if x["length"] is not None else 0)
        if not n:
            token.append(-1)
            continue
        f = first[b] + k
        w = p[f].float().clone()
        whole = w.nan_to_num(nan=0.0, posinf=math.inf).clamp(min=0)
        if k < n - 1:
            d = tokens[f + 1]
            if q is not None:
                w = w - q[f].float()
            elif 0 <= d < vocab:
                w[d] = 0
        w = w.nan_to_num(nan=0.0, posinf=math.inf).clamp(min=0).double()
        if not w.sum() > 0:
            w = whole.double()
        if not w.sum() > 0:
            token.append(-1)
            continue
        over = torch.cumsum(w, 0) > sample[b] * w.sum()
        token.append(int(torch.nonzero(over & (w > 0))[0]) if (over & (w > 0)).any() else int(torch.nonzero(w > 0)[-1]))
    return accepted, token, kept


def run(x):
    from biv_b200.verify import verify
    return verify(x["p"], x["tokens"], x["uniform"], x["sample"], x["first"], q=x["q"], length=x["length"])


def check(x):
    got, (accepted, token, kept) = run(x), reference(x)
    assert got.accepted.tolist() == accepted
    assert got.token.tolist() == token
    assert got.kept is None if x["length"] is None else got.kept.tolist() == kept
    return accepted


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4096, 32003, 100003])
def test_vocabularies(dtype, drafted, vocab):
    accepted = check(make([5, 1, 3, 0, 2, 5, 4], vocab, dtype, drafted, seed=vocab))
    if vocab > 1000 and dtype == torch.float32:
        assert any(accepted) and not all(a == n - 1 for a, n in zip(accepted, [5, 1, 3, 0, 2, 5, 4]))


@gpu
@pytest.mark.parametrize("seqs", [1, 40, 100, 300])
@pytest.mark.parametrize("drafted", [True, False])
def test_numbers_of_requests(seqs, drafted):
    check(make([1 + i % 5 for i in range(seqs)], 1031, torch.float32, drafted, seed=seqs))


@gpu
@pytest.mark.parametrize("seqs,vocab", [(600, 700), (3, 1 << 24), (700, 200001)])
def test_the_ends_of_the_sizes(seqs, vocab):
    """More requests than run at once, the widest vocabulary, and requests that share a few rows of a wide one."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n = min(seqs, 8)
    p = torch.rand((n, vocab), generator=g, device="cuda").half()
    first = torch.tensor([i * n // seqs for i in range(seqs + 1)], dtype=torch.int32, device="cuda")      # none or one row each
    ints = torch.zeros(n, dtype=torch.int32, device="cuda")
    x = dict(p=p, q=None, tokens=ints, uniform=torch.rand(n, generator=g, device="cuda"), sample=torch.rand(seqs, generator=g, device="cuda"),
             first=first, length=None)
    check(x)


@gpu
def test_many_drafts():
    check(make([700, 1, 3], 50, torch.float32, True, seed=4, accept=0.999))
    x = make([700], 50, torch.float32, False, seed=5, accept=1.0)
    x["uniform"].zero_()
    assert check(x) == [699]


@gpu
def test_strides_and_no_length():
    x = make([4, 3], 1003, torch.bfloat16, True, seed=1)
    wide = torch.zeros((7, 2, 1011), dtype=torch.bfloat16, device="cuda")
    wide[:, 0, 3:1006], wide[:, 1, 5:1008] = x["p"], x["q"]
    x["p"], x["q"], x["length"] = wide[:, 0, 3:1006], wide[:, 1, 5:1008], None       # p and q not alike within 16 bytes
    check(x)
    x["q"] = wide[:, 1, 3:1006]
    check(x)


@gpu
@pytest.mark.parametrize("vocab", [700, 9001])
def test_borders(vocab):
    """Weights of whole numbers: sums are exact, and the sample lies on their borders."""
    x = make([1] * 24, vocab, torch.float32, True, seed=3)
    g = torch.Generator().manual_seed(1)
    w = torch.randint(0, 3, (24, vocab), generator=g).float()
    w[:, 0] += 1
    total = w.sum(1)
    w[:, -1] += 2 ** 16 - total                              # a sum of 2^16: sample * sum is exact
    x["p"] = w.cuda()
    upto = torch.cumsum(w.double(), 1)
    x["sample"] = (upto[torch.arange(24), torch.linspace(0, vocab - 2, 24).long()] / 2 ** 16).float().cuda()
    check(x)
    x["sample"] = torch.zeros(24, device="cuda")
    check(x)
    x["sample"] = torch.full((24,), 1 - 2.0 ** -24, device="cuda")
    check(x)
    x["sample"] = torch.ones(24, device="cuda")              # past the range: the last token of positive weight
    x["p"][:, vocab // 2:] = 0
    check(x)


@gpu
def test_rows_without_weight_and_drafts_outside():
    x = make([3, 3, 3, 2, 2, 1], 517, torch.float32, True, seed=9)
    x["q"][:6] = x["p"][:6]                                  # nothing is left of p - q: p itself
    x["uniform"][0] = 1.0                                    # rejected all the same (outside its range)
    x["p"][9:11] = 0.0                                       # nothing positive at all
    x["p"][13] = math.nan
    x["tokens"][4], x["tokens"][7] = -1, 517
    accepted = check(x)
    assert accepted[0] == 0 and accepted[1] == 0 and accepted[2] == 0
    assert run(x).token.tolist()[3] == -1 and run(x).token.tolist()[5] == -1
    x["q"] = None
    check(x)


@gpu
def test_not_a_number_among_the_weights():
    x = make([2, 1, 2], 1500, torch.float32, True, seed=2)
    x["p"][:, ::7] = math.nan
    x["q"][:, ::11] = math.nan
    check(x)


@gpu
def test_distribution():
    """Drafts drawn from q, verified against p: the first tokens that come out are distributed as p."""
    g = torch.Generator().manual_seed(0)
    n, vocab = 40000, 8
    p, q = torch.softmax(torch.randn((2, vocab), generator=g), -1)
    draft = torch.multinomial(q, n, replacement=True, generator=g)
    first = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32)
    tokens = torch.zeros(2 * n, dtype=torch.int32)
    tokens[1::2] = draft.to(torch.int32)
    from biv_b200.verify import verify
    r = verify(p.repeat(2 * n, 1).cuda(), tokens.cuda(), torch.rand(2 * n, generator=g).cuda(), torch.rand(n, generator=g).cuda(), first.cuda(),
               q=q.repeat(2 * n, 1).cuda())
    out = torch.where(r.accepted.cpu() > 0, draft, r.token.cpu().long())
    share = torch.bincount(out, minlength=vocab).double() / n
    # five standard deviations of a share
    assert ((share - p.double()).abs() <= 5 * torch.sqrt(p.double() * (1 - p.double()) / n)).all()


@gpu
def test_captured_and_replayed():
    x, y = make([5] * 20, 5003, torch.bfloat16, True, seed=1), make([5] * 20, 5003, torch.bfloat16, True, seed=2)
    run(x)
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        got = run(x)
    want = reference(y)
    for k in ("p", "q", "tokens", "uniform", "sample", "length"):
        x[k].copy_(y[k])
    g.replay()
    torch.cuda.synchronize()
    assert (got.accepted.tolist(), got.token.tolist(), got.kept.tolist()) == want


@gpu
def test_refusals():
    from biv_b200.verify import verify
    x = make([2, 2], 100, torch.float32, True, seed=1)
    good = dict(p=x["p"], tokens=x["tokens"], uniform=x["uniform"], sample=x["sample"], first=x["first"], q=x["q"], length=x["length"])
    verify(**good)
    for bad in (dict(p=x["p"].double()), dict(p=x["p"].cpu()), dict(p=x["p"].T), dict(p=x["p"][:, :0]), dict(q=x["q"].half()), dict(q=x["q"][:3]),
                dict(tokens=x["tokens"].long()), dict(tokens=x["tokens"][:3]), dict(uniform=x["uniform"].double()), dict(sample=x["sample"].cpu()),
                dict(first=x["first"][:2]), dict(length=x["length"][:1])):
        with pytest.raises(ValueError):
            verify(**{**good, **bad})
    none = verify(x["p"], x["tokens"], x["uniform"], x["sample"][:0], x["first"][:1])
    assert none.accepted.numel() == 0 and none.kept is None


def test_arguments_are_checked_without_a_device():
    import ctypes as C
    L = capi.lib()
    assert L.bivmoe_verify(None, None) == capi.ERR_ARGUMENT
    good = dict(p=4096, p_stride=100, ggml_type=0, vocab=100, tokens=4096, first=4096, uniform=4096, sample=4096, accepted=4096, token=4096,
                n_seq=1, n_tokens=1)
    for change, code in ((dict(ggml_type=8), capi.ERR_UNSUPPORTED), (dict(vocab=0), capi.ERR_ARGUMENT), (dict(vocab=1 << 25), capi.ERR_ARGUMENT),
                         (dict(n_seq=-1), capi.ERR_ARGUMENT), (dict(p=0), capi.ERR_ARGUMENT), (dict(token=0), capi.ERR_ARGUMENT),
                         (dict(length=4096), capi.ERR_ARGUMENT), (dict(p=4098), capi.ERR_ARGUMENT), (dict(first=4097), capi.ERR_ARGUMENT)):
        a = capi.VerifyArgs(**{**good, **change})
        assert L.bivmoe_verify(C.byref(a), None) == code, change
    a = capi.VerifyArgs(**{**good, "n_seq": 0})
    assert L.bivmoe_verify(C.byref(a), None) == capi.OK


def test_the_calls_module_is_built():
    assert importlib.util.find_spec("biv_b200._step_calls") is not None


def decided(p, q, tokens, uniform, sample, vocab):
    """One request's (accepted, token), value by value as the header has it: comparisons that NaN never passes, weights of NaN zero."""
    k, n = 0, len(tokens)
    while k < n - 1:
        d = tokens[k + 1]
        if not (0 <= d < vocab and (uniform[k] * q[k][d] if q else uniform[k]) < p[k][d]):
            break
        k += 1
    for residual in ([True, False] if k < n - 1 else [False]):
        w = []
        for t in range(vocab):
            x = p[k][t]
            if residual:
                x = x - q[k][t] if q else (0.0 if t == tokens[k + 1] else x)
            w.append(x if x > 0 else 0.0)                    # (NaN is not)
        if sum(w) > 0:
            break
    else:
        return k, -1
    upto, border = 0.0, sample * sum(w)
    for t, x in enumerate(w):
        upto += x
        if upto > border:
            return k, t
    return k, max(t for t, x in enumerate(w) if x > 0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 1503, 9001])
@pytest.mark.parametrize("drafted", [True, False])
def test_what_is_not_finite_as_the_header_has_it(vocab, dtype, drafted):
    """Weights of whole numbers, whose sums are exact, with NaN and infinities at the drafts and among the weights; both ways that p and q
    may lie to one another."""
    g = torch.Generator().manual_seed(vocab)
    bad = [math.nan, math.inf, -math.inf]
    n, rows, drafts = 48, 3, 5
    p, q = (torch.randint(0, 4, (n * rows, vocab), generator=g).double() for _ in range(2))
    tokens = torch.randint(0, drafts, (n * rows,), generator=g) * (vocab // drafts)
    for r in range(n * rows):
        d = int(tokens[min(r + 1, n * rows - 1)])
        if r % 4 == 0:
            p[r, d] = bad[r // 4 % 3]
        if r % 4 == 1:
            q[r, d] = bad[r // 4 % 3]
        if r % 3 == 0:                                       # NaN in many places, of p, of q, of both
            p[r, r % 7::7] = math.nan
            q[r, r % 5::5] = math.nan
        if r % 5 == 0:                                       # some infinite weights, infinity less infinity
            p[r, vocab // 3:vocab // 2:3] = math.inf
            q[r, vocab // 3:vocab // 2:6] = math.inf
    uniform = torch.randint(0, 3, (n * rows,), generator=g).float() / 2
    sample = torch.randint(0, 16, (n,), generator=g).float() / 16
    want = []
    for b in range(n):
        at = slice(b * rows, (b + 1) * rows)
        want.append(decided(p[at].tolist(), q[at].tolist() if drafted else None, tokens[at].tolist(), uniform[at].tolist(), float(sample[b]), vocab))
    assert len({k for k, _ in want}) == 3                    # (drafts pass and fail)
    ints = dict(dtype=torch.int32, device="cuda")
    for apart in (8, 9):                                     # q and p alike within 16 bytes, and not
        both = torch.zeros((n * rows, 2, 8 + vocab + apart), dtype=dtype, device="cuda")
        rows_p, rows_q = both[:, 0, 8:8 + vocab], both[:, 1, apart:apart + vocab]
        rows_p.copy_(p)
        rows_q.copy_(q)
        x = dict(p=rows_p, q=rows_q if drafted else None, tokens=tokens.to(**ints), uniform=uniform.cuda(), sample=sample.cuda(),
                 first=torch.arange(0, n * rows + 1, rows, **ints), length=None)
        got = run(x)
        assert list(zip(got.accepted.tolist(), got.token.tolist())) == want


def test_the_definition_of_these_tests():
    inf, nan = math.inf, math.nan
    p, q = [[1.0, 2.0, 1.0], [nan, 3.0, 1.0]], [[1.0, 4.0, 0.0], [1.0, nan, 1.0]]
    assert decided(p, q, [0, 1], [0.25, 0.0], 0.0, 3) == (1, 1)               # accepted; then p's own, without its NaN
    assert decided(p, q, [0, 1], [0.5, 0.0], 0.9, 3) == (0, 2)                # 2 < 2 is not: what p has over q
    assert decided([[1.0, 2.0], [0.0, 0.0]], [[1.0, nan], [0.0, 0.0]], [0, 1], [0.0, 0.0], 0.5, 2) == (0, 1)   # 0 * NaN: not accepted; p itself
    assert decided([[inf, 1.0, inf, 1.0]], None, [0], [0.0], 0.0, 4) == (0, 3)


@gpu
def test_offsets_that_pass_the_rows_or_decrease():
    """Past n_tokens they count as n_tokens, decreasing ones as no rows, negative ones as zero."""
    x = make([4, 0, 5, 3], 1003, torch.float32, True, seed=6)
    want = run(x)
    x["first"] = torch.tensor([-9, 4, 4, 9, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got = run(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x["first"] = torch.tensor([9, 4, 12, -(2 ** 31), 3], dtype=torch.int32, device="cuda")       # rows 4 to 11, and 0 to 2
    got, length = run(x), x["length"]
    x["first"], x["length"], x["sample"] = torch.tensor([4, 12], dtype=torch.int32, device="cuda"), length[1:2], x["sample"][[1, 3]]
    accepted, token, kept = reference({**x, "sample": x["sample"][:1]})
    more = reference({**x, "first": torch.tensor([0, 3], dtype=torch.int32), "length": length[3:], "sample": x["sample"][1:]})
    assert got.accepted.tolist() == [0, accepted[0], 0, more[0][0]]
    assert got.token.tolist() == [-1, token[0], -1, more[1][0]]
    assert got.kept.tolist() == [int(length[0]), kept[0], int(length[2]), more[2][0]]


@gpu
def test_rows_more_than_32_bits_apart():
    x = make([5] * 28, 1003, torch.bfloat16, True, seed=8)
    apart = 2 ** 24 + 2 ** 10 + 1                            # (a row of p now and then begins on 16 bytes)
    room = torch.empty(140 * apart, dtype=torch.bfloat16, device="cuda")
    for i, name in enumerate(("p", "q")):
        view = room[4096 * i:].as_strided((140, 1003), (apart, 1))
        view.copy_(x[name])
        x[name] = view
    check(x)
