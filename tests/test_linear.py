"""Linear attention with a decay for each head (``biv_b200.linear``) against the recurrence in 64 bits, token by token.

Tolerances.  Without the delta rule every term of the state and of an output is a product of inputs and decays, so the same
recurrence on absolute values, A, bounds what any order of f32 sums can lose: with n tokens each element passes at most 2 n + 8
roundings of 2^-24, an output dim_k + 8 more, and where the kernel for prompts works (bf16) 2^-8 (half a step) for the weights of a
chunk's tokens among one another and for the state on its way to q, and 2^-15 for what is in two bf16 terms (each cut off, not rounded).  With the delta rule and keys of length one a step is a contraction, so that local errors add
up: a step's are at most (dim_k / 8 + 12) 2^-24 of the state's and the value's length.  (The kernel for prompts of that kind has bf16
terms of the state and of T, off by 2^-18, and an f32 inverse, whose errors its chunk's tolerance, 64 times as many steps of 2^-24, holds
by far; its outputs meet u and the state rounded to bf16, half a step each: 2^-8 of the recurrence on the absolute values of u.)  The output's own rounding is half a step
of its type: finfo.eps / 2 of its value, and below the type's smallest normal number, finfo.tiny, where the steps no longer shrink
with the value, half of tiny * eps (f16: 2^-14 * 2^-10 / 2)."""
import math

import pytest
import torch

import importlib.util

from biv_b200 import capi

gpu = pytest.mark.gpu
HAVE = importlib.util.find_spec("biv_b200._step_calls") is not None
EPS = 2.0 ** -24


def make(lengths, h, hk, dk, dv, dtype, delta, seed=0, device="cuda", rate=None):
    g = torch.Generator().manual_seed(seed)
    t = sum(lengths)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x = dict(q=unit(rand(t, hk, dk)), k=unit(rand(t, hk, dk)), v=rand(t, h, dv))
    x = {n: v.to(dtype).to(device) for n, v in x.items()}
    r = torch.exp(torch.linspace(math.log(1e-3), math.log(8.0), h, dtype=torch.float64)) if rate is None else torch.full((h,), rate, dtype=torch.float64)
    x["decay"] = (-r * torch.rand((t, h), generator=g, dtype=torch.float64)).float().to(device)
    x["beta"] = torch.sigmoid(rand(t, h)).float().to(device) if delta else None
    x["states"] = (0.5 * rand(len(lengths) + 3, h, dv, dk)).float().to(device)
    x["slots"] = torch.randperm(len(lengths) + 3, generator=g)[:len(lengths)].to(torch.int32).to(device)
    first = [0]
    for n in lengths:
        first.append(first[-1] + n)
    x["first"] = torch.tensor(first, dtype=torch.int32, device=device)
    return x


def reference(x, past=None, keep=None, scale=None, absolute=False):
    """(out, states, lengths) in f64; `absolute`: the recurrence on absolute values, with the delta rule on those of what each token
    adds, u."""
    if absolute and x["beta"] is not None:
        x = {**x, "v": additions(x, past), "beta": None}
    f = (lambda t: t.double().cpu().abs()) if absolute else (lambda t: t.double().cpu())
    q, k, v, states = f(x["q"]), f(x["k"]), f(x["v"]), f(x["states"])
    decay = x["decay"].double().cpu().clamp(max=0)
    beta = None if x["beta"] is None else x["beta"].double().cpu()
    h, dk = v.shape[1], k.shape[2]
    rep = h // k.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    scale = dk ** -0.5 if scale is None else scale
    out = torch.full(v.shape, float("nan"), dtype=torch.float64)
    first, slots = x["first"].tolist(), x["slots"].tolist()
    size = torch.zeros(len(slots), h, dtype=torch.float64)          # the longest a state and a value got
    for b, slot in enumerate(slots):
        n = first[b + 1] - first[b]
        has = 0 <= slot < states.shape[0] and slot not in slots[:b]
        s = states[slot].clone() if has and (past is None or past[b]) else torch.zeros((h, v.shape[2], dk), dtype=torch.float64)
        kept = n if keep is None else min(max(keep[b], 0), n)
        for i in range(n):
            r = first[b] + i
            s = s * torch.exp(decay[r])[:, None, None]
            vt = v[r]
            if beta is not None:
                vt = beta[r][:, None] * (vt - torch.einsum("hvk,hk->hv", s, k[r]))
            s = s + vt[:, :, None] * k[r][:, None, :]
            out[r] = abs(scale) * torch.einsum("hvk,hk->hv", s, q[r]) if absolute else scale * torch.einsum("hvk,hk->hv", s, q[r])
            size[b] = torch.maximum(size[b], s.flatten(1).norm(dim=1) + v[r].norm(dim=1))
            if i + 1 == kept and has:
                states[slot] = s
    return out, states, size


def additions(x, past=None):
    """What each token adds along its key with the delta rule: beta (v - exp(decay) S k), in f64."""
    k, v, states = x["k"].double().cpu(), x["v"].double().cpu(), x["states"].double().cpu()
    decay, beta = x["decay"].double().cpu().clamp(max=0), x["beta"].double().cpu()
    k = k.repeat_interleave(v.shape[1] // k.shape[1], 1)
    u, first, slots = torch.zeros_like(v), x["first"].tolist(), x["slots"].tolist()
    for b, slot in enumerate(slots):
        has = 0 <= slot < states.shape[0] and slot not in slots[:b] and (past is None or past[b])
        s = states[slot].clone() if has else torch.zeros(v.shape[1:] + k.shape[2:], dtype=torch.float64)
        for r in range(first[b], first[b + 1]):
            s = s * torch.exp(decay[r])[:, None, None]
            u[r] = beta[r][:, None] * (v[r] - torch.einsum("hvk,hk->hv", s, k[r]))
            s = s + u[r][:, :, None] * k[r][:, None, :]
    return u


def layer(x, dtype, h=None):
    from biv_b200.linear import LinearAttention
    return LinearAttention(x["v"].shape[1], x["k"].shape[1], x["k"].shape[2], x["v"].shape[2], max_seqs=max(1, x["slots"].numel()), dtype=dtype)


def check(x, out, states, dtype, past=None, keep=None, scale=None, prompt=False):
    want, want_states, size = reference(x, past, keep, scale)
    first = x["first"].tolist()
    n = max([b - a for a, b in zip(first, first[1:])] + [1])
    dk, h = x["k"].shape[2], x["v"].shape[1]
    rows = torch.zeros(x["v"].shape[0], dtype=torch.bool)
    rows[:first[-1]] = True
    got, got_states = out.double().cpu(), states.double().cpu()
    half = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).tiny * half
    if x["beta"] is None:
        a_out, a_states, _ = reference(x, past, keep, scale, absolute=True)
        tol_s = (2 * n + 8) * EPS * a_states
        tol_o = ((2 * n + dk + 16) * EPS + (2.0 ** -8 + 2.0 ** -15 if prompt else 0.0)) * a_out + 1.01 * half * want.abs() + 1.01 * least
        assert ((got_states - want_states).abs() <= tol_s + 1e-30).all(), float(((got_states - want_states).abs() / (tol_s + 1e-30)).max())
    else:
        per = (dk / 8 + 12) * EPS * n
        err = (got_states - want_states).flatten(2).norm(dim=2)
        for b, slot in enumerate(x["slots"].tolist()):
            if 0 <= slot < err.shape[0]:
                assert (err[slot] <= per * size[b] + 1e-30).all(), float((err[slot] / (per * size[b] + 1e-30)).max())
                err[slot] = 0
        assert (err == 0).all()
        long = torch.zeros_like(want)
        for b in range(len(first) - 1):
            long[first[b]:first[b + 1]] = size[b][None, :, None]
        qn = x["q"].double().cpu().norm(dim=2).repeat_interleave(h // x["q"].shape[1], 1)[..., None]
        tol_o = abs(scale or dk ** -0.5) * (per + (dk / 8 + 12) * EPS) * long * qn + 1.01 * half * want.abs() + 1.01 * least
        if prompt:
            tol_o += (2.0 ** -8 + 2.0 ** -15) * reference(x, past, keep, scale, absolute=True)[0]
    bad = (got - want).abs()[rows] > (tol_o[rows] + 1e-30)
    assert not bad.any(), float(((got - want).abs()[rows] / (tol_o[rows] + 1e-30)).max())


SHAPES = [
    # lengths, heads, heads of q and k, dim_k, dim_v
    ([1], 1, 1, 64, 64),
    ([1, 1, 1, 1, 1], 4, 2, 128, 128),
    ([3, 0, 9, 1, 8, 7], 6, 2, 128, 64),
    ([5, 17], 3, 3, 64, 128),
    ([2, 31], 2, 1, 256, 256),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_steps(shape, delta, dtype):
    lengths, h, hk, dk, dv = shape
    x = make(lengths, h, hk, dk, dv, dtype, delta, seed=len(lengths))
    lay = layer(x, dtype)
    states = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=max(lengths))
    lay.status()
    check(x, out, states, dtype)


@gpu
@pytest.mark.parametrize("rows", [64, 700, 2500])      # of all states' 148 x 64 and x 256: each number of rows to a thread
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_steps_of_many_heads(rows, delta, dim):
    h = 16
    b = max(1, rows * 64 // (h * dim))
    x = make([1 + i % 2 for i in range(b)], h, 4, dim, dim, torch.bfloat16, delta, seed=rows)
    lay = layer(x, torch.bfloat16)
    states = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=2)
    check(x, out, states, torch.bfloat16)


PROMPTS = [
    # lengths, heads, heads of q and k
    ([64], 1, 1),
    ([17, 1, 63, 65, 0, 128, 130], 4, 2),
    ([200, 3, 500], 6, 6),
    ([700], 2, 1),            # several blocks to a request and head: two,
    ([2100, 40], 3, 1),       # four
    ([4300], 2, 2),           # and eight
    ([1100] * 5, 16, 8),
]


@gpu
@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("shape", PROMPTS)
def test_prompts(shape, delta, fresh):
    lengths, h, hk = shape
    x = make(lengths, h, hk, 128, 128, torch.bfloat16, delta, seed=sum(lengths))
    lay = layer(x, torch.bfloat16)
    states = x["states"].clone()
    past = [0 if fresh else 5] * len(lengths)
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"],
                     past=torch.tensor(past, dtype=torch.int32, device="cuda"), max_new=max(lengths))
    lay.status()
    check(x, out, states, torch.bfloat16, past=past, prompt=True)
    again = x["states"].clone()
    assert torch.equal(out, lay.attend(x["q"], x["k"], x["v"], x["decay"], again, x["slots"], x["first"], beta=x["beta"],
                                       past=torch.tensor(past, dtype=torch.int32, device="cuda"), max_new=max(lengths)))
    assert torch.equal(again, states)


@gpu
@pytest.mark.parametrize("delta", [False, True])
def test_prompts_in_chunks_and_at_once(delta):
    """A prompt of 300 tokens as 170, 1 and 129 of them, within the tolerance of one at once."""
    x = make([300], 3, 3, 128, 128, torch.bfloat16, delta, seed=8)
    lay = layer(x, torch.bfloat16)
    states = x["states"].clone()
    out = torch.empty_like(x["v"])
    at = 0
    for n in (170, 1, 129):
        rows = slice(at, at + n)
        part = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        lay.attend(x["q"][rows], x["k"][rows], x["v"][rows], x["decay"][rows], states, x["slots"], part,
                   beta=x["beta"][rows] if delta else None, max_new=n, out=out[rows])
        at += n
    check(x, out, states, torch.bfloat16, prompt=True)


@gpu
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("max_new", [0, 9])
def test_past_keep_and_slots_that_are_not_there(delta, max_new):
    x = make([4, 9, 3, 0, 2, 5, 1], 4, 2, 128, 128, torch.bfloat16, delta)
    slots = x["slots"].tolist()
    slots[2], slots[4], slots[5] = -1, 10 ** 6, slots[0]            # none, past the states, taken
    x["slots"] = torch.tensor(slots, dtype=torch.int32, device="cuda")
    past, keep = [0, 7, 5, 1, 3, 2, 4], [4, 5, 2, 1, 2, 5, 0]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lay = layer(x, torch.bfloat16)
    states = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], past=ints(past), keep=ints(keep),
                     max_new=max_new)
    check(x, out, states, torch.bfloat16, past, keep)
    untouched = [s for s in range(states.shape[0]) if s not in (slots[0], slots[1])]
    assert torch.equal(states[untouched], x["states"][untouched])
    # the states alone
    again = x["states"].clone()
    lay.advance(x["k"], x["v"], x["decay"], again, x["slots"], x["first"], beta=x["beta"], past=ints(past), keep=ints(keep), max_new=max_new)
    assert torch.equal(again, states)


@gpu
@pytest.mark.parametrize("dtype,max_new", [(torch.bfloat16, 5), (torch.float32, 5)])
def test_drafts_taken_back(dtype, max_new):
    """Five tokens with keep 0, then the two that were accepted: the state of two tokens at once."""
    x = make([5, 5, 5], 4, 4, 128, 128, dtype, True)
    lay = layer(x, dtype)
    states = x["states"].clone()
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], keep=none, max_new=max_new)
    assert torch.equal(states, x["states"])
    kept = torch.tensor([2, 1, 5], dtype=torch.int32, device="cuda")
    lay.advance(x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], keep=kept, max_new=max_new)
    check(x, out, states, dtype, keep=[2, 1, 5])


@gpu
def test_strides_scale_and_rows_behind_the_last():
    h, hk, d, n = 4, 2, 128, 7
    x = make([3, n - 3], h, hk, d, d, torch.bfloat16, False)
    x = dict(x)
    rows = torch.zeros((n + 4, 3, 2 * hk + h + 1, d), dtype=torch.bfloat16, device="cuda")[:, 1]      # a gap between rows
    views = dict(q=rows[:, :hk], k=rows[:, hk:2 * hk], v=rows[:, 2 * hk:2 * hk + h])
    for name, view in views.items():
        view[:n] = x[name]
        view[n:] = float("nan")
    big = torch.zeros((x["states"].shape[0], h + 1, d, d), device="cuda")
    big[:, :h] = x["states"]
    decay = torch.full((n + 4, 2 * h), float("nan"), device="cuda")
    decay[:n, :h] = x["decay"]
    out = torch.full((n + 4, h, d), 3.0, dtype=torch.bfloat16, device="cuda")
    lay = layer(x, torch.bfloat16)
    r = lay.attend(views["q"], views["k"], views["v"], decay[:, :h], big[:, :h], x["slots"], x["first"], scale=-0.3, max_new=4, out=out)
    assert r is out and (out[n:] == 3.0).all() and (big[:, h] == 0).all()
    check(x, out[:n], big[:, :h], torch.bfloat16, scale=-0.3)


@gpu
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("max_new", [0, 4])
def test_decays_at_the_ends_of_their_range(max_new, delta):
    x = make([6, 70], 6, 6, 128, 128, torch.bfloat16, delta)
    x["decay"][:, 1] = 0.0
    x["decay"][::3, 2] = -math.inf
    x["decay"][::4, 3] = torch.finfo(torch.float32).min
    x["decay"][::2, 4] = 5.0                                  # counts as zero
    x["decay"][:, 5] = -90.0
    lay = layer(x, torch.bfloat16)
    states = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=max_new)
    lay.status()
    check(x, out, states, torch.bfloat16, prompt=True)


@gpu
@pytest.mark.parametrize("name", ["q", "k", "v", "decay", "beta"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("max_new", [200, 1])          # (wrong on purpose: it decides the kernel alone)
def test_what_is_not_finite_reaches_no_earlier_token_and_no_other_head(name, value, delta, max_new):
    if name == "beta" and not delta:
        pytest.skip("no beta")
    lengths = [70, 200]
    x = make(lengths, 3, 3, 128, 128, torch.bfloat16, delta)
    lay = layer(x, torch.bfloat16)
    call = lambda y, s: lay.attend(y["q"], y["k"], y["v"], y["decay"], s, x["slots"], x["first"], beta=y["beta"], max_new=max_new)  # noqa: E731
    s0 = x["states"].clone()
    clean = call(x, s0)
    y = {k: v.clone() if v is not None else None for k, v in x.items()}
    at, place = 70 + 83, 5
    if name == "decay":
        y["decay"][at, 1] = math.nan
    elif name == "beta":
        y["beta"][at, 1] = value
    else:
        y[name][at, 1, place] = value
    s1 = x["states"].clone()
    got = call(y, s1)
    lay.status()
    assert torch.equal(got[:at], clean[:at])
    assert torch.equal(got[:, [0, 2]], clean[:, [0, 2]])
    slot = int(x["slots"][1])
    others = [i for i in range(s0.shape[0]) if i != slot]
    assert torch.equal(s1[others], s0[others]) and torch.equal(s1[slot][[0, 2]], s0[slot][[0, 2]])
    if name == "q":
        assert not got[at, 1].isfinite().any() and torch.equal(got[at + 1:], clean[at + 1:]) and torch.equal(s0, s1)
    elif name == "v":
        assert not got[at:, 1, place].isfinite().any() and not s1[slot, 1, place].isfinite().any()
        rest = [i for i in range(128) if i != place]
        assert torch.equal(got[:, 1, rest], clean[:, 1, rest]) and torch.equal(s1[slot, 1, rest], s0[slot, 1, rest])
    else:
        assert not got[at, 1].isfinite().any()


@gpu
def test_captured_and_replayed_and_other_streams():
    x = make([1] * 6, 4, 2, 128, 128, torch.bfloat16, True)
    lay = layer(x, torch.bfloat16)
    args = lambda s: (x["q"], x["k"], x["v"], x["decay"], s, x["slots"], x["first"])  # noqa: E731
    want = x["states"].clone()
    outs = [lay.attend(*args(want), beta=x["beta"], max_new=1) for _ in range(3)]
    states = x["states"].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = lay.attend(*args(states), beta=x["beta"], max_new=1)
        got = []
        for _ in range(3):
            g.replay()
            got.append(out.clone())
    side.synchronize()
    assert torch.equal(states, want) and all(torch.equal(a, b) for a, b in zip(got, outs))


@gpu
def test_nothing_to_do():
    x = make([0, 0], 2, 2, 64, 64, torch.float32, False)
    lay = layer(x, torch.float32)
    s = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], s, x["slots"], x["first"])
    assert out.shape == (0, 2, 64) and torch.equal(s, x["states"])
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    lay.attend(x["q"], x["k"], x["v"], x["decay"], s, none, torch.zeros(1, dtype=torch.int32, device="cuda"))


@gpu
def test_refusals():
    from biv_b200.linear import LinearAttention
    for bad in (dict(dim_k=96), dict(dim_v=32), dict(n_head=3), dict(max_seqs=0), dict(max_seqs=4096), dict(n_head=0)):
        with pytest.raises(capi.BivMoeError):
            LinearAttention(**{**dict(n_head=4, n_head_qk=2, dim_k=64, dim_v=64, max_seqs=2), **bad})
    with pytest.raises(ValueError):
        LinearAttention(4, 2, 64, 64, 2, dtype=torch.float64)
    x = make([2, 2], 4, 2, 64, 64, torch.bfloat16, True)
    lay = layer(x, torch.bfloat16)
    good = {k: x[k] for k in ("q", "k", "v", "decay", "states", "slots", "first", "beta")}
    lay.attend(**good)
    wide = torch.zeros((4, 2, 64 + 4), dtype=torch.bfloat16, device="cuda")
    for change in (dict(q=x["q"].float()), dict(k=x["k"].cpu()), dict(v=x["v"][:, :2]), dict(k=x["k"][:3]), dict(decay=x["decay"].double()),
                   dict(decay=x["decay"].T.contiguous().T), dict(states=x["states"].half()), dict(states=x["states"].transpose(2, 3)),
                   dict(slots=x["slots"].long()), dict(first=x["first"][:2]), dict(beta=x["beta"][:, :3]), dict(max_new=2 ** 40),
                   dict(past=x["slots"][:1]), dict(keep=x["slots"].float())):
        with pytest.raises(ValueError):
            lay.attend(**{**good, **change})
    for change in (dict(q=wide[:, :, :64]), dict(k=wide[:, :, 4:]), dict(max_new=-1)):   # a stride, a start, a number
        with pytest.raises(capi.BivMoeError):
            lay.attend(**{**good, **change})
    more = make([1] * 3, 4, 2, 64, 64, torch.bfloat16, False)
    with pytest.raises(capi.BivMoeError):
        lay.attend(more["q"], more["k"], more["v"], more["decay"], more["states"], more["slots"], more["first"])
    lay.close()
    with pytest.raises(ValueError):
        lay.attend(**good)


def test_reference_holds_the_formula():
    """The recurrence of the tests against sums written out: no delta rule, one head."""
    x = make([6], 1, 1, 64, 64, torch.float32, False, device="cpu")
    out, states, _ = reference(x)
    q, k, v = (x[n][:, 0].double() for n in "qkv")
    s0 = x["states"][int(x["slots"][0]), 0].double()
    g = x["decay"][:, 0].double().cumsum(0)
    for t in range(6):
        o = torch.exp(g[t]) * s0 @ q[t] + sum(torch.exp(g[t] - g[j]) * v[j] * (k[j] @ q[t]) for j in range(t + 1))
        assert torch.allclose(out[t, 0], o / 8, rtol=1e-12, atol=1e-12)


def test_descriptors_are_checked_without_a_device():
    import ctypes as C
    L = capi.lib()
    h = C.c_void_p()
    good = dict(ggml_type=30, n_head=4, n_head_qk=2, dim_k=64, dim_v=64, max_seqs=2, device=0)
    for change, code in ((dict(ggml_type=8), capi.ERR_UNSUPPORTED), (dict(dim_k=80), capi.ERR_UNSUPPORTED), (dict(n_head_qk=3), capi.ERR_ARGUMENT),
                         (dict(n_head_qk=0), capi.ERR_ARGUMENT), (dict(max_seqs=-1), capi.ERR_ARGUMENT), (dict(n_head=2000, n_head_qk=2), capi.ERR_ARGUMENT)):
        d = capi.LinearDesc(**{**good, **change})
        assert L.bivmoe_linear_create(C.byref(d), C.byref(h)) == code and not h.value
    assert L.bivmoe_linear_create(None, C.byref(h)) == capi.ERR_ARGUMENT
    assert L.bivmoe_linear_attend(None, None, None) == capi.ERR_ARGUMENT
    assert L.bivmoe_linear_status(None, None) == capi.ERR_ARGUMENT
    L.bivmoe_linear_destroy(None)


@gpu
@pytest.mark.parametrize("rows", [64, 700, 2500])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens_of_many_heads(rows, delta, dim):
    h = 16
    b = max(1, rows * 64 // (h * dim))
    x = make([i % 5 != 3 for i in range(b)], h, 4, dim, dim, torch.float16, delta, seed=rows)
    lay = layer(x, torch.float16)
    states = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=1)
    check(x, out, states, torch.float16)


@gpu
@pytest.mark.parametrize("rows", [64, 2500])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_token_by_token_of_many_heads(rows, delta, dim):
    h = 16
    b = max(1, rows * 64 // (h * dim))
    x = make([1 + 7 * i % 36 for i in range(b)], h, 4, dim, dim, torch.float16, delta, seed=rows)
    lay = layer(x, torch.float16)
    states = x["states"].clone()
    keep = [i % 40 for i in range(b)]
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=36,
                     keep=torch.tensor(keep, dtype=torch.int32, device="cuda"))
    check(x, out, states, torch.float16, keep=keep)


@gpu
@pytest.mark.parametrize("delta", [False, True])
def test_prompts_of_more_requests_than_rows_say(delta):
    """More than 64 requests, empty ones among them; fewer tokens told than there are; two streams at once, one of them a graph."""
    lengths = [(0, 20, 64, 1, 90)[i % 5] for i in range(70)]
    x = make(lengths, 4, 2, 128, 128, torch.bfloat16, delta, seed=70)
    y = make([2000, 30], 4, 2, 128, 128, torch.bfloat16, delta, seed=71)
    lay = layer(x, torch.bfloat16)
    call = lambda x, s, out, **more: lay.attend(x["q"], x["k"], x["v"], x["decay"], s, x["slots"], x["first"], beta=x["beta"], out=out, **more)  # noqa: E731
    runs = [(x, torch.cuda.Stream(), 20), (y, torch.cuda.Stream(), 17)]
    kept = []
    for x, stream, told in runs:
        states, out = x["states"].clone(), torch.empty_like(x["v"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call(x, states, out, max_new=told)
        kept.append((g, states, out))
    for _ in range(2):
        torch.cuda.synchronize()
        for (x, stream, _), (g, states, out) in zip(runs, kept):
            with torch.cuda.stream(stream):
                states.copy_(x["states"])
                g.replay()
    torch.cuda.synchronize()
    lay.status()
    for (x, _, _), (_, states, out) in zip(runs, kept):
        check(x, out, states, torch.bfloat16, prompt=True)


@gpu
@pytest.mark.parametrize("delta", [False, True])
def test_more_tokens_than_were_told(delta):
    """max_new decides the kernel alone: one token told, or eight, of some forty."""
    x = make([3, 1, 40, 0, 9], 4, 2, 128, 128, torch.bfloat16, delta, seed=12)
    lay = layer(x, torch.bfloat16)
    for told in (1, 8):
        states = x["states"].clone()
        out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=told)
        check(x, out, states, torch.bfloat16)


@gpu
def test_what_lies_over_one_another_is_not_written():
    x = make([20, 20], 4, 2, 128, 128, torch.bfloat16, False)
    lay = layer(x, torch.bfloat16)
    good = {k: x[k] for k in ("q", "k", "v", "decay", "states", "slots", "first")}
    one = torch.zeros((1, 4, 128), dtype=torch.bfloat16, device="cuda")
    for change in (dict(out=one.expand(40, 4, 128)), dict(out=one[:, :1].expand(40, 4, 128)), dict(states=x["states"][:1].expand(5, 4, 128, 128)),
                   dict(states=x["states"][:, :1].expand(5, 4, 128, 128))):
        with pytest.raises(capi.BivMoeError):
            lay.attend(**{**good, **change})
    # rows that are read may lie so: the copy engine takes no such stride, and the tokens are taken one by one
    same = {**x, "k": x["k"][:1].expand(40, 2, 128)}
    states = x["states"].clone()
    out = lay.attend(same["q"], same["k"], same["v"], same["decay"], states, same["slots"], same["first"])
    check(same, out, states, torch.bfloat16)


# Slots that are not there, one that is taken, past zero and not, without `keep`: by the kernels for prompts.  Lengths of one chunk, of
# some, and of as many as make clusters of two, four and eight blocks (148 multiprocessors; with them requests of one chunk, whose
# clusters have blocks without any).  A [700], above, is eleven chunks and has one block: clusters begin with sixteen.
SLOTS = [
    # lengths, heads, heads of q and k
    ([30, 70, 200, 0, 17, 1, 64, 300], 4, 2),
    ([1100], 40, 20),                              # two: 80 blocks; by four they would not run at once
    ([1100, 5, 1300], 14, 7),                      # two
    ([2100, 40, 1, 1500], 3, 1),                   # four, or as many as there is room for
    ([4300, 3, 64, 0, 4200, 130], 1, 1),           # eight
]


@gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("shape", SLOTS)
def test_prompts_whose_slots_are_not_there(shape, delta, which):
    """`which` turns the parts about: every length once has a state, none, and a slot that an earlier request has."""
    lengths, h, hk = shape
    x = make(lengths, h, hk, 128, 128, torch.bfloat16, delta, seed=sum(lengths) + which)
    slots = x["slots"].tolist()
    n = len(lengths)
    for b in range(n):
        part = (b + which) % 3
        if part == 1:
            slots[b] = (-1, 10 ** 6, x["states"].shape[0])[b % 3]
        elif part == 2 and b:
            slots[b] = slots[b - 1] if slots[b - 1] >= 0 else slots[0]
    past = [(0, 9, 4)[(b + b // 3 + which) % 3] for b in range(n)]
    x["slots"] = torch.tensor(slots, dtype=torch.int32, device="cuda")
    lay = layer(x, torch.bfloat16)
    states = x["states"].clone()
    out = lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"],
                     past=torch.tensor(past, dtype=torch.int32, device="cuda"), max_new=max(lengths))
    lay.status()
    check(x, out, states, torch.bfloat16, past=past, prompt=True)
    kept = {s for b, s in enumerate(slots) if 0 <= s < states.shape[0] and s not in slots[:b] and lengths[b]}
    left = [s for s in range(states.shape[0]) if s not in kept]
    assert torch.equal(states[left], x["states"][left])


@gpu
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("where", [0, 63, 64, 700, 1099])
def test_what_is_not_finite_in_clusters_and_at_the_ends_of_chunks(where, delta):
    """A value of v that is not finite, in the first pass of a cluster's stretch or the second, at the ends of chunks."""
    x = make([1100], 40, 20, 128, 128, torch.bfloat16, delta, seed=3)
    lay = layer(x, torch.bfloat16)
    call = lambda v, s: lay.attend(x["q"], x["k"], v, x["decay"], s, x["slots"], x["first"], beta=x["beta"], max_new=1100)  # noqa: E731
    s0, s1 = x["states"].clone(), x["states"].clone()
    clean = call(x["v"], s0)
    v = x["v"].clone()
    v[where, 7, 100], v[where, 7, 31] = math.inf, math.nan
    got = call(v, s1)
    lay.status()
    slot = int(x["slots"][0])
    rest = [i for i in range(128) if i not in (31, 100)]
    assert not got[where:, 7, [31, 100]].isfinite().any() and not s1[slot, 7, [31, 100]].isfinite().any()
    assert torch.equal(got[:where], clean[:where]) and torch.equal(got[:, 7, rest], clean[:, 7, rest]) and torch.equal(s1[slot, 7, rest], s0[slot, 7, rest])
    others = [i for i in range(40) if i != 7]
    assert torch.equal(got[:, others], clean[:, others]) and torch.equal(s1[slot, others], s0[slot, others])


@gpu
@pytest.mark.parametrize("dtype,lengths,dim", [(torch.bfloat16, [1, 1, 1], 128), (torch.float32, [5, 40], 64), (torch.bfloat16, [300, 30], 128),
                                               (torch.bfloat16, [2100], 128)])
@pytest.mark.parametrize("delta", [False, True])
def test_out_may_be_v_and_nothing_else(lengths, dim, dtype, delta):
    """Each kernel reads a row of v, of a head, in the block that writes that place of out, and before it does."""
    x = make(lengths, 4, 4, dim, dim, dtype, delta, seed=len(lengths))
    lay = layer(x, dtype)
    call = lambda s, **more: lay.attend(**{**{k: x[k] for k in ("q", "k", "v", "decay", "slots", "first", "beta")}, "states": s,  # noqa: E731
                                           "max_new": max(lengths), **more})
    s0, s1 = x["states"].clone(), x["states"].clone()
    want = call(s0)
    wide = torch.zeros((sum(lengths), 9, dim), dtype=dtype, device="cuda")
    v = wide[:, 2:6]
    v.copy_(x["v"])
    for bad in (dict(out=x["q"]), dict(out=x["k"]), dict(v=v, out=wide[:, 2::2])):
        with pytest.raises(capi.BivMoeError):
            call(s1, **bad)
    got = call(s1, v=v, out=v)
    assert got is v and torch.equal(v, want) and torch.equal(s1, s0)
    assert not wide[:, :2].any() and not wide[:, 6:].any()


@gpu
@pytest.mark.parametrize("delta", [False, True])
def test_prompts_and_single_tokens_of_one_batch_in_two_calls(delta):
    """The rows of a batch, its prompts first: each call takes a part of the lists, the offsets of the second begin behind the first's rows, and
    each leaves the other's rows and states alone."""
    lengths = [200, 33, 90] + [1] * 20
    x = make(lengths, 4, 2, 128, 128, torch.bfloat16, delta, seed=9)
    lay = layer(x, torch.bfloat16)
    states, out = x["states"].clone(), torch.full_like(x["v"], 5.0)
    call = lambda part, told: lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"][part], x["first"][part.start:part.stop + 1],  # noqa: E731
                                         beta=x["beta"], max_new=told, out=out)
    call(slice(3, 23), 1)
    prompts = x["slots"][:3].long()
    assert (out[:323] == 5).all() and torch.equal(states[prompts], x["states"][prompts])
    singles, rows = states.clone(), out[323:].clone()
    call(slice(0, 3), 200)
    others = [s for s in range(states.shape[0]) if s not in prompts.tolist()]
    assert torch.equal(out[323:], rows) and torch.equal(states[others], singles[others])
    check(x, out, states, torch.bfloat16, prompt=True)


@gpu
@pytest.mark.parametrize("delta", [False, True])
def test_a_long_request_takes_no_longer_behind_another(delta):
    """Blocks that are scheduled before the call ahead has ended go where that leaves room: those of a long request, which all run at once, were
    put several to one multiprocessor, for one and a half times the time."""
    x = make([1024], 32, 16, 128, 128, torch.float32, delta, seed=1)
    lay = layer(x, torch.float32)
    states, out = x["states"].clone(), torch.empty_like(x["v"])
    call = lambda: lay.attend(x["q"], x["k"], x["v"], x["decay"], states, x["slots"], x["first"], beta=x["beta"], max_new=1024, out=out)  # noqa: E731

    def time(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        for _ in range(n):
            call()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b) / n

    time(3)
    alone, behind = (sorted(time(n) for _ in range(7))[3] for n in (1, 30))
    assert behind < 1.08 * alone, (alone, behind)


@gpu
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("lengths,h,hk", [([65, 130], 4, 2), ([30, 1, 200], 3, 1), ([1100], 40, 20), ([2100, 40], 3, 1)])
def test_prompts_in_wide_rows_and_rows_behind_the_last(lengths, h, hk, delta):
    """q, k and v as parts of wider rows, every second one; decays and states with gaps; behind the last sequence, and before the first, rows of
    NaN, which a chunk's copies may bring in but nothing may reach, and outputs that stay."""
    d, n, before = 128, sum(lengths), 5
    x = make(lengths, h, hk, d, d, torch.bfloat16, delta, seed=n)
    t = before + n + 70
    rows = torch.full((t, 2, 2 * hk + h + 1, d), math.nan, dtype=torch.bfloat16, device="cuda")[:, 1]
    views = dict(q=rows[:, :hk], k=rows[:, hk:2 * hk], v=rows[:, 2 * hk:2 * hk + h])
    for name, view in views.items():
        view[before:before + n] = x[name]
    scalars = torch.full((t, 3 * h), math.nan, device="cuda")
    scalars[before:before + n, :h] = x["decay"]
    if delta:
        scalars[before:before + n, h:2 * h] = x["beta"]
    big = torch.full((x["states"].shape[0], 2, h + 1, d, d), 7.0, device="cuda")
    big[:, 1, :h] = x["states"]
    states = big[:, 1, :h]
    wide_out = torch.full((t, h + 2, d), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide_out[:, 1:h + 1]
    lay = layer(x, torch.bfloat16)
    first = x["first"] + before
    lay.attend(views["q"], views["k"], views["v"], scalars[:, :h], states, x["slots"], first, beta=scalars[:, h:2 * h] if delta else None,
               scale=-0.3, max_new=max(lengths), out=out)
    lay.status()
    check(x, out[before:before + n], states, torch.bfloat16, scale=-0.3, prompt=True)
    assert (wide_out[:, 0] == 3).all() and (wide_out[:, h + 1] == 3).all() and (out[:before] == 3).all() and (out[before + n:] == 3).all()
    assert (big[:, 0] == 7).all() and (big[:, 1, h] == 7).all()


@gpu
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("max_new", [0, 16, 200])
def test_offsets_that_pass_the_rows_or_decrease(max_new, delta):
    """Past n_tokens they count as n_tokens, decreasing ones as no tokens, negative ones as zero."""
    x = make([90, 0, 40], 4, 2, 128, 128, torch.bfloat16, delta, seed=4)
    lay = layer(x, torch.bfloat16)
    run = lambda first, s: lay.attend(x["q"], x["k"], x["v"], x["decay"], s, x["slots"],  # noqa: E731
                                      torch.tensor(first, dtype=torch.int32, device="cuda"), beta=x["beta"], max_new=max_new)
    s0, s1, s2 = (x["states"].clone() for _ in range(3))
    want = run([0, 90, 90, 130], s0)
    check(x, want, s0, torch.bfloat16, prompt=max_new != 16)
    assert torch.equal(run([-7, 90, 90, 2 ** 31 - 1], s1), want) and torch.equal(s1, s0)
    got = run([90, 20, 130, -(2 ** 31)], s2)                 # only the second request has rows: 20 to 129
    y = {**x, "first": torch.tensor([20, 20, 130, 130], dtype=torch.int32, device="cuda")}
    out, states, _ = reference(y)
    assert torch.equal(s2[x["slots"][[0, 2]].long()], x["states"][x["slots"][[0, 2]].long()])
    err = (s2.double().cpu() - states).norm() / states.norm()
    assert err < 1e-5 and (got[20:].double().cpu() - out[20:]).norm() / out[20:].norm() < 1e-2


@gpu
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("lengths,told", [([1, 3, 2], 3), ([100, 1, 70], 100)])
def test_rows_and_states_more_than_32_bits_apart(lengths, told, delta):
    """Rows 2^24 + 2^20 values from one another, 171 of them; slots of 2^18 values, the last of 9000 among them."""
    n, h, d, apart = sum(lengths), 4, 128, 2 ** 24 + 2 ** 20
    x = make(lengths, h, h, d, d, torch.bfloat16, delta, seed=2)
    room = torch.empty(n * apart, dtype=torch.bfloat16, device="cuda")
    views = {name: room[i * h * d:].as_strided((n, h, d), (apart, d, 1)) for i, name in enumerate(("q", "k", "v", "out"))}
    for name in ("q", "k", "v"):
        views[name].copy_(x[name])
    slots = [8999, 3, 8192]
    far = torch.empty((9000, 4, h, d, d), device="cuda")[:, 1]     # 2^18 values a slot: past 2^31 from the 8192nd on
    kept = torch.zeros((9, h, d, d), device="cuda")
    for i, (a, b) in enumerate(zip(slots, x["slots"].tolist())):
        far[a] = x["states"][b]
        kept[i] = x["states"][b]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lay = layer(x, torch.bfloat16)
    out = lay.attend(views["q"], views["k"], views["v"], x["decay"], far, ints(slots), x["first"], beta=x["beta"], max_new=told, out=views["out"])
    lay.status()
    y = {**x, "states": kept, "slots": ints([0, 1, 2])}
    got = kept.clone()
    got[:3] = far[slots]
    check(y, out, got, torch.bfloat16, prompt=told > 16)
