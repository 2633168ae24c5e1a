"""Attention over visible key ranges on the GPU, against the formulas in 64 bits.

Tolerances count roundings: a bf16 value is off by at most 2^-8 of itself.  The kernel rounds P and dS to bf16
before they are multiplied, and o, dq, dk, dv once at the end; delta is formed from the rounded o.  What the
special functions and f32 sums add (exponentials and tanh are good to about 2^-20, sums of n terms to n 2^-24)
is covered by 2^-11 of the same sums of absolute values.
"""
import random

import pytest
import torch

from oxidizr_b200.ops import api

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8     # one rounding to bf16
REST = 2.0 ** -11    # f32 arithmetic


def layout(B, S, mean, seed, pad=True):
    rng = random.Random(seed)
    doc, flag = [], []
    for _ in range(B):
        row, fl, d = [], [], 0
        while len(row) < S:
            n = 1 + int(rng.expovariate(1.0 / mean))
            p = rng.randint(0, n)
            row += [-1 if pad and rng.random() < 0.15 else d] * n
            fl += [True] * p + [False] * (n - p)
            d += 1
        doc.append(row[:S])
        flag.append(fl[:S])
    return torch.tensor(doc, device="cuda"), torch.tensor(flag, device="cuda")


def oracle(q, k, v, do, scale, m, cap, slopes):
    """o, dq, dk, dv in 64 bits and how far each may be off."""
    B, S, Hq, D = q.shape
    G = Hq // k.shape[2]
    empty = (m.hi <= m.lo)
    z64 = lambda t: t.detach().double().masked_fill(empty[..., None, None], 0.0).transpose(1, 2)  # noqa: E731
    q, k, v, do = z64(q), z64(k), z64(v), z64(do)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    pos = torch.arange(S, device=q.device)
    sees = ((pos >= m.lo[..., None]) & (pos < m.hi[..., None]))[:, None]
    z = scale * q @ k.transpose(2, 3)
    f = 1.0
    if cap:
        t = torch.tanh(z / cap)
        z, f = cap * t, 1 - t * t
    if slopes is not None:
        z = z - slopes.double().view(-1, 1, 1) * (pos[:, None] - pos).abs()
    p = torch.softmax(z.masked_fill(~(sees | empty[:, None, :, None]), -float("inf")), -1) * sees
    o = p @ v
    o_tol = HALF * o.abs() + (HALF + REST) * (p @ v.abs())
    dp = do @ v.transpose(2, 3)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * f
    # dS before it is rounded: delta is off by o's error, P and dP by f32 arithmetic
    ds_err = p * f * ((do.abs() * o_tol).sum(-1, keepdim=True) + REST * (do.abs() @ v.abs().transpose(2, 3) + delta.abs()))
    ds_tol = HALF * ds.abs() + (1 + HALF) * ds_err
    dq, dk, dv = scale * ds @ k, scale * ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do
    dq_tol = scale * ds_tol @ k.abs()
    dk_tol = scale * ds_tol.transpose(2, 3) @ q.abs()
    dv_tol = (HALF + REST) * p.transpose(2, 3) @ do.abs()

    def fold(t):  # sum over the query heads of a key head
        return t.view(B, -1, G, S, t.shape[-1]).sum(2)

    outs = [(o, o_tol)]
    for g, tol, n in ((dq, dq_tol, 1), (dk, dk_tol, G), (dv, dv_tol, G)):
        g, tol = (fold(g), fold(tol)) if n > 1 else (g, tol)
        outs.append((g, tol + HALF * (g.abs() + tol)))
    return [(a.transpose(1, 2), b.transpose(1, 2) + 1e-30) for a, b in outs]


def check(got, want):
    for name, x, (y, tol) in zip(("o", "dq", "dk", "dv"), got, want):
        assert x.shape == y.shape, name
        off = ((x.double() - y).abs() / tol).nan_to_num(float("inf")).max().item() if x.numel() else 0.0
        assert off <= 1.0, f"{name}: {off:.2f} of the tolerance"


def inputs(B, S, Hq, Hk, D, Dv, seed=0, sharp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k = (rnd(B, S, Hq, D) * sharp).bfloat16(), (rnd(B, S, Hk, D) * sharp).bfloat16()
    return q, k, rnd(B, S, Hk, Dv).bfloat16(), rnd(B, S, Hq, Dv).bfloat16()


def run(q, k, v, do, scale, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = api.attention(*leaves, scale, **kw)
    return [o.detach(), *torch.autograd.grad(o, leaves, do)]


def finish():
    from oxidizr_b200.ops._C import check_status
    torch.cuda.synchronize()
    check_status("cuda")


@pytest.mark.parametrize("B,S", [(1, 1), (2, 2), (3, 64), (2, 127), (2, 128), (1, 129), (2, 257), (1, 500), (1, 1000)])
@pytest.mark.parametrize("kind", ["ids", "prefix", "both ways", "separator"])
def test_ranges_are_the_reference(B, S, kind):
    from oxidizr_b200.ops import reference as R
    doc, flags = layout(B, S, max(1, S // 5), S)
    args = {"ids": (None, None, None, True), "prefix": (None, None, flags, True), "both ways": (None, None, None, False),
            "separator": (1, 2, flags, True)}[kind]
    if kind == "separator":
        doc = doc.abs() % 5
    m = api.document_mask(doc, *args[:2], prefix=args[2], causal=args[3])
    lo, hi = R.document_ranges(doc.cpu(), *args[:2], args[2].cpu() if args[2] is not None else None, args[3])
    assert torch.equal(m.lo.cpu(), lo) and torch.equal(m.hi.cpu(), hi)
    # the tile tables, from the ranges
    lo, hi = lo.long(), hi.long()
    for b in range(B):
        for t in range((S + 127) // 128):
            a, e = lo[b, t * 128:t * 128 + 128], hi[b, t * 128:t * 128 + 128]
            some = e > a
            want = [int(a[some].min()), int(e[some].max())] if some.any() else [0, 0]
            got = m.qt[b, t].tolist()
            assert got[:2] == want
            if some.all():
                assert got[2:] == [int(a.max()), int(e.min())]
            else:
                assert got[2] == 2 ** 31 - 1
            sees = [u for u in range(m.qt.shape[1]) if m.qt[b, u, 0] < t * 128 + 128 and m.qt[b, u, 1] > t * 128]
            assert m.kt[b, t].tolist()[:3] == [sees[0] if sees else 0, sees[-1] + 1 if sees else 0, int(not some.all())]


def test_long_rows():
    """Rows of many words per thread of the mask kernel, and the longest one."""
    from oxidizr_b200.ops import reference as R
    for S in (40001, 262144):
        doc, flags = layout(1, S, 3000, S)
        m = api.document_mask(doc, prefix=flags)
        lo, hi = R.document_ranges(doc, prefix=flags)
        assert torch.equal(m.lo, lo) and torch.equal(m.hi, hi)
    with pytest.raises(ValueError, match="at most"):
        api.document_mask(torch.zeros(1, 262145, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("S", [1, 2, 63, 128, 129, 256, 300, 513])
@pytest.mark.parametrize("cap,alibi", [(0.0, False), (8.0, False), (0.0, True), (8.0, True)])
def test_lengths_and_scores(S, cap, alibi):
    B, Hq, Hk, D = 2, 4, 2, 64
    x = inputs(B, S, Hq, Hk, D, D, S, 1.5)
    doc, flags = layout(B, S, max(1, S // 3), S + 1)
    m = api.document_mask(doc, prefix=flags)
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.0], device="cuda") if alibi else None
    scale = D ** -0.5
    check(run(*x, scale, mask=m, softcap=cap, alibi=slopes), oracle(*x, scale, m, cap, slopes))
    finish()


@pytest.mark.parametrize("D,Dv", [(8, 8), (32, 32), (40, 32), (64, 64), (80, 64), (96, 64), (64, 128), (72, 120), (128, 128),
                                  (128, 8)])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (6, 2), (4, 4)])
def test_head_layouts(D, Dv, Hq, Hk):
    B, S = 2, 200
    x = inputs(B, S, Hq, Hk, D, Dv, D + Hq)
    doc, _ = layout(B, S, 60, D)
    m = api.document_mask(doc)
    check(run(*x, D ** -0.5, mask=m), oracle(*x, D ** -0.5, m, 0.0, None))
    finish()


@pytest.mark.parametrize("causal", [True, False])
def test_without_a_mask(causal):
    B, S, D = 2, 333, 128
    x = inputs(B, S, 4, 2, D, D, 9, 2.0)
    m = api.document_mask(torch.zeros(B, S, dtype=torch.int64, device="cuda"), causal=causal)
    want = oracle(*x, D ** -0.5, m, 20.0, None)
    check(run(*x, D ** -0.5, causal=causal, softcap=20.0), want)
    check(run(*x, D ** -0.5, causal=causal, mask=m, softcap=20.0), want)
    finish()


def test_documents_both_ways():
    B, S, D = 2, 400, 64
    x = inputs(B, S, 2, 2, D, D, 10)
    doc, _ = layout(B, S, 90, 10)
    m = api.document_mask(doc, causal=False)
    check(run(*x, D ** -0.5, causal=False, mask=m), oracle(*x, D ** -0.5, m, 0.0, None))
    finish()


@pytest.mark.parametrize("D,Dv", [(64, 64), (96, 64), (128, 128)])
def test_padding_may_hold_anything(D, Dv):
    """NaN and infinities in the padding rows of q, k, v and the gradient reach nothing."""
    B, S = 3, 384
    q, k, v, do = inputs(B, S, 4, 2, D, Dv, 3)
    doc, _ = layout(B, S, 50, 3)
    doc[1] = -1           # a row of nothing but padding
    doc[2, 100:] = -1     # a padded batch row
    m = api.document_mask(doc)
    want = oracle(q, k, v, do, D ** -0.5, m, 15.0, None)
    empty = m.hi <= m.lo
    for i, t in enumerate((q, k, v, do)):
        t[empty] = (float("nan"), float("inf"), float("nan"), -float("inf"))[i]
    got = run(q, k, v, do, D ** -0.5, mask=m, softcap=15.0)
    check(got, want)
    for t in got:
        assert (t[empty] == 0).all()
    finish()


def test_scores_far_apart():
    """Large scores: the running maximum moves in every tile, and capped scores sit at the cap."""
    B, S, D = 1, 700, 64
    q, k, v, do = inputs(B, S, 2, 1, D, D, 4)
    k = (k.float() * torch.linspace(0.1, 12.0, S, device="cuda")[None, :, None, None]).bfloat16()
    m = api.document_mask(torch.zeros(B, S, dtype=torch.int64, device="cuda"))
    for cap in (0.0, 2.0, 500.0):
        check(run(q, k, v, do, 1.0, mask=m, softcap=cap), oracle(q, k, v, do, 1.0, m, cap, None))
    finish()


def test_strides_and_projection():
    """Heads-first views, a fused projection with a row stride, an unaligned view, an expanded gradient."""
    B, S, Hq, Hk, D = 2, 150, 4, 2, 64
    q, k, v, do = inputs(B, S, Hq, Hk, D, D, 5)
    doc, _ = layout(B, S, 40, 5)
    m = api.document_mask(doc)
    scale = D ** -0.5
    want = run(q, k, v, do, scale, mask=m)
    hf = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for a, b in zip(run(*hf, do, scale, mask=m), want):
        assert torch.equal(a, b)
    wide = torch.randn(B, S, (Hq + 2 * Hk) * D + 8, device="cuda").bfloat16()
    for off in (8, 3):
        qkv = wide[..., off:off + (Hq + 2 * Hk) * D]
        qkv.copy_(torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1))
        leaf = qkv.detach().requires_grad_(True)
        o = api.attention_qkv(leaf, Hq, Hk, D, scale, mask=m)
        (g,) = torch.autograd.grad(o, leaf, do.flatten(2))
        assert torch.equal(o, want[0].flatten(2))
        assert torch.equal(g, torch.cat([t.flatten(2) for t in want[1:]], -1))
    leaf = q.detach().requires_grad_(True)
    one = torch.ones((), device="cuda", dtype=torch.bfloat16)
    (g,) = torch.autograd.grad(api.attention(leaf, k, v, scale, mask=m), leaf, one.expand(B, S, Hq, D))
    check([g], [oracle(q, k, v, one.expand(B, S, Hq, D), scale, m, 0.0, None)[1]])
    finish()


def test_gradient_against_differences():
    """The directional derivative of sum(o w) along random directions, in 64-bit differences of the definition."""
    B, S, D = 1, 160, 64
    q, k, v, w = inputs(B, S, 2, 2, D, D, 6)
    doc, flags = layout(B, S, 50, 6)
    m = api.document_mask(doc, prefix=flags)
    slopes = torch.tensor([0.3, 0.05], device="cuda")
    grads = run(q, k, v, w, D ** -0.5, mask=m, softcap=4.0, alibi=slopes)[1:]
    tol = [t for _, t in oracle(q, k, v, w, D ** -0.5, m, 4.0, slopes)[1:]]

    def f(q, k, v):
        from oxidizr_b200.ops import reference as R
        o = R.attention_ranges(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), D ** -0.5, m.lo, m.hi, 4.0, slopes)
        return (o.transpose(1, 2) * w.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i in range(3):
        d = torch.randn_like(x[i])
        h = 1e-4
        hi, lo = (f(*[t + s * h * d if j == i else t for j, t in enumerate(x)]) for s in (1, -1))
        diff = ((hi - lo) / (2 * h)).item()
        assert abs((grads[i].double() * d).sum().item() - diff) <= (tol[i] * d.abs()).sum().item() + 1e-5 * abs(diff)


def test_deterministic_and_capturable():
    """Two runs agree bit for bit, on another stream and replayed from a graph with other inputs too."""
    B, S, Hq, Hk, D = 2, 520, 4, 2, 128
    x, y = inputs(B, S, Hq, Hk, D, D, 7, 2.0), inputs(B, S, Hq, Hk, D, D, 8, 2.0)
    docs = [layout(B, S, 100, s)[0] for s in (7, 8)]
    scale = D ** -0.5

    def step(q, k, v, do, doc):
        return run(q, k, v, do, scale, mask=api.document_mask(doc), softcap=30.0)

    want = [step(*x, docs[0]), step(*y, docs[1])]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step(*x, docs[0])
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(other, want[0]):
        assert torch.equal(a, b)
    static, sdoc = [t.clone() for t in x], docs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*static, sdoc)
    for inp, d, w in ((y, docs[1], want[1]), (x, docs[0], want[0])):
        for a, b in zip(static, inp):
            a.copy_(b)
        sdoc.copy_(d)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, w):
            assert torch.equal(a, b)
    finish()


def test_other_types_take_the_stated_math():
    q, k, v, do = (t.float() for t in inputs(1, 70, 2, 1, 16, 16, 11))
    doc, _ = layout(1, 70, 20, 11)
    m = api.document_mask(doc)
    got = run(q, k, v, do, 0.25, mask=m, softcap=5.0)
    # (some hosts' f32 matrix products keep 16 bits of their operands: the 64-bit form is what holds everywhere)
    for a, (b, _) in zip(got, oracle(q, k, v, do, 0.25, m, 5.0, None)):
        # an f32 evaluation of sums of up to 70 terms
        assert (a.double() - b).abs().max() <= 70 * 2 ** -22 * b.abs().max()


def test_refusals_on_the_gpu():
    q, k, v, _ = inputs(1, 16, 2, 1, 16, 16, 12)
    m = api.document_mask(torch.zeros(1, 16, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="mask is for"):
        api.attention(q, k, v, 0.25, mask=api.document_mask(torch.zeros(1, 16, dtype=torch.int64)))
    with pytest.raises(ValueError, match="mask is for"):
        api.attention(q[:, :8], k[:, :8], v[:, :8], 0.25, mask=m)
    with pytest.raises(ValueError, match="slope"):
        api.attention(q, k, v, 0.25, mask=m, alibi=torch.ones(2))


def test_graph_is_kept_and_second_derivatives_are_refused():
    torch.manual_seed(3)
    qkv = torch.randn(2, 70, 3 * 64, device="cuda").bfloat16().requires_grad_()
    o = api.attention_qkv(qkv, 1, 1, 64, 0.125, softcap=20.0)
    do = torch.randn_like(o)
    a, = torch.autograd.grad(o, qkv, do, retain_graph=True)
    b, = torch.autograd.grad(o, qkv, do, retain_graph=True)
    assert torch.equal(a, b)
    a2, = torch.autograd.grad(o, qkv, do, create_graph=True)
    assert torch.equal(a, a2)
    with pytest.raises(RuntimeError, match="first derivatives"):
        a2.float().sum().backward()
    q, k, v = (t.unflatten(-1, (1, 64)) for t in qkv.split(64, -1))
    o2 = api.attention(q, k, v, 0.125, softcap=20.0)
    assert torch.equal(o2.flatten(2), o)
    c, = torch.autograd.grad(o2, qkv, do.view_as(o2))
    assert torch.equal(a, c)
    with torch.no_grad():
        assert not api.attention(q, k, v, 0.125, softcap=20.0).requires_grad


def test_only_some_operands_want_gradients():
    torch.manual_seed(4)
    q, k, v = (torch.randn(1, 90, 2, 64, device="cuda").bfloat16() for _ in range(3))
    do = torch.randn_like(q)
    for t in (q, k, v):
        t.requires_grad_()
    full = torch.autograd.grad(api.attention(q, k, v, 0.125, softcap=5.0), (q, k, v), do)
    k.requires_grad_(False)
    part = torch.autograd.grad(api.attention(q, k, v, 0.125, softcap=5.0), (q, v), do)
    assert torch.equal(part[0], full[0]) and torch.equal(part[1], full[2])


def test_launches_of_backward_passes_are_counted():
    from oxidizr_b200.ops._C import launch_counter
    qkv = torch.randn(1, 70, 3 * 64, device="cuda").bfloat16().requires_grad_()
    launch_counter.count = 0
    launch_counter.enabled = True
    try:
        api.attention_qkv(qkv, 1, 1, 64, 0.125, softcap=20.0).sum().backward()
    finally:
        launch_counter.enabled = False
    n = launch_counter.count
    assert n == 2
    api.attention_qkv(qkv, 1, 1, 64, 0.125, softcap=20.0).sum().backward()
    assert launch_counter.count == n


@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_negative_slopes(cap):
    """A bias that grows with the distance: scores far above the cap, whose sums must not overflow."""
    S = 400
    m = api.document_mask(torch.zeros(1, S, dtype=torch.int64, device="cuda"))
    slopes = torch.tensor([-1.0, 0.5], device="cuda")
    q, k, v, do = inputs(1, S, 2, 1, 64, 64, seed=11)
    got = run(q, k, v, do, 0.125, mask=m, softcap=cap, alibi=slopes)
    check(got, oracle(q, k, v, do, 0.125, m, cap, slopes))
    finish()


def test_operands_off_the_alignment():
    """Contiguous operands whose first element is not at a multiple of 16 bytes are copied."""
    q, k, v, do = inputs(2, 130, 2, 2, 64, 64, seed=12)
    want = run(q, k, v, do, 0.125, softcap=20.0)

    def shifted(t):
        buf = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")
        buf[3:].copy_(t.detach().reshape(-1))
        return buf[3:].view(t.shape)

    got = run(*(shifted(t).requires_grad_() for t in (q, k, v)), shifted(do), 0.125, softcap=20.0)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    finish()


@pytest.mark.parametrize("S", [4097, 8192, 12417, 33000])
@pytest.mark.parametrize("mean", [30, 5000, 10 ** 6])
def test_ranges_across_slices(S, mean):
    """Documents, prompts and padding that reach over several CTAs' slices of a row, and none that do."""
    from oxidizr_b200.ops import reference as R
    doc, flags = layout(3, S, mean, S + mean)
    long = torch.arange(S, device="cuda").expand(3, S) < torch.tensor([[S], [S // 2], [4096]], device="cuda")
    for prefix, causal in ((None, True), (None, False), (flags, True), (long, True), (~long, True)):
        m = api.document_mask(doc, prefix=prefix, causal=causal)
        lo, hi = R.document_ranges(doc, prefix=prefix, causal=causal)
        assert torch.equal(m.lo, lo) and torch.equal(m.hi, hi)
        nt = (S + 127) // 128
        pad = nt * 128 - S
        some = torch.nn.functional.pad(hi > lo, (0, pad)).view(3, nt, 128)
        a = torch.nn.functional.pad(lo, (0, pad)).view(3, nt, 128)
        e = torch.nn.functional.pad(hi, (0, pad)).view(3, nt, 128)
        kmin = a.masked_fill(~some, 2 ** 31 - 1).amin(-1) * some.any(-1)
        kmax = e.masked_fill(~some, 0).amax(-1)
        assert torch.equal(m.qt[..., 0], kmin.int()) and torch.equal(m.qt[..., 1], kmax)
        k0 = torch.arange(nt, device="cuda") * 128
        sees = (kmin[:, :, None] < k0 + 128) & (kmax[:, :, None] > k0)  # [B, query tile, key tile]
        n = torch.arange(nt, device="cuda")[:, None]
        end = torch.where(sees, n + 1, 0).amax(1)
        first = torch.where(sees, n, nt).amin(1) * (end > 0)
        assert torch.equal(m.kt[..., 0], first.int()) and torch.equal(m.kt[..., 1], end.int())


@pytest.mark.parametrize("mean,cap", [(1.5, 0.0), (3, 20.0), (12, 0.0), (100, 50.0), (700, 20.0)])
def test_sharp_scores_keep_the_gradients(mean, cap):
    """Rows with one dominant key, whose dP - delta nearly cancels.  In the 2-norm a gradient is off by the rounding
    of its bf16 terms and its own, each at most 2^-8 / sqrt 3 of a value (rms): 0.82 x 2^-8 together, and the rest
    of 2^-8 for the forward's rounded weights."""
    B, S = 2, 900
    q, k, v, do = inputs(B, S, 4, 2, 64, 64, seed=int(mean * 10), sharp=2.0)
    doc = layout(B, S, mean, int(mean), pad=False)[0] if mean > 2 else torch.arange(S, device="cuda").expand(B, S) * 2 // 3
    m = api.document_mask(doc)
    got = run(q, k, v, do, 0.125, mask=m, softcap=cap)
    want = oracle(q, k, v, do, 0.125, m, cap, None)
    check(got, want)
    for name, x, (y, _) in zip(("o", "dq", "dk", "dv"), got, want):
        assert (x.double() - y).norm() <= HALF * y.norm(), name
    finish()


@pytest.mark.parametrize("D,Dv", [(64, 64), (96, 64), (128, 128)])
def test_tiles_of_padding_alone(D, Dv):
    """Tiles with nothing to compute: their zeros are staged where operands land, which must have landed."""
    B, S = 16, 2048
    q, k, v, do = inputs(B, S, 4, 4, D, Dv, seed=21)
    doc = torch.where(torch.arange(S, device="cuda") < 200, 0, -1).expand(B, S)
    m = api.document_mask(doc)
    first = None
    for _ in range(20):
        got = run(q, k, v, do, D ** -0.5, mask=m)
        for x in got:
            assert not x[:, 200:].any()
        if first is None:
            first = got
        for x, y in zip(got, first):
            assert torch.equal(x, y)
    finish()


@pytest.mark.parametrize("S", [1, 2, 3, 130, 700])
@pytest.mark.parametrize("causal", [True, False])
def test_plain_attention_runs_the_same_kernels(S, causal):
    """Without a mask, a cap or slopes too, both entry points."""
    q, k, v, do = inputs(2, S, 4, 2, 64, 64, seed=S)
    lo = torch.zeros(2, S, dtype=torch.int64, device="cuda")
    hi = torch.arange(1, S + 1, device="cuda").expand(2, S) if causal else torch.full((2, S), S, device="cuda")
    m = type("M", (), {"lo": lo, "hi": hi})
    got = run(q, k, v, do, 0.125, causal=causal)
    check(got, oracle(q, k, v, do, 0.125, m, 0.0, None))
    qkv = torch.cat([t.flatten(2) for t in (q, k, v)], -1).requires_grad_()
    o = api.attention_qkv(qkv, 4, 2, 64, 0.125, causal=causal)
    g, = torch.autograd.grad(o, qkv, do.flatten(2))
    assert torch.equal(o, got[0].flatten(2)) and torch.equal(g, torch.cat([t.flatten(2) for t in got[1:]], -1))
    finish()


@pytest.mark.parametrize("S,causal", [(1, True), (1, False), (300, True)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_one_key_gets_no_gradient_through_its_score(S, causal, cap):
    """A softmax over one key is constant: dQ and dK are zeros, not what rounding leaves."""
    q, k, v, do = inputs(2, S, 4, 2, 64, 32, seed=31)
    masks = [api.document_mask(torch.arange(S, device="cuda").expand(2, S), causal=causal)] + ([None] if S == 1 else [])
    for m in masks:
        o, dq, dk, dv = run(q, k, v, do, 0.125, mask=m, softcap=cap, causal=causal)
        assert torch.equal(o, v.repeat_interleave(2, 2)) and not dq.any() and not dk.any()
        want = do.double().unflatten(2, (2, 2)).sum(3)
        assert ((dv.double() - want).abs() <= HALF * want.abs() + 2 * (HALF + REST) * do.double().unflatten(2, (2, 2)).abs().sum(3)).all()
    finish()


def test_offsets_past_31_bits():
    """The last row of a batch of 2.4e9 elements gives what it gives alone."""
    B, S, H, D = 24, 8192, 32, 128
    qkv = torch.empty(B, S, 3 * H * D, dtype=torch.bfloat16, device="cuda").normal_().requires_grad_()
    doc = (torch.arange(S, device="cuda") // 200).expand(B, S)
    do = torch.empty(B, S, H * D, dtype=torch.bfloat16, device="cuda").normal_()
    o = api.attention_qkv(qkv, H, H, D, D ** -0.5, mask=api.document_mask(doc))
    g, = torch.autograd.grad(o, qkv, do)
    one = qkv.detach()[-1:].clone().requires_grad_()
    o1 = api.attention_qkv(one, H, H, D, D ** -0.5, mask=api.document_mask(doc[-1:]))
    g1, = torch.autograd.grad(o1, one, do[-1:])
    assert torch.equal(o[-1:], o1) and torch.equal(g[-1:], g1)
    finish()


def test_nothing_to_attend():
    """No tokens, and no rows."""
    for B, S in ((2, 0), (0, 5)):
        m = api.document_mask(torch.zeros(B, S, dtype=torch.int64, device="cuda"))
        assert m.lo.shape == (B, S)
        q, k, v, do = inputs(B, S, 2, 1, 64, 64)
        for kw in (dict(mask=m), dict(softcap=5.0), {}):
            for x, y in zip(run(q, k, v, do, 0.125, **kw), (q, q, k, v)):
                assert x.shape == y.shape
    finish()


def test_two_streams_at_once():
    """Passes on two streams, which share nothing."""
    args = [inputs(2, 700, 4, 2, D, D, seed=D) for D in (64, 128)]
    doc = layout(2, 700, 90, 3)[0]

    def step(q, k, v, do):
        return run(q, k, v, do, 0.1, mask=api.document_mask(doc), softcap=30.0)

    want = [step(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(step(*a))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        for x, y in zip(r, want[i % 2]):
            assert torch.equal(x, y)
    finish()


@pytest.mark.parametrize("D,Dv,S,causal", [(64, 64, 16, True), (64, 64, 300, True), (64, 64, 130, False), (96, 64, 64, True),
                                           (128, 64, 100, True), (128, 128, 128, False)])
def test_many_short_rows(D, Dv, S, causal):
    """Plain attention whose rows are too short for the backward's CTAs runs the kernels that are faster there: the same
    mathematics on either side of the rule's border."""
    from oxidizr_b200.ops.doc_attention import takes_plain
    H, B = 8, -(-10 * 148 // (8 * ((S + 127) // 128)))
    q, k, v, do = inputs(B, S, H, H, D, Dv, seed=S)
    scale = D ** -0.5
    many = (H, H, D, Dv, scale, causal, True)
    assert not takes_plain(q, *many) and takes_plain(q[1:], *many)
    assert takes_plain(q, *many[:-1], False) == (S > 64)
    lo = torch.zeros(B, S, dtype=torch.int64, device="cuda")
    hi = torch.arange(1, S + 1, device="cuda").expand(B, S) if causal else torch.full((B, S), S, device="cuda")
    for first in (0, 1):
        x = [t[first:] for t in (q, k, v, do)]
        got = run(*x, scale, causal=causal)
        check(got, oracle(*x, scale, type("M", (), {"lo": lo[first:], "hi": hi[first:]}), 0.0, None))
        if D == Dv:
            qkv = torch.cat([t.flatten(2) for t in x[:3]], -1).requires_grad_()
            o = api.attention_qkv(qkv, H, H, D, scale, causal=causal)
            g, = torch.autograd.grad(o, qkv, x[3].flatten(2))
            assert torch.equal(o, got[0].flatten(2))
            check([*(t.unflatten(2, (H, D)) for t in g.split(H * D, -1))], oracle(
                *x, scale, type("M", (), {"lo": lo[first:], "hi": hi[first:]}), 0.0, None)[1:])
    with torch.no_grad():
        check([api.attention(q, k, v, scale, causal=causal)], oracle(q, k, v, do, scale, type("M", (), {"lo": lo, "hi": hi}), 0.0, None))
    finish()


@pytest.mark.parametrize("D,Dv,Hq,Hk", [(96, 64, 3, 3), (128, 64, 4, 1), (128, 128, 4, 2), (40, 32, 2, 2), (64, 128, 2, 1)])
@pytest.mark.parametrize("mean,cap,alibi", [(3, 0.0, False), (12, 20.0, True), (100, 0.0, True), (700, 50.0, False)])
def test_sharp_scores_keep_the_gradients_at_every_width(D, Dv, Hq, Hk, mean, cap, alibi):
    """In the 2-norm, as above: delta from the two-part output (from o as it is rounded, dQ would be off by 1.5 x 2^-8)."""
    B, S = 2, 700
    q, k, v, do = inputs(B, S, Hq, Hk, D, Dv, seed=D + mean, sharp=2.0 * (64 / D) ** 0.25)
    slopes = torch.tensor([0.3, 0.05, 0.01, 0.0], device="cuda")[:Hq] if alibi else None
    m = api.document_mask(layout(B, S, mean, mean, pad=False)[0])
    got = run(q, k, v, do, D ** -0.5, mask=m, softcap=cap, alibi=slopes)
    want = oracle(q, k, v, do, D ** -0.5, m, cap, slopes)
    check(got, want)
    for name, x, (y, _) in zip(("o", "dq", "dk", "dv"), got, want):
        assert (x.double() - y).norm() <= HALF * y.norm(), name
    finish()


@pytest.mark.parametrize("S,D", [(2, 64), (3, 128), (40, 64)])
def test_many_short_rows_of_any_layout(S, D):
    """Operands and gradients off the alignment, of odd strides and expanded: on either side of the rule's border, as
    without it.  Second derivatives are refused by both."""
    H = 8
    for B in (200, 30):
        q, k, v, do = inputs(B, S, H, H, D, D, seed=S)
        scale = D ** -0.5
        want = run(q, k, v, do, scale)
        hi = torch.arange(1, S + 1, device="cuda").expand(B, S)
        m = type("M", (), {"lo": torch.zeros_like(hi), "hi": hi})
        ref = oracle(q, k, v, do, scale, m, 0.0, None)
        check(want, ref)

        def off(t, by):
            buf = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
            buf[by:].copy_(t.reshape(-1))
            return buf[by:].view(t.shape)

        check(run(off(q, 3), k, v, do, scale), ref)
        check(run(q, k, v, off(do, 1), scale), ref)
        wide = torch.zeros(B, S, H, D + 1, device="cuda").bfloat16()
        wide[..., :D] = v
        check(run(q, k, wide[..., :D], do, scale), ref)
        heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
        check(run(*heads, do, scale), ref)
        qkv = off(torch.cat([t.flatten(2) for t in (q, k, v)], -1), 5).requires_grad_()
        o = api.attention_qkv(qkv, H, H, D, scale)
        (g,) = torch.autograd.grad(o, qkv, off(do.flatten(2), 7))
        check([o.unflatten(2, (H, D)), *(t.unflatten(2, (H, D)) for t in g.split(H * D, -1))], ref)
        leaf = q.detach().requires_grad_(True)
        one = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(B, S, H, D)
        (g,) = torch.autograd.grad(api.attention(leaf, k, v, scale), leaf, one)
        check([g], [oracle(q, k, v, one, scale, m, 0.0, None)[1]])
        (g,) = torch.autograd.grad(api.attention(leaf, k, v, scale), leaf, do, create_graph=True)
        with pytest.raises(RuntimeError, match="first derivatives|once_differentiable"):
            g.float().sum().backward()
    finish()
