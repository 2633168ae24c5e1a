"""Expert routing and the scaled embedding on the GPU, against 64-bit statements.

Tolerances count roundings: f32 values are off by at most 2^-24 of themselves, bf16 by 2^-8.
"""
import pytest
import torch

from oxidizr_b200.ops import api
from oxidizr_b200.ops import reference as R

pytestmark = pytest.mark.gpu
F32, BF16 = 2.0 ** -24, 2.0 ** -8


def finish():
    from oxidizr_b200.ops._C import check_status
    torch.cuda.synchronize()
    check_status("cuda")


# ------------------------------------------------------------------ routing
def route_both(x, k, dw, du, **kw):
    leaf = x.detach().requires_grad_(True)
    got = api.route_topk(leaf, k, **kw)
    got = [t.detach() for t in got] + list(torch.autograd.grad(got[1:3], leaf, (dw, du)))
    wide = x.detach().double().requires_grad_(True)
    want = R.route_topk(wide, k, kw.get("score", "softmax"), kw.get("bias"), kw.get("groups", 1), kw.get("top_groups", 1),
                        kw.get("group_top", 2), kw.get("renorm", True), kw.get("scale", 1.0))
    want = [t.detach() for t in want] + list(torch.autograd.grad(want[1:3], wide, (dw.double(), du.double())))
    return got, want


def check_route(x, k, dw, du, **kw):
    got, want = route_both(x, k, dw, du, **kw)
    T, E = x.shape
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])
    # an exponential is good to 2 steps, its sum over E terms to log E more, a quotient or two: 24 steps
    assert ((got[1].double() - want[1]).abs() <= 24 * F32 * want[1].abs() + 1e-30).all()
    # usage adds T positive terms, in runs of at most T / 32 after one another
    assert ((got[2].double() - want[2]).abs() <= (24 + 2 * (T // 32 + 32)) * F32 * want[2].abs() + 1e-30).all()
    # the gradient is a difference of sums: its parts in absolute values bound what f32 does to it
    s = torch.softmax(x.double(), -1) if kw.get("score", "softmax") == "softmax" else torch.sigmoid(x.double())
    S = s.sum(-1, keepdim=True)
    sel = s.gather(1, want[0])
    n = sel.sum(-1, keepdim=True) if kw.get("renorm", True) else torch.ones_like(S)
    g = dw.double().abs() * kw.get("scale", 1.0) / n
    g = g + (g * sel).sum(-1, keepdim=True) / n
    part = torch.zeros_like(s).scatter_add_(1, want[0], g)
    u = du.double().abs() / T
    part = part + (u + (u * s).sum(-1, keepdim=True) / S) / S
    size = s * (part + (s * part).sum(-1, keepdim=True))
    step = BF16 if x.dtype == torch.bfloat16 else F32
    assert ((got[4].double() - want[4]).abs() <= step * want[4].abs() + 64 * F32 * size + 1e-30).all()
    finish()


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 2, 2), (100, 5, 3), (257, 32, 4), (64, 33, 8), (500, 64, 8), (77, 100, 16),
                                   (300, 256, 8), (200, 257, 9), (50, 512, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_routing(T, E, k, score, biased, dt):
    g = torch.Generator(device="cuda").manual_seed(T + E)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    check_route((rnd(T, E) * 1.5).to(dt), k, rnd(T, k), rnd(E), score=score, renorm=(T % 2 == 0), scale=1.5,
                bias=rnd(E) * (0.1 if score == "sigmoid" else 0.3 / E) if biased else None)


@pytest.mark.parametrize("E,groups,top_groups,group_top,k", [(8, 8, 3, 2, 3), (12, 4, 2, 2, 5), (64, 8, 4, 2, 8), (96, 3, 1, 1, 8),
                                                             (160, 8, 3, 2, 6), (256, 8, 4, 2, 8), (256, 2, 1, 3, 8),
                                                             (512, 32, 7, 2, 16), (320, 32, 9, 2, 12)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_grouped_routing(E, groups, top_groups, group_top, k, score, biased):
    T = 301
    g = torch.Generator(device="cuda").manual_seed(E + groups)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    check_route(rnd(T, E).bfloat16(), k, rnd(T, k), rnd(E), score=score, groups=groups, top_groups=top_groups,
                group_top=group_top, scale=2.5, bias=rnd(E) * (0.1 if score == "sigmoid" else 0.3 / E) if biased else None)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_near_ties_are_decided_in_64_bits(score):
    """Scores whose order f32 cannot tell: pairs a rounding step of a bias apart, and exact ties."""
    T, E, k = 512, 64, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randint(-3, 4, (T, E), generator=g, device="cuda").float() / 2)
    s = torch.softmax(x[0].double(), -1) if score == "softmax" else torch.sigmoid(x[0].double())
    # bias that makes the first token's scores all but equal in f32, in no particular order in f64
    bias = (s.max() - s).float()
    dw, du = torch.randn(T, k, device="cuda"), torch.randn(E, device="cuda")
    x[1::2] = x[0]
    check_route(x, k, dw, du, score=score, bias=bias)
    check_route(x, k, dw, du, score=score, bias=torch.zeros(E, device="cuda"))
    check_route(x, k, dw, du, score=score)
    check_route(x, k, dw, du, score=score, bias=bias, groups=8, top_groups=3)
    check_route(torch.zeros_like(x), k, dw, du, score=score, groups=8, top_groups=3)


def test_masked_experts_and_extreme_logits():
    """Experts shut out by a logit of -inf, and logits far out, where exponentials vanish."""
    T, E, k = 40, 48, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(T, E, generator=g, device="cuda") * 20
    x[:, 5:20] = -float("inf")
    topi, topw, usage, counts = api.route_topk(x, k)
    ti, tw, tu, tc = R.route_topk(x.double(), k)
    assert torch.equal(topi, ti) and torch.equal(counts, tc) and (counts[5:20] == 0).all() and (usage[5:20] == 0).all()
    assert ((topw.double() - tw).abs() <= 64 * F32 * tw + 1e-30).all()
    topi, topw, _, _ = api.route_topk(x, k, "sigmoid")
    assert torch.equal(topi, ti) and torch.isfinite(topw).all()
    # bias of -inf: never chosen while others are left
    bias = torch.zeros(E, device="cuda")
    bias[::2] = -float("inf")
    topi = api.route_topk(x.clamp(min=-1e4), k, "sigmoid", bias)[0]
    assert (topi % 2 == 1).all()
    finish()


def test_routing_layouts_streams_and_graphs():
    T, E, k = 130, 64, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(T, 3 * E + 1, generator=g, device="cuda").bfloat16()
    x = wide[:, E + 1:2 * E + 1]
    dw, du = torch.randn(T, k, device="cuda"), torch.randn(E, device="cuda")
    kw = dict(score="sigmoid", bias=torch.randn(E, device="cuda") * 0.1, groups=4, top_groups=2)
    check_route(x, k, dw, du, **kw)
    check_route(x.t().contiguous().t(), k, dw, du, **kw)
    want = route_both(x, k, dw, du, **kw)[0]
    # one of the two outputs alone passes a gradient
    leaf = x.detach().requires_grad_(True)
    out = api.route_topk(leaf, k, **kw)
    (a,) = torch.autograd.grad(out[1], leaf, dw, retain_graph=True)
    (b,) = torch.autograd.grad(out[2], leaf, du)
    assert (a.float() + b.float() - want[4].float()).abs().max() <= 4 * BF16 * want[4].abs().max()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [t.detach() for t in api.route_topk(x, k, **kw)]
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(other, want):
        assert torch.equal(p, q)  # usage too: the same sums in the same order
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = api.route_topk(static, k, **kw)
    static.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0].flip(0)) and torch.equal(out[3], want[3])
    empty = api.route_topk(x[:0], k, **kw)
    assert empty[0].shape == (0, k) and (empty[2] == 0).all() and (empty[3] == 0).all()
    finish()


def test_larger_routers_take_the_stated_math():
    x = torch.randn(9, 600, device="cuda")
    topi, topw, usage, counts = api.route_topk(x, 40)
    ti, tw, tu, tc = R.route_topk(x.double(), 40)
    assert torch.equal(topi, ti) and torch.equal(counts, tc)
    assert ((topw.double() - tw).abs() <= 64 * F32 * tw).all()


# ------------------------------------------------------------------ embedding
def check_embedding(ids, V, H, dt, scale, seed=0, misalign=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, H, generator=g, device="cuda").to(dt)
    flat = torch.randn(ids.numel() * H + misalign, generator=g, device="cuda").to(dt)
    dy = flat[misalign:].view(*ids.shape, H)
    step = BF16 if dt == torch.bfloat16 else F32
    leaf = w.detach().requires_grad_(True)
    y = api.embedding(ids, leaf, scale=scale)
    want = w.double()[ids] * scale
    assert ((y.double() - want).abs() <= (step + F32) * want.abs()).all()
    (dw,) = torch.autograd.grad(y, leaf, dy)
    sums = torch.zeros(V, H, dtype=torch.float64, device="cuda")
    mags = torch.zeros_like(sums)
    sums.index_add_(0, ids.flatten(), dy.double().view(-1, H) * scale)
    mags.index_add_(0, ids.flatten(), dy.double().abs().view(-1, H) * abs(scale))
    n = torch.bincount(ids.flatten(), minlength=V)[:, None].double()
    # f32 sums of n terms, the scale, and the rounding to the result's type
    tol = step * sums.abs() + (n + 2) * F32 * mags * (1 + step)
    assert dw.dtype == dt and ((dw.double() - sums).abs() <= tol).all()
    assert (dw[n[:, 0] == 0] == 0).all()
    (again,) = torch.autograd.grad(api.embedding(ids, leaf, scale=scale), leaf, dy)
    assert torch.equal(dw, again)
    # into main_grad, as the optimizer's buffer takes it
    p = torch.nn.Parameter(w.clone())
    p.main_grad = torch.randn(V, H, generator=g, device="cuda")
    before = p.main_grad.clone()
    api.embedding(ids, p, scale=scale).backward(dy)
    assert p.grad is None
    acc = before.double() + sums
    assert ((p.main_grad.double() - acc).abs() <= (n + 2) * F32 * mags + F32 * acc.abs()).all()
    assert torch.equal(p.main_grad[n[:, 0] == 0], before[n[:, 0] == 0])
    finish()


@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (1, 1000, 64), (31, 5, 8), (32, 3, 256), (33, 50, 264), (1000, 511, 128),
                                   (1024, 512, 96), (1025, 513, 1000), (5000, 128354, 64), (40000, 300, 16)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_embedding(T, V, H, dt):
    g = torch.Generator().manual_seed(T)
    ids = (torch.rand(T, generator=g) ** 3 * V).long().clamp(max=V - 1).cuda()
    check_embedding(ids, V, H, dt, 1.0 if T % 2 else 11.5)


@pytest.mark.parametrize("H", [1, 7, 20, 132])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_embedding_odd_widths(H, dt):
    ids = torch.randint(0, 40, (3, 77), device="cuda")
    check_embedding(ids, 40, H, dt, 0.5)


def test_embedding_runs_of_one_token():
    """Segments that end at, before and after a block's edge, fill many blocks, or are all there is."""
    for runs in ([(3, 32), (4, 32)], [(3, 31), (4, 33), (5, 1)], [(9, 5000)], [(0, 1), (1, 70), (2, 64), (3, 1), (4, 300)],
                 [(7, 96), (8, 32), (9, 1)]):
        ids = torch.cat([torch.full((n,), v) for v, n in runs]).cuda()
        perm = torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1)).cuda()
        check_embedding(ids, 10, 72, torch.bfloat16, 1.0)
        check_embedding(ids[perm], 10, 72, torch.float32, 1.0)


def test_embedding_misaligned_gradient():
    check_embedding(torch.randint(0, 9, (50,), device="cuda"), 9, 64, torch.bfloat16, 1.0, misalign=1)


def test_embedding_ids_out_of_range():
    from oxidizr_b200.ops._C import read_status
    w = torch.randn(6, 16, device="cuda").bfloat16().requires_grad_(True)
    ids = torch.tensor([5, -1, 6, 2, 10 ** 12, 5], device="cuda")
    y = api.embedding(ids, w)
    assert read_status("cuda") == 3  # reported, and cleared for the next call
    ok = torch.tensor([True, False, False, True, False, True], device="cuda")
    assert torch.equal(y[ok], w.detach()[ids[ok]]) and (y[~ok] == 0).all()
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert g[5].eq(2).all() and g[2].eq(1).all() and (g[[0, 1, 3, 4]] == 0).all()
    finish()


def test_embedding_empty_and_captured():
    w = torch.randn(30, 64, device="cuda").bfloat16().requires_grad_(True)
    y = api.embedding(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), w)
    (g,) = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert y.shape == (2, 0, 64) and (g == 0).all()
    # an eager graph of the leaf that outlives the capture would keep its gradient on the eager stream
    del y, g
    ids = torch.randint(0, 30, (4, 200), device="cuda")
    other = torch.randint(0, 30, (4, 200), device="cuda")
    dy = torch.randn(4, 200, 64, device="cuda").bfloat16()

    def step(i):
        y = api.embedding(i, w, scale=8.0)
        return [y, *torch.autograd.grad(y, w, dy)]

    want = [[t.detach().clone() for t in step(i)] for i in (ids, other)]
    static = ids.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i, ref in ((other, want[1]), (ids, want[0])):
        static.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, ref):
            assert torch.equal(a, b)
    finish()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [2, 40, 256])
def test_one_renormalised_expert(E, score):
    """Its weight is the scale whatever the logits: what reaches them is the usage's gradient alone, to f32's accuracy."""
    T = 4000
    g = torch.Generator(device="cuda").manual_seed(E)
    x = torch.randn(T, E, generator=g, device="cuda")
    dw, du = torch.randn(T, 1, generator=g, device="cuda"), torch.randn(E, generator=g, device="cuda")
    got, want = route_both(x, 1, dw, du, score=score, scale=2.5)
    # per element an f32 chain of 64 steps over parts that are at most a few times the result's size, in the 2-norm
    assert (got[4].double() - want[4]).norm() <= 256 * F32 * want[4].norm()
    got, _ = route_both(x, 1, dw, torch.zeros_like(du), score=score, scale=2.5)
    assert not got[4].any()


def test_embedding_offsets_past_31_bits():
    """Rows of a table of 2.3e9 elements, the last of them too."""
    V, H = 1_150_000, 2048
    w = torch.empty(V, H, dtype=torch.bfloat16, device="cuda").normal_().requires_grad_()
    ids = torch.tensor([[V - 1, 0, V - 1, 1_100_000]], device="cuda")
    y = api.embedding(ids, w)
    assert torch.equal(y, w.detach()[ids])
    dy = torch.randn(1, 4, H, device="cuda").bfloat16()
    g, = torch.autograd.grad(y, w, dy)
    want = (dy[0, 0].float() + dy[0, 2].float()).bfloat16()
    assert torch.equal(g[V - 1], want) and torch.equal(g[0], dy[0, 1]) and torch.equal(g[1_100_000], dy[0, 3])
    assert int((g != 0).any(1).sum()) == 3
    finish()


def test_routing_of_no_tokens():
    x = torch.zeros(0, 16, device="cuda").requires_grad_()
    topi, topw, usage, counts = api.route_topk(x, 2)
    assert topi.shape == topw.shape == (0, 2) and not usage.any() and not counts.any()
    g, = torch.autograd.grad(topw.sum() + usage.sum(), x)
    assert g.shape == x.shape
    finish()


@pytest.mark.parametrize("T", [1, 31, 33, 255, 256, 257, 500])
@pytest.mark.parametrize("H,dt", [(40, torch.bfloat16), (256, torch.float32), (7, torch.float32)])
@pytest.mark.parametrize("hot", [0.0, 0.8])
def test_embedding_of_few_tokens(T, H, dt, hot):
    """Either side of the size where the gradient sorts, with one token that is most of the batch; new and added to."""
    from oxidizr_b200.ops._C import ext
    V = 90
    g = torch.Generator(device="cuda").manual_seed(T + H)
    ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    ids = torch.where(torch.rand(T, generator=g, device="cuda") < hot, 5, ids)
    dy = torch.randn(T, H, generator=g, device="cuda").to(dt)
    want = torch.zeros(V, H, dtype=torch.float64, device="cuda").index_add_(0, ids, dy.double())
    size = torch.zeros_like(want).index_add_(0, ids, dy.double().abs())
    got = ext().embedding_bwd(ids, dy, V, 2.0, None)
    step = BF16 if dt == torch.bfloat16 else F32
    # a sum of up to T terms in f32, the scale and the rounding of the type
    assert ((got.double() - 2 * want).abs() <= step * 2 * want.abs() + (T + 4) * F32 * 2 * size + 1e-30).all()
    acc = torch.ones(V, H, device="cuda")
    ext().embedding_bwd(ids, dy, V, 2.0, acc)
    assert ((acc.double() - 1 - 2 * want).abs() <= (T + 6) * F32 * (1 + 2 * size)).all()
    assert torch.equal(acc[size.sum(1) == 0], torch.ones_like(acc[size.sum(1) == 0]))


@pytest.mark.parametrize("main_grad", [False, True])
@pytest.mark.parametrize("shape", [(3, 50), (700,)])
def test_ids_overwritten_before_the_backward(shape, main_grad):
    """Ids in a buffer that the next batch is copied into: the gradient of the old batch is refused, not scattered to the
    new one's rows."""
    ids = torch.randint(0, 30, shape, device="cuda")
    for view in (ids, ids.t()) if len(shape) == 2 else (ids, ids[::2]):
        w = torch.nn.Parameter(torch.randn(30, 16, device="cuda").bfloat16())
        if main_grad:
            w.main_grad = torch.zeros(30, 16, device="cuda")
        y = api.embedding(view, w)
        ids.copy_(ids.flip(0))
        # (ids that are not contiguous may have been copied: then the old batch's rows are what they get)
        if view.is_contiguous() or not main_grad:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
    finish()


def test_outputs_overwritten_before_the_backward():
    x = torch.randn(40, 16, device="cuda", requires_grad=True)
    topi, topw, _, _ = api.route_topk(x, 3)
    topi.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        topw.sum().backward()
    finish()


@pytest.mark.parametrize("E,k", [(6, 2), (64, 8), (200, 8)])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_gradient_of_saturated_sigmoids(E, k, renorm, dt):
    """Logits out to 30, where s is 1 to f32 and 1 - s is not nothing: the gradient is held relative to s (1 - s)."""
    T, scale = 300, 2.5
    g = torch.Generator(device="cuda").manual_seed(E)
    x = ((torch.rand(T, E, generator=g, device="cuda") * 2 - 1) * 30).to(dt)
    x[::7] = x[::7].abs()  # tokens with positive logits alone
    dw, du = torch.randn(T, k, generator=g, device="cuda"), torch.randn(E, generator=g, device="cuda")
    got, want = route_both(x, k, dw, du, score="sigmoid", renorm=renorm, scale=scale)
    assert torch.equal(got[0], want[0])
    s, q = torch.sigmoid(x.double()), torch.sigmoid(-x.double())
    S = s.sum(-1, keepdim=True)
    sel = s.gather(1, want[0])
    n = sel.sum(-1, keepdim=True) if renorm else torch.ones_like(S)
    a = dw.double().abs() * scale / n
    # renormalised, of differences from the first gradient: up to twice each, and their mean
    a = 2 * a + 2 * (a * sel).sum(-1, keepdim=True) / n if renorm else a
    part = torch.zeros_like(s).scatter_add_(1, want[0], a)
    u = du.double().abs() / T
    part = part + (u + (u * s).sum(-1, keepdim=True) / S) / S
    # e^x is off by |x| + 4 steps of f32, in s or in 1 - s and in the sums of s; quotients, products and sums 40 more
    tol = (2 * 30 + 48) * F32 * s * q * part
    step = BF16 if dt == torch.bfloat16 else F32
    assert ((got[4].double() - want[4]).abs() <= step * want[4].abs() + tol + 1e-30).all()
    finish()


@pytest.mark.parametrize("T,V,H", [(1024, 700, 40), (1025, 1, 36), (1500, 3, 7), (5000, 128354, 64), (20000, 2 ** 18 + 1, 8),
                                   (70000, 511, 24), (300001, 40000, 8)])
@pytest.mark.parametrize("hot", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_embedding_order_made_beside_the_lookup(T, V, H, hot, dt):
    """The tokens' order of a lookup that trains, and of a gradient that makes its own: the same bits; ids outside the
    rows, one token that is most of the batch, sums of thousands of parts."""
    from oxidizr_b200.ops._C import ext, read_status
    g = torch.Generator(device="cuda").manual_seed(T + H)
    ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    ids = torch.where(torch.rand(T, generator=g, device="cuda") < hot, V // 2, ids)
    ids[::97] = torch.tensor([-1, V], device="cuda").repeat(T)[:ids[::97].numel()]
    there = (ids >= 0) & (ids < V)
    w = torch.randn(V, H, generator=g, device="cuda").to(dt).requires_grad_(True)
    dy = torch.randn(T, H, generator=g, device="cuda").to(dt)
    y, other = api.embedding(ids, w, scale=2.0), api.embedding(ids.flip(0), w)
    assert read_status("cuda") == 3  # the ids outside
    assert torch.equal(y[there], (w.detach()[ids[there]].float() * 2.0).to(dt)) and not y[~there].any()
    (dw,) = torch.autograd.grad(y, w, dy, retain_graph=True)
    (again,) = torch.autograd.grad(y, w, dy)
    assert torch.equal(dw, again) and torch.equal(dw, ext().embedding_bwd(ids, dy, V, 2.0, None))
    want = torch.zeros(V, H, dtype=torch.float64, device="cuda").index_add_(0, ids[there], dy[there].double())
    size = torch.zeros_like(want).index_add_(0, ids[there], dy[there].double().abs())
    step = BF16 if dt == torch.bfloat16 else F32
    # runs of up to 32 terms, one sum of their parts, the scale and the rounding of the type
    steps = 32 + T // 32 + 4
    assert ((dw.double() - 2 * want).abs() <= step * 2 * want.abs() + steps * F32 * 2 * size + 1e-30).all()
    (dw,) = torch.autograd.grad(other, w, dy.flip(0))
    assert ((dw.double() - want).abs() <= step * want.abs() + steps * F32 * size + 1e-30).all()
    # added to an optimizer's buffer: bit for bit the same each time
    p = torch.nn.Parameter(w.detach().clone())
    got = []
    for _ in range(2):
        p.main_grad = torch.ones(V, H, device="cuda")
        api.embedding(ids, p, scale=2.0).backward(dy)
        got.append(p.main_grad)
    assert torch.equal(*got) and read_status("cuda") == 3
    assert ((got[0].double() - 1 - 2 * want).abs() <= F32 * (1 + 2 * want.abs()) + steps * F32 * 2 * size).all()
    finish()


def test_embedding_of_many_tokens_captured_and_on_another_stream():
    T, V, H = 3000, 500, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    ids = [torch.randint(0, V, (T,), generator=g, device="cuda") for _ in range(2)]
    w = torch.randn(V, H, generator=g, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(T, H, generator=g, device="cuda").bfloat16()

    def step(i):
        y = api.embedding(i, w)
        return [y.detach(), *torch.autograd.grad(y, w, dy)]

    want = [step(i) for i in ids]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step(ids[0])
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(other, want[0]))
    static = ids[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in (1, 0, 1):
        static.copy_(ids[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
    finish()


@pytest.mark.parametrize("T", [6, 1500])
def test_embedding_differentiated_twice(T):
    """A penalty on the gradient's size: its derivative by what came back, which is a lookup, and by the weights."""
    V, H, scale = 40, 8, 3.0
    g = torch.Generator(device="cuda").manual_seed(T)
    ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    w = torch.randn(V, H, generator=g, device="cuda")

    def penalty(look, w):
        y = look(w)
        (dw,) = torch.autograd.grad((y * y * y).sum(), w, create_graph=True)
        assert dw.requires_grad
        return torch.autograd.grad((dw * dw).sum(), w)[0]

    got = penalty(lambda w: api.embedding(ids, w, scale=scale), w.clone().requires_grad_(True))
    want = penalty(lambda w: w[ids] * scale, w.double().requires_grad_(True))
    # sums of up to n rows that are products of a few rounded factors, twice; all terms of a row have one sign each
    n = int(torch.bincount(ids, minlength=V).max())
    assert ((got.double() - want).abs() <= (2 * n + 24) * F32 * want.abs()).all()
    finish()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,renorm", [(8, 2, True), (300, 20, True), (300, 20, False)])
def test_routing_differentiated_twice(E, k, renorm, score):
    """A penalty on the router's gradient, differentiated by the logits and by what came back."""
    T = 33
    g = torch.Generator(device="cuda").manual_seed(E)
    x, dw, du = (torch.randn(*s, generator=g, device="cuda") for s in ((T, E), (T, k), (E,)))

    def second(route, x, dw, du):
        x, dw, du = (t.clone().requires_grad_(True) for t in (x, dw, du))
        topi, topw, usage, _ = route(x * 1.0)
        (dx,) = torch.autograd.grad((topw, usage), x, (dw, du), create_graph=True)
        return [dx.detach(), *torch.autograd.grad((dx * dx).sum(), (x, dw, du))]

    kw = dict(score=score, renorm=renorm, scale=1.5)
    got = second(lambda v: api.route_topk(v, k, **kw), x, dw, du)
    want = second(lambda v: R.route_topk(v, k, score, None, 1, 1, 2, renorm, 1.5), *(t.double() for t in (x, dw, du)))
    for a, b in zip(got, want):
        # f32 sums of E terms and their derivatives, in the 2-norm
        assert (a.double() - b).norm() <= (E + 64) * F32 * b.norm()
    # the gradient that is recorded is the one that is not
    leaf = x.clone().requires_grad_(True)
    out = api.route_topk(leaf, k, **kw)
    (plain,) = torch.autograd.grad((out[1], out[2]), leaf, (dw, du))
    assert (plain - got[0]).norm() <= (E + 64) * F32 * plain.norm()
    finish()


def test_routing_of_other_layouts_differentiated_twice():
    """Logits whose rows are not contiguous, which the kernel takes as a copy."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x, dw = torch.randn(12, 30, generator=g, device="cuda"), torch.randn(30, 3, generator=g, device="cuda")

    def second(x, route):
        x = x.clone().requires_grad_(True)
        w = route(x.t())[1]
        (dx,) = torch.autograd.grad(w, x, dw.to(x.dtype), create_graph=True)
        return dx.detach(), torch.autograd.grad((dx * dx).sum(), x)[0]

    got = second(x, lambda v: api.route_topk(v, 3, "sigmoid"))
    want = second(x.double(), lambda v: R.route_topk(v, 3, "sigmoid"))
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 80 * F32 * b.norm()
    finish()
