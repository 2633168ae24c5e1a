"""Routing and the scaled embedding on the CPU: the reference against loops, and every refusal."""
import math
import random

import pytest
import torch

from oxidizr_b200.ops import api


def route_by_loops(x, k, score, bias, groups, top_groups, group_top, renorm, scale):
    """topi, topw of one token, in Python floats."""
    E = len(x)
    if score == "softmax":
        m = max(x)
        s = [math.exp(v - m) for v in x]
        s = [v / sum(s) for v in s]
    else:
        s = [1.0 / (1.0 + math.exp(-v)) for v in x]
    b = [v + (bias[e] if bias else 0.0) for e, v in enumerate(s)]
    n = E // groups
    rank = [sum(sorted(b[g * n:(g + 1) * n], reverse=True)[:group_top]) for g in range(groups)]
    keep = sorted(range(groups), key=lambda g: (-rank[g], g))[:top_groups]
    pick = sorted((e for e in range(E) if e // n in keep), key=lambda e: (-b[e], e))[:k]
    total = sum(s[e] for e in pick) if renorm else 1.0
    return pick, [scale * s[e] / total for e in pick], [v / sum(s) for v in s]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,k,groups,top_groups,group_top", [(1, 1, 1, 1, 2), (7, 3, 1, 1, 2), (12, 4, 4, 2, 2),
                                                             (12, 2, 4, 2, 1), (8, 3, 8, 5, 2), (30, 9, 3, 3, 2)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_topk_is_the_definition(score, with_bias, E, k, groups, top_groups, group_top, renorm):
    torch.manual_seed(E * k)
    x = torch.randn(17, E)
    bias = torch.randn(E) * 0.1 if with_bias else None
    leaf = x.double().requires_grad_(True)
    topi, topw, usage, counts = api.route_topk(leaf, k, score, bias, groups, top_groups, group_top, renorm, 1.7)
    share = torch.zeros(E, dtype=torch.float64)
    for t in range(17):
        pick, w, u = route_by_loops(x[t].tolist(), k, score, bias.tolist() if with_bias else None, groups, top_groups,
                                    group_top, renorm, 1.7)
        assert topi[t].tolist() == pick
        assert (topw[t] - torch.tensor(w, dtype=torch.float64)).abs().max() < 1e-13
        share += torch.tensor(u, dtype=torch.float64) / 17
    assert (usage - share).abs().max() < 1e-13
    assert counts.dtype == torch.int32 and counts.tolist() == [int((topi == e).sum()) for e in range(E)]
    assert torch.autograd.gradcheck(lambda v: api.route_topk(v, k, score, bias, groups, top_groups, group_top, renorm,
                                                             1.7)[1:3], (leaf,), eps=1e-6, atol=1e-6)


def test_equal_scores_take_the_lowest_index():
    x = torch.zeros(2, 6)
    topi = api.route_topk(x, 3)[0]
    assert topi.tolist() == [[0, 1, 2]] * 2
    topi = api.route_topk(x, 2, "sigmoid", None, groups=3, top_groups=1)[0]
    assert topi.tolist() == [[0, 1]] * 2


def test_route_topk_refusals():
    x = torch.randn(4, 12)
    for bad, match in [((x[0], 2), "T, E"), ((x.long(), 2), "floating"), ((x, 2, "relu"), "softmax or sigmoid"),
                       ((x, 0), "choose"), ((x, 13), "choose"), ((x, 2, "softmax", None, 5), "groups"),
                       ((x, 2, "softmax", None, 4, 5), "groups"), ((x, 2, "softmax", None, 4, 0), "groups"),
                       ((x, 4, "softmax", None, 4, 1), "choose"), ((x, 2, "softmax", None, 4, 1, 0), "groups"),
                       ((x, 2, "softmax", torch.zeros(11)), "bias")]:
        with pytest.raises(ValueError, match=match):
            api.route_topk(*bad)


def test_scaled_embedding():
    w = torch.randn(11, 6, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[1, 1, 4], [10, 0, 1]], dtype=torch.int32)
    y = api.embedding(ids, w, scale=3.0)
    assert torch.equal(y, w.detach()[ids.long()] * 3.0)
    dy = torch.randn_like(y)
    (g,) = torch.autograd.grad(y, w, dy)
    want = torch.zeros_like(w)
    for i, row in zip(ids.flatten().tolist(), dy.flatten(0, 1)):
        want[i] += 3.0 * row
    assert (g - want).abs().max() < 1e-14
    assert torch.equal(api.embedding(ids, w), w.detach()[ids.long()])


def test_embedding_refusals():
    w = torch.randn(4, 8)
    with pytest.raises(ValueError, match="ids"):
        api.embedding(torch.tensor([1.0]), w)
    with pytest.raises(ValueError, match="V, H"):
        api.embedding(torch.tensor([1]), w[0])


def test_the_extension_refuses_with_exceptions():
    from oxidizr_b200.ops._C import raw_ext
    e = raw_ext()
    ids, w = torch.tensor([1]), torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="embedding"):
        e.embedding_fwd(ids, w, 1.0, torch.zeros(16, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="embedding"):
        e.embedding_bwd(ids, w, 4, 1.0, None)
    with pytest.raises(RuntimeError, match="router logits"):
        e.router_fwd(w, 2, False, None, 1, 1, 2, True, 1.0)
    with pytest.raises(RuntimeError, match="router logits"):
        e.router_bwd(w, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), None, False, True, 1.0)


def test_gradient_of_saturated_sigmoids():
    """s (1 - s) is 1e-7 at 16 and 9e-14 at 30: not zero, and not what rounding s to f32 leaves of 1 - s."""
    x = torch.tensor([[16.0, 20.0, 30.0, -30.0, 12.0]], requires_grad=True)
    topw = api.route_topk(x, 4, "sigmoid", renorm=False)[1]
    (g,) = torch.autograd.grad(topw.sum(), x)
    e = torch.exp(-x.detach().double().abs())
    # -30 is the one that is not chosen; an exponential, two quotients and a product in f32
    assert ((g.double() - (e / (1 + e) ** 2).index_fill(1, torch.tensor([3]), 0.0)).abs() <= 8 * 2 ** -24 * e).all()
    # and the second derivative is that of the formula
    wide = x.detach().double().requires_grad_(True)
    assert torch.autograd.gradgradcheck(lambda v: api.route_topk(v / 8, 4, "sigmoid", renorm=False)[1], (wide,))
