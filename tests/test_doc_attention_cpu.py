"""Document masks and masked attention on the CPU: ranges against a token-by-token statement, the
reference attention against a loop over rows, and every refusal."""
import math
import random

import pytest
import torch

from oxidizr_b200.ops import api


def rows_of(tokens, separator=None, pad=None, prefix=None, causal=True):
    """lo, hi by walking each row one token after another."""
    out = []
    for b, row in enumerate(tokens.tolist()):
        is_pad = [(t < 0) if separator is None else (pad is not None and t == pad) for t in row]
        ids, n = [], 0
        for i, t in enumerate(row):
            if i and (is_pad[i] != is_pad[i - 1] or (row[i - 1] == separator if separator is not None else t != row[i - 1])):
                n += 1
            ids.append(n)
        for i in range(len(row)):
            if is_pad[i]:
                out.append((0, 0))
                continue
            doc = [j for j in range(len(row)) if ids[j] == ids[i]]
            end = i + 1
            if not causal:
                end = doc[-1] + 1
            elif prefix is not None:
                p = doc[0]
                while p <= doc[-1] and prefix[b][p]:
                    p += 1
                end = max(end, p)
            out.append((doc[0], end))
    return torch.tensor(out, dtype=torch.int32).view(*tokens.shape, 2).unbind(-1)


def random_docs(B, S, seed, pad=True):
    rng = random.Random(seed)
    rows = []
    for _ in range(B):
        row, d = [], 0
        while len(row) < S:
            n = rng.randint(1, max(1, S // 3))
            row += [-1 - d % 2 if pad and rng.random() < 0.2 else d] * n
            d += 1
        rows.append(row[:S])
    return torch.tensor(rows), torch.tensor([[rng.random() < 0.7 for _ in range(S)] for _ in range(B)])


@pytest.mark.parametrize("B,S", [(1, 1), (2, 7), (3, 64), (1, 130)])
@pytest.mark.parametrize("kind", ["causal", "prefix", "both ways"])
def test_ranges_of_document_ids(B, S, kind):
    doc, flags = random_docs(B, S, B * 1000 + S)
    kw = {"causal": kind != "both ways", "prefix": flags if kind == "prefix" else None}
    m = api.document_mask(doc, **kw)
    lo, hi = rows_of(doc, **kw)
    assert torch.equal(m.lo, lo) and torch.equal(m.hi, hi)
    assert m.lo.dtype == m.hi.dtype == torch.int32


@pytest.mark.parametrize("pad", [None, 3, 7])
def test_ranges_of_separated_tokens(pad):
    rng = random.Random(5)
    ids = torch.tensor([[rng.choice([1, 2, 3, 7]) for _ in range(90)] for _ in range(3)])
    m = api.document_mask(ids, separator=7, pad=pad)
    lo, hi = rows_of(ids, separator=7, pad=pad)
    assert torch.equal(m.lo, lo) and torch.equal(m.hi, hi)


def by_rows(q, k, v, scale, m, cap, slopes):
    B, S, Hq, _ = q.shape
    o = torch.zeros(B, S, Hq, v.shape[-1], dtype=torch.float64)
    G = Hq // k.shape[2]
    for b in range(B):
        for i in range(S):
            lo, hi = int(m.lo[b, i]), int(m.hi[b, i])
            if lo >= hi:
                continue
            for h in range(Hq):
                a = [scale * float(q[b, i, h].double() @ k[b, j, h // G].double()) for j in range(lo, hi)]
                if cap:
                    a = [cap * math.tanh(x / cap) for x in a]
                if slopes is not None:
                    a = [x - float(slopes[h]) * abs(i - j) for x, j in zip(a, range(lo, hi))]
                w = torch.softmax(torch.tensor(a, dtype=torch.float64), 0)
                o[b, i, h] = w @ v[b, lo:hi, h // G].double()
    return o


@pytest.mark.parametrize("cap,alibi", [(0.0, False), (3.0, False), (0.0, True), (3.0, True)])
def test_reference_attention_is_the_definition(cap, alibi):
    torch.manual_seed(0)
    B, S, Hq, Hk = 2, 23, 4, 2
    q, k, v = torch.randn(B, S, Hq, 12), torch.randn(B, S, Hk, 12), torch.randn(B, S, Hk, 5)
    doc, flags = random_docs(B, S, 3)
    m = api.document_mask(doc, prefix=flags)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0]) if alibi else None
    empty = (m.hi <= m.lo)
    want = by_rows(q, k, v, 0.7, m, cap, slopes)
    # what padding holds must not matter
    for t in (q, k, v):
        t[empty] = float("nan")
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    o = api.attention(*leaves, 0.7, mask=m, softcap=cap, alibi=slopes)
    # 64-bit sums of at most 23 terms of about unit size
    assert (o - want).abs().max() < 1e-12
    do = torch.randn(o.shape, dtype=torch.float64)
    do[empty] = float("nan")
    for g in torch.autograd.grad(o, leaves, do):
        assert torch.isfinite(g).all() and (g[empty] == 0).all()


def test_fused_projection_is_the_separate_one():
    torch.manual_seed(1)
    qkv = torch.randn(2, 9, (4 + 2 * 2) * 8, requires_grad=True)
    doc, _ = random_docs(2, 9, 4)
    m = api.document_mask(doc)
    o = api.attention_qkv(qkv, 4, 2, 8, 0.4, mask=m, softcap=5.0)
    q, k, v = (t.unflatten(-1, (-1, 8)) for t in qkv.split([32, 16, 16], -1))
    assert torch.equal(o, api.attention(q, k, v, 0.4, mask=m, softcap=5.0).flatten(2))


def test_without_options_the_path_is_the_plain_one():
    torch.manual_seed(2)
    q, k, v = torch.randn(2, 9, 4, 8), torch.randn(2, 9, 2, 8), torch.randn(2, 9, 2, 8)
    one = api.document_mask(torch.zeros(2, 9, dtype=torch.int64))
    # one document, f32: sums of 9 terms, a few rounding steps apart
    assert (api.attention(q, k, v, 0.3, mask=one) - api.attention(q, k, v, 0.3)).abs().max() < 16 * 2 ** -24 * 4
    both = api.document_mask(torch.zeros(2, 9, dtype=torch.int64), causal=False)
    d = api.attention(q, k, v, 0.3, causal=False, mask=both) - api.attention(q, k, v, 0.3, causal=False)
    assert d.abs().max() < 16 * 2 ** -24 * 4


def test_refusals():
    doc = torch.zeros(2, 8, dtype=torch.int64)
    with pytest.raises(ValueError, match="int64 or int32"):
        api.document_mask(doc.float())
    with pytest.raises(ValueError, match="B, S"):
        api.document_mask(doc[0])
    with pytest.raises(ValueError, match="separator"):
        api.document_mask(doc, pad=0)
    with pytest.raises(ValueError, match="prefix"):
        api.document_mask(doc, prefix=torch.ones(2, 7, dtype=torch.bool))
    with pytest.raises(ValueError, match="prefix"):
        api.document_mask(doc, prefix=torch.ones(2, 8))
    with pytest.raises(ValueError, match="causal"):
        api.document_mask(doc, prefix=torch.ones(2, 8, dtype=torch.bool), causal=False)
    m = api.document_mask(doc)
    q, k, v = torch.randn(2, 8, 4, 8), torch.randn(2, 8, 2, 8), torch.randn(2, 8, 2, 8)
    ok = dict(mask=m)
    api.attention(q, k, v, 0.3, **ok)
    for bad in ((q, k[:, :7], v), (q, k, v[:, :, :1]), (q[:, :, :3], k, v), (q, k[..., :4], v)):
        with pytest.raises(ValueError, match="go together"):
            api.attention(*bad, 0.3, **ok)
    with pytest.raises(ValueError, match="scale"):
        api.attention(q, k, v, 0.0, **ok)
    with pytest.raises(ValueError, match="softcap"):
        api.attention(q, k, v, 0.3, softcap=-1.0)
    with pytest.raises(ValueError, match="softcap"):
        api.attention(q, k, v, 0.3, softcap=float("nan"))
    with pytest.raises(ValueError, match="mask is for"):
        api.attention(q[:1], k[:1], v[:1], 0.3, **ok)
    with pytest.raises(ValueError, match="causal"):
        api.attention(q, k, v, 0.3, causal=False, **ok)
    with pytest.raises(ValueError, match="slope"):
        api.attention(q, k, v, 0.3, alibi=torch.ones(3))
    with pytest.raises(ValueError, match="constants"):
        api.attention(q, k, v, 0.3, alibi=torch.ones(4, requires_grad=True))


def test_the_extension_refuses_with_exceptions():
    """What the bindings refuse comes back as an exception, also where the message holds numbers."""
    from oxidizr_b200.ops._C import raw_ext
    e = raw_ext()
    x = torch.zeros(1, 4, 2, 8, dtype=torch.bfloat16)
    st = torch.zeros(16, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="document_mask"):
        e.document_mask(torch.zeros(1, 4, dtype=torch.int64), None, None, None, True)
    with pytest.raises(RuntimeError):
        e.doc_attention(x, x, x, 0.1, 0.0, None, True, [], st)
    with pytest.raises(RuntimeError):
        e.doc_attention_qkv(x.flatten(2), 1, 1, 8, 0.1, 0.0, None, True, [], st)


def test_no_heads_are_refused():
    k = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError, match="do not go together"):
        api.attention(torch.zeros(1, 4, 0, 8), k, k, 0.1, softcap=1.0)
