"""Work of the packed-document training operators: document masks, attention over documents (with capped
scores, a distance bias, prefixes, padding), the scaled embedding with its gradient, and routing to experts.

``run`` computes a case in elementary torch operations (``own`` false) or through
``oxidizr_b200.ops.api`` (``own`` true); ``exact`` states the same results in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def attention_case(name, B, S, Hq, Hk, Dqk, Dv, doc=0, prefix=False, pad=False, cap=0.0, alibi=False, train=True):
    """doc: mean document length (0: plain causal, without a mask); prefix: prompts at the front of the
    documents that all of their document sees; pad: rows end with padding."""
    return dict(op="attention", name=name, B=B, S=S, Hq=Hq, Hk=Hk, Dqk=Dqk, Dv=Dv, doc=doc, prefix=prefix, pad=pad,
                cap=cap, alibi=alibi, train=train)


def documents_case(name, B, S, doc, prefix=False, pad=False):
    return dict(op="documents", name=name, B=B, S=S, doc=doc, prefix=prefix, pad=pad)


def embedding_case(name, T, V, H, dtype="bf16", scale=1.0, pad=0.0):
    """pad: the share of tokens that are one and the same id (the separator or padding token)."""
    return dict(op="embedding", name=name, T=T, V=V, H=H, dtype=dtype, scale=scale, pad=pad)


def routing_case(name, T, E, k, score="softmax", bias=False, groups=1, top_groups=1, renorm=True, scale=1.0,
                 dtype="bf16", train=True):
    return dict(op="routing", name=name, T=T, E=E, k=k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                renorm=renorm, scale=scale, dtype=dtype, train=train)


def listed():
    return [
        # evaluation of one short packed row with the latent attention heads of the smallest example model: latency
        attention_case("attention_eval_64", 1, 64, 4, 4, 40, 32, doc=20, cap=30.0, train=False),
        # a training step of a small model: ragged length, distance bias, short documents, padding
        attention_case("attention_train_alibi_500", 4, 500, 6, 6, 64, 64, doc=120, pad=True, alibi=True),
        # the hybrid benchmark model's latent attention (head widths 64 + 32 and 64) over packed documents
        attention_case("attention_train_latent_1024", 16, 1024, 12, 12, 96, 64, doc=300),
        # the grouped-query benchmark model's attention (16 / 8 heads of 128), packed documents, capped scores
        attention_case("attention_train_capped_2048", 8, 2048, 16, 8, 128, 128, doc=700, cap=50.0),
        # one long document per row, four query heads on one key head, its prompt visible both ways
        attention_case("attention_train_prefix_16384", 1, 16384, 4, 1, 128, 128, doc=12000, prefix=True),
        # masks of one micro-batch of the example configuration, and of a batch of long rows
        documents_case("documents_512", 4, 512, 90, pad=True),
        documents_case("documents_32768", 8, 32768, 900, prefix=True),
        # embeddings of the smallest example model's micro-batch: latency
        embedding_case("embedding_256x128", 256, 100315, 128, "f32", scale=128 ** 0.5, pad=0.1),
        # the grouped-query benchmark model's micro-batch (8 x 2048 tokens), scaled by the root of the width
        embedding_case("embedding_16384x2048", 16384, 128354, 2048, "bf16", scale=2048 ** 0.5, pad=0.05),
        # the hybrid benchmark model's router, evaluation of one short batch: latency
        routing_case("routing_eval_256x32", 256, 32, 4, train=False),
        # the fine-grained expert benchmark model's router (64 experts, 8 a token) in a training step
        routing_case("routing_train_16384x64", 16384, 64, 8, score="sigmoid", bias=True, scale=2.5),
        # many experts in groups, sigmoid scores with a selection bias, of which four groups take part
        routing_case("routing_train_grouped_32768x256", 32768, 256, 8, score="sigmoid", bias=True, groups=8,
                     top_groups=4, scale=2.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "documents", "embedding", "routing"])
    if op == "attention":
        Dqk, Dv = rng.choice([(40, 32), (64, 64), (80, 64), (96, 64), (128, 128), (128, 64), (32, 32), (112, 112)])
        Hk = rng.choice([1, 2, 3, 4, 8])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        S = _log(rng, 1, 4096)
        B = max(1, min(rng.choice([1, 2, 3, 8, 16]), 2 ** 28 // (Hq * S * S)))
        doc = rng.choice([0, max(1, S // 9), max(1, S // 3), 2 * S])
        return attention_case(None, B, S, Hq, Hk, Dqk, Dv, doc, doc > 0 and rng.random() < 0.4,
                              doc > 0 and rng.random() < 0.5, rng.choice([0.0, 0.0, 20.0, 50.0]), rng.random() < 0.3,
                              rng.random() < 0.8)
    if op == "documents":
        S = _log(rng, 1, 32768)
        return documents_case(None, rng.choice([1, 3, 4, 8]), S, max(1, S // rng.choice([1, 4, 30, 100])),
                              rng.random() < 0.5, rng.random() < 0.5)
    if op == "embedding":
        return embedding_case(None, _log(rng, 1, 16384), _log(rng, 50, 128354), 8 * _log(rng, 4, 256),
                              rng.choice(["bf16", "bf16", "f32"]), rng.choice([1.0, 16.0, 0.3]),
                              rng.choice([0.0, 0.1, 0.7]))
    groups = rng.choice([1, 1, 2, 4, 8])
    E = groups * _log(rng, 2, 256 // groups)
    top_groups = rng.randint(1, groups)
    k = rng.randint(1, min(16, top_groups * (E // groups)))
    return routing_case(None, _log(rng, 1, 32768), E, k, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.6, groups,
                        top_groups, rng.random() < 0.7, rng.choice([1.0, 2.5]), rng.choice(["bf16", "f32"]),
                        rng.random() < 0.8)


# ------------------------------------------------------------------ inputs
def _layout(case, seed):
    """Document ids (negative: padding) and prompt flags of a batch, numpy [B, S]."""
    rng = np.random.default_rng([seed, 17])
    B, S = case["B"], case["S"]
    doc = np.zeros((B, S), np.int64)
    flag = np.zeros((B, S), bool)
    for b in range(B):
        used = S - (int(rng.integers(0, S // 4 + 1)) if case["pad"] else 0)
        n = int(2 * used / max(1, case["doc"])) + 16
        lens = 1 + rng.exponential(max(0, case["doc"] - 1), n).astype(np.int64)
        while lens.sum() < used:
            lens = np.concatenate([lens, 1 + rng.exponential(max(0, case["doc"] - 1), n).astype(np.int64)])
        ids = np.repeat(np.arange(len(lens)), lens)[:used]
        starts = np.repeat(np.cumsum(lens) - lens, lens)[:used]
        prompt = np.repeat((lens * rng.uniform(0.0, 0.6, len(lens))).astype(np.int64), lens)[:used]
        doc[b, :used], doc[b, used:] = ids, -1
        flag[b, :used] = np.arange(used) - starts < prompt
    return doc, flag


def _pairs(case):
    """Visible (query, key) pairs of one query head: the mean of three layouts of this case."""
    S = case["S"]
    if not case["doc"]:
        return case["B"] * S * (S + 1) // 2
    n = 0
    for seed in range(3):
        lo, hi = _ranges(*(torch.from_numpy(x) for x in _layout(case, seed)), case["prefix"])
        n += int((hi - lo).sum())
    return max(1, n // 3)


def _zipf(case):
    p = 1.0 / (np.arange(case["V"]) + 2.7)
    p *= (1.0 - case["pad"]) / p.sum()
    p[0] += case["pad"]
    return p


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 11)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    st = {"case": case}
    if case["op"] in ("attention", "documents"):
        if case["doc"]:
            doc, flag = _layout(case, seed)
            st["doc"] = torch.from_numpy(doc).to(dev)
            st["prefix"] = torch.from_numpy(flag).to(dev) if case["prefix"] else None
    if case["op"] == "attention":
        B, S, Hq, Hk, Dqk, Dv = (case[n] for n in ("B", "S", "Hq", "Hk", "Dqk", "Dv"))
        # projections of normalised activations: about unit values, sharper where scores are capped
        sharp = 2.0 if case["cap"] else 1.0
        bf = torch.bfloat16
        if Dqk == Dv:
            # the fused projection's output, q | k | v heads
            std = torch.ones((Hq + 2 * Hk) * Dqk, device=dev)
            std[:(Hq + Hk) * Dqk] = sharp
            st["qkv"] = (normal(B, S, (Hq + 2 * Hk) * Dqk) * std).to(bf)
            st["leaves"] = [st["qkv"]]
        else:
            st["q"] = normal(B, S, Hq, Dqk, std=sharp, dtype=bf)
            st["k"] = normal(B, S, Hk, Dqk, std=sharp, dtype=bf)
            st["v"] = normal(B, S, Hk, Dv, dtype=bf)
            st["leaves"] = [st["q"], st["k"], st["v"]]
        st["do"] = normal(B, S, Hq * Dv, dtype=bf)
        st["scale"] = 1.0 / math.sqrt(Dqk)
        st["slopes"] = None
        if case["alibi"]:
            st["slopes"] = torch.exp2(-8.0 * (torch.arange(Hq, device=dev, dtype=torch.float32) + 1) / Hq)
        for t in st["leaves"]:
            t.requires_grad_(case["train"])
    elif case["op"] == "embedding":
        dt = DTYPES[case["dtype"]]
        cdf = torch.from_numpy(np.cumsum(_zipf(case))).to(dev)
        rank = torch.searchsorted(cdf, torch.rand(case["T"], generator=g, device=dev, dtype=torch.float64))
        st["ids"] = torch.randperm(case["V"], generator=g, device=dev)[rank.clamp_(max=case["V"] - 1)]
        st["w"] = normal(case["V"], case["H"], std=0.02, dtype=dt).requires_grad_(True)
        st["dy"] = normal(case["T"], case["H"], std=1e-2, dtype=dt)
    elif case["op"] == "routing":
        T, E = case["T"], case["E"]
        skew = normal(1, E, std=0.5)  # some experts are liked more
        st["logits"] = (normal(T, E) + skew).to(DTYPES[case["dtype"]]).requires_grad_(case["train"])
        st["bias"] = normal(E, std=0.05 if case["score"] == "sigmoid" else 0.5 / E) if case["bias"] else None
        st["dtopw"] = normal(T, case["k"], std=1e-2)
        st["dusage"] = normal(E, std=1e-2)
    return st


# ------------------------------------------------------------------ plain forms
def _ranges(doc, prefix, use_prefix):
    """First visible key and the one past the last of every token, int32 [B, S]."""
    B, S = doc.shape
    pos = torch.arange(S, device=doc.device).expand(B, S)
    start = torch.ones_like(doc, dtype=torch.bool)
    start[:, 1:] = doc[:, 1:] != doc[:, :-1]
    lo = torch.where(start, pos, torch.zeros_like(pos)).cummax(1).values
    hi = pos + 1
    if use_prefix:
        # the next token that is not flagged, or starts a document, after each token
        stop = torch.where(start | ~prefix, pos, torch.full_like(pos, S))
        after = torch.cat([stop[:, 1:], torch.full_like(pos[:, :1], S)], 1).flip(1).cummin(1).values.flip(1)
        end = torch.where(prefix, after, pos).gather(1, lo)
        hi = torch.maximum(hi, end)
    pad = doc < 0
    return lo.masked_fill(pad, 0).int(), hi.masked_fill(pad, 0).int()


def _plain_attention(st):
    case = st["case"]
    B, S, Hq, Hk, Dqk, Dv = (case[n] for n in ("B", "S", "Hq", "Hk", "Dqk", "Dv"))
    G = Hq // Hk
    if "qkv" in st:
        x = st["qkv"].detach().float()
        q, k, v = x.split([Hq * Dqk, Hk * Dqk, Hk * Dqk], -1)
    else:
        q, k, v = (st[n].detach().float() for n in ("q", "k", "v"))
    # [B, Hk, G * S, D] queries against [B, Hk, S, D] keys
    q = q.reshape(B, S, Hk, G, Dqk).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * S, Dqk)
    k = k.reshape(B, S, Hk, Dqk).transpose(1, 2).contiguous()
    v = v.reshape(B, S, Hk, Dv).transpose(1, 2).contiguous()
    pos = torch.arange(S, device=q.device)
    if case["doc"]:
        lo, hi = _ranges(st["doc"], st["prefix"], case["prefix"])
        hidden = (pos < lo[..., None]) | (pos >= hi[..., None])
    else:
        hidden = (pos > pos[:, None]).expand(B, S, S)
    hidden = hidden[:, None, None]
    u = torch.matmul(q * st["scale"], k.transpose(2, 3))
    if case["cap"]:
        u = torch.tanh_(u.div_(case["cap"]))
        s = u * case["cap"]
    else:
        s = u
    s = s.view(B, Hk, G, S, S)
    if case["alibi"]:
        s = s - st["slopes"].view(Hk, G, 1, 1) * (pos[:, None] - pos).abs()
    s = s.masked_fill(hidden, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    del s
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, Hk, G * S, S)
    o = torch.matmul(p, v)

    def out(t, H):  # [B, Hk, .., S, D] -> [B, S, H * D]
        return t.reshape(B, H, S, -1).transpose(1, 2).reshape(B, S, -1).to(torch.bfloat16)

    if not case["train"]:
        return [out(o, Hq)]
    do = st["do"].float().reshape(B, S, Hk, G, Dv).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * S, Dv)
    dv = torch.matmul(p.transpose(2, 3), do)
    dz = torch.matmul(do, v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    del p
    if case["cap"]:
        dz = dz.mul_(u.square_().neg_().add_(1.0))
    del u
    dq = torch.matmul(dz, k) * st["scale"]
    dk = torch.matmul(dz.transpose(2, 3), q) * st["scale"]
    if "qkv" in st:
        return [out(o, Hq), torch.cat([out(dq, Hq), out(dk, Hk), out(dv, Hk)], -1)]
    return [out(o, Hq), out(dq, Hq).view(B, S, Hq, Dqk), out(dk, Hk).view(B, S, Hk, Dqk), out(dv, Hk).view(B, S, Hk, Dv)]


def _plain_embedding(st):
    w, ids, dy, scale = st["w"].detach(), st["ids"], st["dy"], st["case"]["scale"]
    y = (w[ids].float() * scale).to(w.dtype)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device).index_add_(0, ids, dy.double())
    return [y, dw.mul_(scale).to(w.dtype)]


def _plain_routing(st):
    case, x = st["case"], st["logits"].detach()
    T, E, k, G = (case[n] for n in ("T", "E", "k", "groups"))
    # the choice in 64 bits: scores at the border of it may be a rounding apart
    x64 = x.double()
    b64 = torch.softmax(x64, -1) if case["score"] == "softmax" else torch.sigmoid(x64)
    if st["bias"] is not None:
        b64 = b64 + st["bias"].double()
    if G > 1:
        per = b64.view(T, G, E // G)
        rank = per.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        best = rank.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        taken = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, best, True)
        b64 = per.masked_fill(~taken[..., None], -math.inf).view(T, E)
    topi = b64.sort(dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
    s = torch.softmax(x.float(), -1) if case["score"] == "softmax" else torch.sigmoid(x.float())
    sel = s.gather(1, topi)
    norm = sel.sum(-1, keepdim=True) if case["renorm"] else torch.ones_like(sel[:, :1])
    topw = sel / norm * case["scale"]
    total = s.sum(-1, keepdim=True)
    usage = (s / total).double().mean(0).float()
    counts = torch.zeros(E, dtype=torch.int32, device=x.device)
    counts.index_add_(0, topi.view(-1), torch.ones(T * k, dtype=torch.int32, device=x.device))
    if not case["train"]:
        return [topi, topw, usage, counts]
    dsel = st["dtopw"] * case["scale"] / norm
    if case["renorm"]:
        dsel = dsel - (dsel * sel).sum(-1, keepdim=True) / norm
    ds = torch.zeros_like(s).scatter_(1, topi, dsel)
    gu = st["dusage"] / T
    ds = ds + (gu - (gu * s).sum(-1, keepdim=True) / total) / total
    if case["score"] == "softmax":
        dx = s * (ds - (s * ds).sum(-1, keepdim=True))
    else:
        dx = ds * s * (1 - s)
    return [topi, topw, usage, counts, dx.to(x.dtype)]


# ------------------------------------------------------------------ the framework's operators
def _own(st):
    from oxidizr_b200.ops import api
    case = st["case"]
    if case["op"] == "documents":
        m = api.document_mask(st["doc"], prefix=st["prefix"])
        return [m.lo, m.hi]
    if case["op"] == "attention":
        mask = api.document_mask(st["doc"], prefix=st["prefix"]) if case["doc"] else None
        kw = dict(mask=mask, softcap=case["cap"], alibi=st["slopes"])
        if "qkv" in st:
            o = api.attention_qkv(st["qkv"], case["Hq"], case["Hk"], case["Dqk"], st["scale"], **kw)
        else:
            o = api.attention(st["q"], st["k"], st["v"], st["scale"], **kw).flatten(2)
        if not case["train"]:
            return [o]
        return [o.detach(), *torch.autograd.grad(o, st["leaves"], st["do"])]
    if case["op"] == "embedding":
        y = api.embedding(st["ids"], st["w"], scale=case["scale"])
        return [y.detach(), *torch.autograd.grad(y, st["w"], st["dy"])]
    topi, topw, usage, counts = api.route_topk(
        st["logits"], case["k"], score=case["score"], bias=st["bias"], groups=case["groups"],
        top_groups=case["top_groups"], renorm=case["renorm"], scale=case["scale"])
    if not case["train"]:
        return [topi, topw, usage, counts]
    (dx,) = torch.autograd.grad((topw, usage), st["logits"], (st["dtopw"], st["dusage"]))
    return [topi, topw.detach(), usage.detach(), counts, dx]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "documents":
        return list(_ranges(state["doc"], state["prefix"], state["case"]["prefix"]))
    if op == "attention":
        return _plain_attention(state)
    return _plain_embedding(state) if op == "embedding" else _plain_routing(state)


def work(case):
    if case["op"] == "documents":
        n = case["B"] * case["S"]
        return {"bytes": n * (8 + 8 + (1 if case["prefix"] else 0)), "flops": 0}
    if case["op"] == "attention":
        B, S, Hq, Hk, Dqk, Dv = (case[n] for n in ("B", "S", "Hq", "Hk", "Dqk", "Dv"))
        qkv = Hq * Dqk + Hk * (Dqk + Dv)
        per_pair = 2 * (Dqk + Dv)
        row = 2 * (qkv + Hq * Dv)
        if case["train"]:
            per_pair += 2 * (3 * Dqk + 2 * Dv)
            row += 2 * (qkv + Hq * Dv)
        masks = 0 if not case["doc"] else 8 + (1 if case["prefix"] else 0)
        return {"bytes": B * S * (row + masks), "flops": _pairs(case) * Hq * per_pair}
    if case["op"] == "embedding":
        T, V, H = case["T"], case["V"], case["H"]
        size = 2 if case["dtype"] == "bf16" else 4
        touched = float((1.0 - np.power(1.0 - _zipf(case), T)).sum())
        return {"bytes": int(8 * T + H * size * (touched + 2 * T + V)), "flops": 2 * T * H}
    T, E, k = case["T"], case["E"], case["k"]
    size = 2 if case["dtype"] == "bf16" else 4
    n = T * E * size + T * k * 12 + 8 * E
    if case["train"]:
        n += T * E * size + T * k * 4 + 4 * E
    return {"bytes": n, "flops": T * E * (20 if case["train"] else 10)}


# ------------------------------------------------------------------ in 64 bits
def _exact_attention(st):
    case = st["case"]
    B, S, Hq, Hk, Dqk, Dv = (case[n] for n in ("B", "S", "Hq", "Hk", "Dqk", "Dv"))
    if "qkv" in st:
        x = st["qkv"].detach().double()
        q, k, v = (t.reshape(B, S, -1, Dqk) for t in x.split([Hq * Dqk, Hk * Dqk, Hk * Dqk], -1))
    else:
        q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    do = st["do"].double().view(B, S, Hq, Dv)
    i = torch.arange(S, device=q.device)
    o, dq, dk, dv = (torch.zeros_like(t) for t in (do, q, k, v))
    for b in range(B):
        sees = i[:, None] >= i
        if case["doc"]:
            d = st["doc"][b]
            # documents are runs of one id here, and ids do not come back
            same = (d[:, None] == d) & (d >= 0)[:, None]
            if case["prefix"]:
                first = torch.searchsorted(torch.where(d < 0, d.max() + 1, d), d.clamp(min=0))
                unflagged = torch.cumsum((~st["prefix"][b]).long(), 0)
                in_prompt = st["prefix"][b] & (unflagged == unflagged[first])
                sees = sees | in_prompt[None, :]
            sees = same & sees
        for h in range(Hq):
            with torch.enable_grad():
                qh, kh, vh = (t.detach().clone().requires_grad_(True) for t in
                              (q[b, :, h], k[b, :, h * Hk // Hq], v[b, :, h * Hk // Hq]))
                a = st["scale"] * (qh @ kh.T)
                if case["cap"]:
                    a = case["cap"] * torch.tanh(a / case["cap"])
                if case["alibi"]:
                    a = a - st["slopes"][h].double() * (i[:, None] - i).abs()
                a = a.masked_fill(~sees, -1e300)
                lse = torch.where(sees.any(-1, keepdim=True), torch.logsumexp(a, -1, keepdim=True), 0.0)
                p = torch.exp(a - lse)
                oh = p @ vh
                grads = torch.autograd.grad(oh, (qh, kh, vh), do[b, :, h]) if case["train"] else None
            o[b, :, h] = oh.detach()
            if grads:
                dq[b, :, h] = grads[0]
                dk[b, :, h * Hk // Hq] += grads[1]
                dv[b, :, h * Hk // Hq] += grads[2]
            del a, lse, p, oh, grads
    o = o.flatten(2)
    if not case["train"]:
        return [o]
    if "qkv" in st:
        return [o, torch.cat([dq.flatten(2), dk.flatten(2), dv.flatten(2)], -1)]
    return [o, dq, dk, dv]


def _exact_embedding(st):
    w, ids, scale = st["w"].detach().double(), st["ids"], st["case"]["scale"]
    order = torch.argsort(ids, stable=True)
    sums = torch.zeros(ids.numel() + 1, w.shape[1], dtype=torch.float64, device=w.device)
    sums[1:] = torch.cumsum(st["dy"].double()[order], 0)
    v = torch.arange(w.shape[0] + 1, device=w.device)
    edge = torch.searchsorted(ids[order], v)
    return [w[ids] * scale, (sums[edge[1:]] - sums[edge[:-1]]) * scale]


def _exact_routing(st):
    case = st["case"]
    with torch.enable_grad():
        x = st["logits"].detach().double().requires_grad_(True)
        s = torch.exp(x) if case["score"] == "softmax" else 1.0 / (1.0 + torch.exp(-x))
        share = s / s.sum(-1, keepdim=True)
        if case["score"] == "softmax":
            s = share
        b = s.detach() + (0.0 if st["bias"] is None else st["bias"].double())
        T, E = b.shape
        n = E // case["groups"]
        if case["groups"] > 1:
            two = torch.topk(b.view(T, -1, n), min(2, n), -1).values.sum(-1)
            # a group's place: how many are better, or as good and before it
            g = torch.arange(case["groups"], device=b.device)
            ahead = (two[:, None, :] > two[:, :, None]) | ((two[:, None, :] == two[:, :, None]) & (g < g[:, None]))
            b = torch.where((ahead.sum(-1) < case["top_groups"]).repeat_interleave(n, -1), b, -math.inf)
        picks = []
        for _ in range(case["k"]):
            best = b.amax(-1, keepdim=True)
            e = torch.where(b == best, torch.arange(E, device=b.device), E).amin(-1, keepdim=True)
            b = b.scatter(1, e, -math.inf)
            picks.append(e)
        topi = torch.cat(picks, 1)
        sel = s.gather(1, topi)
        topw = sel * case["scale"]
        if case["renorm"]:
            topw = topw / sel.sum(-1, keepdim=True)
        usage = share.mean(0)
        counts = torch.bincount(topi.reshape(-1), minlength=E).int()
        res = [topi, topw.detach(), usage.detach(), counts]
        if case["train"]:
            res += torch.autograd.grad((topw, usage), x, (st["dtopw"].double(), st["dusage"].double()))
    return res


def _exact_documents(case, seed):
    doc, flag = _layout(case, seed)
    lo, hi = np.zeros(doc.shape, np.int32), np.zeros(doc.shape, np.int32)
    for b, row in enumerate(doc):
        edges = np.concatenate([[0], 1 + np.flatnonzero(row[1:] != row[:-1]), [len(row)]])
        for a, e in zip(edges[:-1], edges[1:]):
            if row[a] >= 0:
                prompt = int(np.cumprod(flag[b, a:e]).sum()) if case["prefix"] else 0
                lo[b, a:e] = a
                hi[b, a:e] = np.maximum(np.arange(a, e) + 1, a + prompt)
    return [torch.from_numpy(lo).cuda(), torch.from_numpy(hi).cuda()]


def exact(case, seed):
    if case["op"] == "documents":
        return _exact_documents(case, seed)
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(st)
    return _exact_embedding(st) if case["op"] == "embedding" else _exact_routing(st)
