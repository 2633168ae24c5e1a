"""Device-dispatching op API used by the models.

bf16 CUDA tensors run the sm_100a kernels (``ops.fused`` and friends); CPU
tensors (and non-bf16 CUDA tensors, e.g. an f32 model moved to the GPU) run
the PyTorch statement of the same math from ``ops.reference`` under autograd.

Upstream: RMSNorm model.rs:9-32, gated RMSNorm mamba2.rs:185-217, Mamba2 LayerNorm
mamba2.rs:768, RoPE model.rs:68-117, SwiGLU model.rs:430-455, attention model.rs:333-386 and
model.rs:196-256, lm_head model.rs:1002.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import reference as R


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and t.dtype == torch.bfloat16


def embedding(ids: torch.Tensor, w: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """w[ids] * scale for integer ids of any shape and w [V, H].  bf16 and f32 weights on the GPU run
    csrc/embed.cu; there an id outside [0, V) gives a zero row, no gradient, and a bounds error in the
    status word (``ops._C.check_status``)."""
    if ids.dtype not in (torch.int64, torch.int32) or w.dim() != 2 or ids.device != w.device:
        raise ValueError(f"embedding: int64 or int32 ids and w [V, H] on one device, got {ids.dtype} on {ids.device}, "
                         f"{list(w.shape)} on {w.device}")
    ids = ids.long()
    if w.is_cuda and w.dtype in (torch.bfloat16, torch.float32):
        from .fused import Embedding
        return Embedding.apply(ids, w, float(scale))
    y = F.embedding(ids, w)
    return y if scale == 1.0 else (y.to(R.wide(w.dtype)) * scale).to(w.dtype)


def rmsnorm(x, w, eps: float = 1e-5):
    if _native(x):
        from .fused import Norm
        return Norm.apply(x, None, w, None, 0, eps)
    return R.rmsnorm(x, w, eps)


def rmsnorm_resid(x, w, eps: float = 1e-5):
    """(rmsnorm(x, w), x) where the second output is the residual stream to add back after
    the sublayer: on the GPU its gradient is added inside the norm backward kernel."""
    if _native(x):
        from .fused import NormResid
        return NormResid.apply(x, w, None, 0, eps)
    return rmsnorm(x, w, eps), x


def layernorm_resid(x, w, b, eps: float = 1e-6):
    """(layernorm(x, w, b), x), the residual stream passing through like rmsnorm_resid."""
    if _native(x):
        from .fused import NormResid
        return NormResid.apply(x, w, b, 1, eps)
    return layernorm(x, w, b, eps), x


def layernorm(x, w, b, eps: float = 1e-6):
    if _native(x):
        from .fused import Norm
        return Norm.apply(x, None, w, b, 1, eps)
    return R.layernorm(x, w, b, eps)


def gated_rmsnorm(y, gate, w, eps: float = 1e-6):
    if _native(y):
        from .fused import Norm
        return Norm.apply(y, gate, w, None, 2, eps)
    return R.gated_rmsnorm(y, gate, w, eps)


class _SplitCols(torch.autograd.Function):
    """Column blocks of a projection output as views; the backward writes the block
    gradients into ONE buffer (a single concatenation) instead of the per-slice
    zero-fill + copy + sum that autograd does for plain slicing."""

    @staticmethod
    def forward(ctx, p, sizes):
        ctx.sizes, ctx.shape, ctx.dtype = sizes, p.shape, p.dtype
        outs, o = [], 0
        for n in sizes:
            outs.append(p.narrow(-1, o, n))
            o += n
        return tuple(outs)

    @staticmethod
    def backward(ctx, *grads):
        lead = ctx.shape[:-1]
        parts = [torch.zeros(*lead, n, dtype=ctx.dtype, device=grads[0].device if grads[0] is not None else None)
                 if g is None else g.to(ctx.dtype) for g, n in zip(grads, ctx.sizes)]
        return torch.cat(parts, -1), None


def split_cols(p, sizes):
    """``p[..., a:b]`` blocks of widths ``sizes`` (summing to p's last dim)."""
    assert sum(sizes) == p.shape[-1], (sizes, p.shape)
    if p.requires_grad and torch.is_grad_enabled():
        return _SplitCols.apply(p, tuple(sizes))
    outs, o = [], 0
    for n in sizes:
        outs.append(p[..., o:o + n])
        o += n
    return tuple(outs)


def linear(x, w, bias=None, resid=None):
    if _native(x):
        from .fused import Linear
        return Linear.apply(x, w, bias, resid)
    y = F.linear(x, w.to(x.dtype), None if bias is None else bias.to(x.dtype))
    return y if resid is None else resid + y


def qkv_rope(x, w_qkv, cos, sin, hd: int, q_cols: int, k_cols: int):
    """x W_qkv^T with rotate-half RoPE applied to the q and k heads.
    cos/sin are [S, hd/2] f32 tables; token rows are [B*S] in sequence order."""
    if _native(x) and hd in (64, 128):
        from .fused import LinearRope
        return LinearRope.apply(x, w_qkv, cos, sin, hd, q_cols, k_cols)
    y = F.linear(x, w_qkv.to(x.dtype))
    B, S = x.shape[0], x.shape[1]
    q = y[..., :q_cols].reshape(B, S, -1, hd).transpose(1, 2)
    k = y[..., q_cols:q_cols + k_cols].reshape(B, S, -1, hd).transpose(1, 2)
    q = R.apply_rope(q, cos[:S], sin[:S]).transpose(1, 2).reshape(B, S, q_cols)
    k = R.apply_rope(k, cos[:S], sin[:S]).transpose(1, 2).reshape(B, S, k_cols)
    return torch.cat([q, k, y[..., q_cols + k_cols:]], -1)


def attention_rope(x, w_qkv, cos, sin, nh: int, kvh: int, hd: int, scale: float, **scores):
    """Causal GQA attention from the block input: qkv_rope + attention_qkv in one autograd
    node whose backward un-rotates dq / dk inside the flash backward.  ``scores``: a mask, cap
    or slopes for ``attention_qkv`` (then the projection and the attention are two nodes)."""
    from .attention import native_ok
    S = x.shape[1]
    if not scores and _native(x) and hd in (64, 128) and native_ok(hd) and cos.shape[0] >= S and x.shape[-1] % 8 == 0:
        from .fused import AttentionQKVRope
        return AttentionQKVRope.apply(x, w_qkv, cos, sin, nh, kvh, hd, scale)
    qkv = qkv_rope(x, w_qkv, cos, sin, hd, nh * hd, kvh * hd)
    return attention_qkv(qkv, nh, kvh, hd, scale, causal=True, **scores)


def mla_qkv(qc, kv, rp, cos, sin, nh: int, hd: int, dr: int):
    """MLA attention operands (model.rs:196-256): q = [q_c, rope(q_rope)], k = [k_c, rope(k_rope)]
    with the one k_rope of a token shared by every head, and v, from q_c [B, S, nh*hd],
    kv [B, S, 2*nh*hd] (k | v) and the rope block rp [B, S, dr + nh*dr] (k_rope | q_rope).
    Returns q, k [B, S, nh, hd + dr] and v [B, S, nh, hd]."""
    B, S = qc.shape[0], qc.shape[1]
    if _native(qc) and hd % 8 == 0 and dr % 2 == 0 and dr <= 64:
        from .mla import MlaPack
        return MlaPack.apply(qc, kv, rp, cos, sin, nh, hd, dr)
    k_r = rp[..., :dr].reshape(B, S, 1, dr)
    q_r = rp[..., dr:].reshape(B, S, nh, dr)
    q_r = R.apply_rope(q_r.transpose(1, 2), cos[:S], sin[:S]).transpose(1, 2)
    k_r = R.apply_rope(k_r.transpose(1, 2), cos[:S], sin[:S]).transpose(1, 2)
    q = torch.cat([qc.view(B, S, nh, hd), q_r.to(qc.dtype)], -1)
    k = torch.cat([kv[..., :nh * hd].view(B, S, nh, hd), k_r.to(kv.dtype).expand(B, S, nh, dr)], -1)
    return q, k, kv[..., nh * hd:].view(B, S, nh, hd)


def swiglu_mlp(x, w_gu, w_down, resid=None):
    """resid + down(silu(gate x) * up x); w_gu rows interleaved [g 128 | u 128]..."""
    I = w_gu.shape[0] // 2
    if _native(x) and I % 128 == 0:
        from .fused import SwiGLUMLP
        return SwiGLUMLP.apply(x, w_gu, w_down, resid)
    gu = F.linear(x, w_gu.to(x.dtype))
    nb = I // 128 if I % 128 == 0 else None
    if nb:
        gu = gu.reshape(*gu.shape[:-1], nb, 2, 128)
        g, u = gu[..., 0, :].reshape(*x.shape[:-1], I), gu[..., 1, :].reshape(*x.shape[:-1], I)
    else:
        g, u = gu[..., :I], gu[..., I:]
    y = F.linear(F.silu(g) * u, w_down.to(x.dtype))
    return y if resid is None else resid + y


def document_mask(tokens, separator=None, pad=None, prefix=None, causal: bool = True):
    """Visible keys of a batch of packed documents, for the attention of every layer.

    tokens [B, S]: document ids (a document is a run of one id; negative ids are padding), or, with
    ``separator``, token ids whose documents end with that token (``pad``: a token id that is padding).
    ``prefix`` (bool [B, S]): the leading flagged run of each document is visible to all of it.
    """
    from .doc_attention import document_mask as _dm
    return _dm(tokens, separator, pad, prefix, causal)


def attention(q, k, v, scale: float, causal: bool = True, mask=None, softcap: float = 0.0, alibi=None):
    """q [B, S, Hq, Dqk], k [B, S, Hk, Dqk], v [B, S, Hk, Dv] -> [B, S, Hq, Dv].  ``mask`` from
    document_mask, ``softcap`` c: scores pass through c tanh(./c), ``alibi`` f32 [Hq]: slopes of a bias
    -slope |i - j| added after the cap."""
    from .doc_attention import attention as _doc, takes_plain
    if mask is None and not softcap and alibi is None:
        same = k.dtype == v.dtype == q.dtype and k.shape == (*q.shape[:2], k.shape[2], q.shape[3]) and v.shape[:3] == k.shape[:3]
        train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
        if not (same and takes_plain(q, q.shape[2], k.shape[2], q.shape[3], v.shape[3], scale, causal, train, (k, v))):
            from .attention import attention as _att
            return _att(q, k, v, scale, causal)
    return _doc(q, k, v, scale, causal, mask, softcap or 0.0, alibi)


def attention_qkv(qkv, Hq: int, Hk: int, D: int, scale: float, causal: bool = True, mask=None, softcap: float = 0.0,
                  alibi=None):
    """``attention`` from the fused [B, S, (Hq + 2 Hk) D] projection; returns [B, S, Hq D]."""
    from .doc_attention import attention_qkv as _doc, takes_plain
    if mask is None and not softcap and alibi is None and not takes_plain(
            qkv, Hq, Hk, D, D, scale, causal, torch.is_grad_enabled() and qkv.requires_grad):
        from .attention import attention_qkv as _aq
        return _aq(qkv, Hq, Hk, D, scale, causal)
    return _doc(qkv, Hq, Hk, D, scale, causal, mask, softcap or 0.0, alibi)


def route_topk(logits, k: int, score: str = "softmax", bias=None, groups: int = 1, top_groups: int = 1,
               group_top: int = 2, renorm: bool = True, scale: float = 1.0):
    """Choose k of E experts per token from router logits [T, E].

    s = softmax or sigmoid of the logits.  The choice goes by s + ``bias`` ([E], the choice alone: it has
    no gradient and is not in the weights): with ``groups`` > 1 the ``top_groups`` groups of neighbouring
    experts with the largest sum of their ``group_top`` best take part, and of those the k best experts,
    largest first; of equals the lowest index.  Weights are s of the chosen, divided by their sum with
    ``renorm``, times ``scale``.

    Returns (topi [T, k] int64, topw [T, k] f32, usage [E] f32: the mean over the tokens of s / sum s,
    counts [E] int32); topw and usage carry gradients to the logits.
    """
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"route_topk: logits must be floating point [T, E], got {logits.dtype} {list(logits.shape)}")
    E = logits.shape[1]
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"route_topk: score must be softmax or sigmoid, got {score!r}")
    if groups < 1 or E % groups or not 1 <= top_groups <= groups or group_top < 1:
        raise ValueError(f"route_topk: {E} experts in {groups} groups of which {top_groups} stay (ranked by their "
                         f"{group_top} best)")
    if not 1 <= k <= top_groups * (E // groups):
        raise ValueError(f"route_topk: cannot choose {k} of {top_groups * (E // groups)} experts")
    if bias is not None:
        if bias.shape != (E,) or bias.device != logits.device:
            raise ValueError(f"route_topk: bias must be one value per expert [{E}] on {logits.device}")
        bias = bias.detach().float().contiguous()
    if logits.is_cuda:
        from .moe_kernels import RouterTopK, router_ok
        if router_ok(logits, k, groups):
            return RouterTopK.apply(logits, k, score, bias, groups, top_groups, group_top, bool(renorm), float(scale))
    return R.route_topk(logits, k, score, bias, groups, top_groups, group_top, renorm, scale)


def linear_cross_entropy(x, w, targets, ignore_index: int = -100):
    if _native(x):
        from .fused import LinearCrossEntropy
        return LinearCrossEntropy.apply(x, w, targets, ignore_index)
    logits = F.linear(x, w.to(x.dtype))
    return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), targets.reshape(-1).long(),
                           ignore_index=ignore_index)


def causal_conv1d(x, w, b, act: bool = True):
    """x [B, S, C] channels-last; w [C, 1, k]; b [C]."""
    if _native(x):
        from .ssm import causal_conv1d_cuda
        return causal_conv1d_cuda(x, w, b, act)
    return R.causal_conv1d(x, w, b, act)
