"""Causal attention over packed documents: visible key ranges, capped scores, a distance bias.

A block of training tokens holds several documents one after another.  ``document_mask`` turns a
batch into the range of keys that each token sees: its own document up to itself, or, for a
document that opens with a prompt, at least that prompt.  Attention over it is

    z_ij = scale q_i . k_j,  u = cap tanh(z / cap) (without a cap: z),  a = u - slope_h |i - j|
    o_i  = sum_{lo_i <= j < hi_i} softmax(a_i)_j v_j

and a token that sees nothing (padding) gets zeros and passes no gradient on.  What padding rows of
q, k, v and the output's gradient hold does not matter, not even NaN.

bf16 CUDA tensors with head widths that are multiples of 8 up to 128 run csrc/doc_attn_fwd.cu and
csrc/doc_attn_bwd.cu (autograd nodes in csrc/ops.cpp, first derivatives only); everything else runs the
statement of the same math in ``ops.reference``.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import reference as R
from ._C import ext, status

MAX_SEQ = 1 << 18  # DOC_MAX_SEQ of csrc/kernels_doc.h: the bit masks of a row stay in shared memory


@dataclass(frozen=True)
class DocMask:
    """Visible keys of a batch: token i of row b sees keys ``lo[b, i] <= j < hi[b, i]`` (int32 [B, S]).

    On CUDA ``qt`` / ``kt`` are the tile tables that the kernels walk.  One mask serves every layer
    of the step it was built for.
    """
    lo: torch.Tensor
    hi: torch.Tensor
    qt: Optional[torch.Tensor]
    kt: Optional[torch.Tensor]
    causal: bool

    def tensors(self):
        return [self.lo, self.hi, self.qt, self.kt]


def document_mask(tokens: torch.Tensor, separator: Optional[int] = None, pad: Optional[int] = None,
                  prefix: Optional[torch.Tensor] = None, causal: bool = True) -> DocMask:
    if tokens.dim() != 2 or tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"document_mask: tokens must be int64 or int32 [B, S], got {tokens.dtype} "
                         f"{list(tokens.shape)}")
    if pad is not None and separator is None:
        raise ValueError("document_mask: pad goes with a separator; document ids mark padding by a negative id")
    if prefix is not None:
        if not causal:
            raise ValueError("document_mask: a prefix needs a causal mask")
        if prefix.dtype != torch.bool or prefix.shape != tokens.shape or prefix.device != tokens.device:
            raise ValueError("document_mask: prefix must be bool, of the tokens' shape and on their device")
    tokens = tokens.long()
    if tokens.is_cuda:
        if tokens.shape[1] > MAX_SEQ:
            raise ValueError(f"document_mask: rows of at most {MAX_SEQ} tokens, got {tokens.shape[1]}")
        if tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        if prefix is not None and prefix.stride(1) != 1:
            prefix = prefix.contiguous()
        lo, hi, qt, kt = ext().document_mask(tokens, prefix, separator, pad, causal)
        return DocMask(lo, hi, qt, kt, causal)
    lo, hi = R.document_ranges(tokens, separator, pad, prefix, causal)
    return DocMask(lo, hi, None, None, causal)


MAX_HEAD = 128  # csrc/doc_attn_fwd.cu: head widths are multiples of 8 up to this


def _kernel_ok(t, Dqk: int, Dv: int) -> bool:
    return (t.is_cuda and t.dtype == torch.bfloat16 and Dqk <= MAX_HEAD and Dv <= MAX_HEAD and Dqk % 8 == 0
            and Dv % 8 == 0)


# Rows of up to this many tokens, by head widths: (causal, both ways)
_FLASH_ROWS = {(64, 64): (384, 200), (96, 64): (256, 200), (128, 64): (200, 128), (128, 128): (200, 128)}
_FLASH_CTAS = 10 * 148


def _flash_layout(t) -> bool:
    """Rows that csrc/flash_attn.cu's tensor maps can address, as they are or copied; these kernels' operands are copied
    wherever they need be."""
    return t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1])


def takes_plain(t, Hq: int, Hk: int, Dqk: int, Dv: int, scale: float, causal: bool, train: bool, others=()) -> bool:
    """Whether plain attention of [B, S, ...] operands of t's type (t and the others) goes to these kernels rather than to
    csrc/flash_attn.cu (of the widths in _FLASH_ROWS) or PyTorch.

    They are the faster ones but for many short rows: forward and backward of 8 x 2048 tokens, 16 query and 8 key heads of
    128, 658 us, there 890; of 12 x 1000 tokens, 16 heads of 64, 341 and 363; but of 192 x 64 tokens 298 and 239, of
    61 x 200 265 and 224, of 32 x 384 241 and 228, because a CTA of the two backward kernels takes 4 us to start and end,
    and such rows give it little to do between.  Few such CTAs, under ten times the SMs, take less than the host
    needs for the call, which is a third less here (89 and 133 us).  Without a gradient the two differ below 64 tokens:
    768 x 16 take 189 and 173 us.  These kernels add no gradient with atomics, and keep more of dQ and dK in short
    rows (off by 0.3 % for 2 tokens, there 0.45 %; one token alone gets the exact zeros that it has here)."""
    B, S = t.shape[:2]
    if not (scale > 0 and S > 0 and 0 < Hk <= Hq <= 65535 and Hq % Hk == 0 and 0 < B <= 65535 and _kernel_ok(t, Dqk, Dv)):
        return False
    rows = _FLASH_ROWS.get((Dqk, Dv))
    short = rows is not None and 1 < S <= ((rows[0] if causal else rows[1]) if train else 64)
    return not (short and B * Hq * ((S + 127) // 128) >= _FLASH_CTAS and all(map(_flash_layout, (t, *others))))


def _check(t, B, S, Hq, scale, causal, mask, softcap, alibi):
    if not scale > 0:
        raise ValueError(f"attention: scale must be positive, got {scale}")
    if not 0 <= softcap < float("inf"):
        raise ValueError(f"attention: softcap must be a positive number, or 0 for none, got {softcap}")
    if mask is not None:
        if mask.lo.shape != (B, S) or mask.lo.device != t.device:
            raise ValueError(f"attention: the mask is for {list(mask.lo.shape)} on {mask.lo.device}, "
                             f"q for {[B, S]} on {t.device}")
        if mask.lo.is_cuda and (mask.qt is None or mask.kt is None):
            raise ValueError("attention: the mask has no tile tables; document_mask makes them")
        if mask.causal != causal:
            raise ValueError(f"attention: causal={causal} with a mask built for causal={mask.causal}")
    if alibi is not None:
        if alibi.shape != (Hq,) or alibi.device != t.device:
            raise ValueError(f"attention: alibi must be one slope per query head [{Hq}] on {t.device}")
        if alibi.requires_grad:
            raise ValueError("attention: alibi slopes are constants, no gradient is computed for them")


def _reference(q, k, v, scale, causal, mask, softcap, alibi):
    lo, hi = (mask.lo, mask.hi) if mask is not None else R.plain_ranges(q.shape[0], q.shape[1], causal, q.device)
    o = R.attention_ranges(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), scale, lo, hi, softcap, alibi)
    return o.transpose(1, 2)


def _options(alibi, mask):
    return (None if alibi is None else alibi.float().contiguous()), (mask.tensors() if mask is not None else [])


def attention(q, k, v, scale: float, causal: bool = True, mask: Optional[DocMask] = None, softcap: float = 0.0,
              alibi: Optional[torch.Tensor] = None) -> torch.Tensor:
    B, S, Hq, D = q.shape
    Hk = k.shape[2]
    if k.shape != (B, S, Hk, D) or v.shape[:3] != (B, S, Hk) or Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"attention: q {list(q.shape)}, k {list(k.shape)}, v {list(v.shape)} do not go together")
    _check(q, B, S, Hq, scale, causal, mask, softcap, alibi)
    if _kernel_ok(q, D, v.shape[3]) and k.dtype == q.dtype and v.dtype == q.dtype:
        slopes, m = _options(alibi, mask)
        return ext().doc_attention(q, k, v, scale, softcap, slopes, causal, m, status(q.device))
    return _reference(q, k, v, scale, causal, mask, softcap, alibi)


def attention_qkv(qkv, Hq: int, Hk: int, D: int, scale: float, causal: bool = True, mask: Optional[DocMask] = None,
                  softcap: float = 0.0, alibi: Optional[torch.Tensor] = None) -> torch.Tensor:
    B, S, N = qkv.shape
    if Hk < 1 or Hq < 1 or Hq % Hk or N != (Hq + 2 * Hk) * D:
        raise ValueError(f"attention: qkv {list(qkv.shape)} does not hold {Hq} query and {Hk} key and value heads of {D}")
    _check(qkv, B, S, Hq, scale, causal, mask, softcap, alibi)
    if _kernel_ok(qkv, D, D):
        slopes, m = _options(alibi, mask)
        return ext().doc_attention_qkv(qkv, Hq, Hk, D, scale, softcap, slopes, causal, m, status(qkv.device))
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([Hq * D, Hk * D, Hk * D], -1))
    return _reference(q, k, v, scale, causal, mask, softcap, alibi).flatten(2)
