"""Verification of drafted tokens.  GPU: csrc/kernels/draft_verify.hip through csrc/bind/decode_ops.cpp; CPU
tensors: plain PyTorch (also the oracle).

A cheap proposal drafts n tokens, the target model scores all of them in one pass, and ``verify_draft`` keeps the longest
prefix the target agrees with plus one token of the target's own - so that the kept tokens are distributed exactly as if
the target had sampled them one by one."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _loader

MAX_DRAFTED = 63


def verify_draft_reference(draft, target, u, proposal=None, counts=None, pad: int = -1) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sequence by sequence in 64 bits."""
    B, n = draft.shape
    V = target.shape[2]
    tokens = torch.full((B, n + 1), pad, dtype=torch.int32)
    accepted = torch.zeros((B,), dtype=torch.int32)
    for b in range(B):
        c = n if counts is None else max(0, min(int(counts[b]), n))
        i = 0
        while i < c:
            x = int(draft[b, i])
            if not 0 <= x < V:
                break
            qx = 1.0 if proposal is None else float(proposal[b, i, x].double())
            if not float(u[b, i].double()) * qx < float(target[b, i, x].double()):
                break
            tokens[b, i] = x
            i += 1
        row = target[b, i].double().cpu()
        w = row
        if i < c:
            if proposal is not None:
                w = row - proposal[b, i].double().cpu()
            elif 0 <= int(draft[b, i]) < V:
                w = row.clone()
                w[int(draft[b, i])] -= 1.0
        zero = torch.zeros((), dtype=torch.float64)
        w = torch.where(w > 0, w, zero)
        if not float(w.sum()) > 0:
            w = torch.where(row > 0, row, zero)
        cdf = w.cumsum(0)
        total = float(cdf[-1])
        hit = 0
        if 0.0 < total < float("inf"):
            x = min(max(float(u[b, n].double()), 0.0), 1.0) * total if float(u[b, n]) == float(u[b, n]) else 0.0
            at = torch.nonzero((cdf > x) & (w > 0))[:, 0]
            hit = int(at[0]) if at.numel() else int(torch.nonzero(w > 0)[-1, 0])
        tokens[b, i] = hit
        accepted[b] = i
    return tokens.to(draft.device), accepted.to(draft.device)


_PIECES: Optional[int] = None
"""Workgroups per row in place of the rule in csrc/bind/decode_ops.cpp: for tests and sweeps."""
_BIND = None


def _bind():
    global _BIND
    _BIND = _loader.bind()
    return _BIND


def verify_draft(draft: torch.Tensor, target: torch.Tensor, u: torch.Tensor, proposal: Optional[torch.Tensor] = None,
                 counts: Optional[torch.Tensor] = None, pad: int = -1) -> Tuple[torch.Tensor, torch.Tensor]:
    """draft: int32 [B, n], the drafted tokens (0 <= n <= 63).  target: [B, n + 1, V] probabilities of the target model at
    the drafted positions and the one behind them; proposal: [B, n, V] probabilities the drafts were drawn from, None when
    they were chosen, not drawn (all of the proposal's probability on the drafted token).  Both bf16, fp16 or fp32, rows of
    any stride.  u: fp32 [B, n + 1] numbers in [0, 1): one per draft, the last for the sampled token.  counts: int32 [B],
    drafts that count per sequence (None: n).

    Draft i is accepted while u[i] * proposal[i, x] < target[i, x]; the first refused one is replaced by a token sampled
    from max(target[i] - proposal[i], 0), and behind ``counts`` accepted drafts one is sampled from target[counts].
    Returns (tokens int32 [B, n + 1]: accepted drafts, the sampled token, ``pad``; accepted int32 [B]).

    Sampling takes the lowest v whose cumulative weight exceeds u times the row's total, in 64 bits.  Rows need not sum to
    one.  A drafted token outside [0, V) is refused.  Where nothing remains (target <= proposal everywhere) the target's
    row is sampled itself; a row without positive finite weight gives token 0."""
    if draft.is_cuda:
        return (_BIND or _bind()).verify_draft(draft, target, u, proposal, counts, pad, _PIECES, _loader.raw_stream(draft.get_device()))
    if draft.dim() != 2 or draft.dtype != torch.int32:
        raise ValueError("draft is int32 [B, n]")
    B, n = draft.shape
    dt = target.dtype
    if n > MAX_DRAFTED:
        raise ValueError(f"at most {MAX_DRAFTED} drafted tokens")
    if target.dim() != 3 or target.shape[:2] != (B, n + 1) or dt not in (torch.bfloat16, torch.float16, torch.float32) or target.shape[2] == 0:
        raise ValueError("target is [B, n + 1, V] bf16, fp16 or fp32")
    if proposal is not None and (proposal.shape != (B, n, target.shape[2]) or proposal.dtype != dt or not _loader.packed(proposal, 2)):
        raise ValueError("proposal is [B, n, V] of the target's type, rows contiguous")
    if u.shape != (B, n + 1) or u.dtype != torch.float32 or not _loader.packed(u, 1):
        raise ValueError("u is fp32 [B, n + 1]")
    if counts is not None and (counts.shape != (B,) or counts.dtype != torch.int32 or not _loader.packed(counts, 0)):
        raise ValueError("counts is int32 [B]")
    if not (_loader.packed(target, 2) and _loader.packed(draft, 1)):
        raise ValueError("the last dimension of target and draft has to be contiguous")
    if any(x is not None and x.device != draft.device for x in (target, u, proposal, counts)):
        raise ValueError("all tensors live on one device")
    return verify_draft_reference(draft, target, u, proposal, counts, pad)
