"""Paged key / value cache of a decoder: appending new tokens (with the position rotation on the way) and attention of one
or a few new tokens per sequence over the cache.  GPU: csrc/kernels/paged_append.hip, csrc/kernels/paged_attention.hip
through csrc/bind/decode_ops.cpp; CPU tensors: plain PyTorch fp32 (also the oracle in tests).

The cache of a layer is two tensors ``k_pages``, ``v_pages`` [pages, page, kv_heads, D] (bf16 or fp16; views of one
buffer are fine as long as D is contiguous, strides are multiples of 8 and the slots of a page lie within 2 GB, 16 MB apart
at most).  Sequence ``b`` keeps position ``p`` in slot
``p % page`` of page ``table[b, p // page]``; ``table`` is int32 [B, width], so a sequence holds at most ``width * page``
tokens.  ``lens`` (int32 [B], on the device) is the number of tokens kept BEFORE a step: both operators take the same
``lens`` within one step, and the caller adds to it afterwards (one token per step, or what ``ops.draft.verify_draft``
accepted plus one - the rejected tokens' slots are simply written again).

* An entry of ``table`` outside [0, pages) is no page: nothing is written there and its positions are invisible.  Unused
  entries hold -1.
* ``lens[b] < 0`` marks an idle row of the batch: nothing is appended, its queries see nothing.
* Positions at or beyond ``width * page`` are dropped.
* Two sequences may share pages they only read; a page that is appended to belongs to one sequence.
* What lies in slots nobody has written (NaN included) does not reach any result.

Everything runs on the current stream of the tensors' device, allocates only through PyTorch and reads no device value on
the host, so a decode step can be captured in a hipGraph and replayed while ``lens`` advances.  Neither operator has a
gradient; tensors that require one are refused outside torch.no_grad(), and so are tensors with a forward-mode tangent.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _loader

_BIND = None


def _bind():
    global _BIND
    _BIND = _loader.bind()
    return _BIND


def rope_tables(positions: int, rot: int, base: float = 10000.0,
                device: Union[str, torch.device] = "cpu") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos, sin (fp32 [positions, rot / 2]) of the angles p * base^(-2 j / rot); the angles are computed in 64 bits
    (at position 10^5 a 32-bit product is off by 4e-3 rad)."""
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def _rotate_reference(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    rot = 2 * cos.shape[-1]
    xf = x.to(cos.dtype)
    a, b = (xf[..., 0:rot:2], xf[..., 1:rot:2]) if interleaved else (xf[..., : rot // 2], xf[..., rot // 2 : rot])
    c, s = cos[:, None], sin[:, None]
    u, w = a * c - b * s, a * s + b * c
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, xf[..., rot:]), -1)


def paged_append_reference(k, v, k_pages, v_pages, table, lens, q=None, cos=None, sin=None, starts=None,
                           interleaved: bool = False) -> Optional[torch.Tensor]:
    """Token by token on any device (host loop); cos / sin may be 64-bit, then so is the maths."""
    B, width = table.shape
    pages, page = k_pages.shape[:2]
    T = k.shape[0]
    qo = torch.zeros(q.shape, dtype=q.dtype, device=q.device) if q is not None else None
    if B == 0 or T == 0:
        return qo
    kept, tab = lens.tolist(), table.tolist()
    ends = starts.tolist() if starts is not None else [T // B * i for i in range(B + 1)]
    for b in range(B):
        for t in range(max(ends[b], 0), min(ends[b + 1], T)):
            pos = kept[b] + t - ends[b]
            if kept[b] < 0 or pos >= width * page:
                continue
            kt = k[t]
            if cos is not None:
                kt = _rotate_reference(k[t : t + 1], cos[pos : pos + 1], sin[pos : pos + 1], interleaved)[0].to(k.dtype)
                if q is not None:
                    qo[t] = _rotate_reference(q[t : t + 1], cos[pos : pos + 1], sin[pos : pos + 1], interleaved)[0].to(q.dtype)
            elif q is not None:
                qo[t] = q[t]
            pid = tab[b][pos // page]
            if 0 <= pid < pages:
                k_pages[pid, pos % page] = kt
                v_pages[pid, pos % page] = v[t]
    return qo


def _check_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor) -> None:
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages are [pages, page, kv_heads, D] of one shape")
    if k_pages.dtype not in (torch.bfloat16, torch.float16) or v_pages.dtype != k_pages.dtype:
        raise ValueError("the cache is bf16 or fp16")
    if table.dtype != torch.int32 or lens.dtype != torch.int32 or table.dim() != 2 or lens.shape != table.shape[:1]:
        raise ValueError("table is int32 [B, width], lens int32 [B]")
    if not all(_loader.packed(t, -1) for t in (k_pages, v_pages, table, lens)):
        raise ValueError("the last dimensions of the cache, of table and of lens have to be contiguous")


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor, q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                 interleaved: bool = False) -> Optional[torch.Tensor]:
    """Write the keys and values of T new tokens into the cache, in place, behind the ``lens`` tokens each sequence keeps.

    k, v: [T, kv_heads, D]; without ``starts`` the T = B * n tokens are n per sequence in order, with ``starts`` (int32
    [B + 1], non-decreasing, on the device) sequence b owns the tokens starts[b] .. starts[b + 1] (tokens outside belong to
    nobody: a padded token batch).  ``cos``, ``sin``: fp32 [P, rot / 2], P >= width * page (``rope_tables``): the first
    ``rot`` dimensions of every key are rotated by its position, as pairs (d, d + rot / 2) or, ``interleaved``,
    (2 d, 2 d + 1).  ``q`` [T, heads, D]: the queries of the same tokens, rotated alike and returned as a new tensor
    (zeros for tokens of nobody, of idle rows and beyond the table); ``q`` itself is left as it is.  Dimensions of k, v
    and q may be strided (slices of a fused projection), the last one contiguous.  D % 8 == 0, rot % 16 == 0."""
    if k.is_cuda:
        return (_BIND or _bind()).paged_append(k, v, k_pages, v_pages, table, lens, q, cos, sin, starts, interleaved,
                                               _loader.raw_stream(k.get_device()))
    _check_cache(k_pages, v_pages, table, lens)
    B, width = table.shape
    page, hkv, D = k_pages.shape[1:]
    dt = k_pages.dtype
    if k.dim() != 3 or k.shape != v.shape or k.shape[1] != hkv or k.shape[2] != D:
        raise ValueError("k and v are [T, kv_heads, D] with the cache's heads and D")
    T = k.shape[0]
    if k.dtype != dt or v.dtype != dt or not (_loader.packed(k, 2) and _loader.packed(v, 2)):
        raise ValueError("k and v have the cache's type and a contiguous last dimension")
    if D % 8 != 0 or hkv == 0:
        raise ValueError("D is a multiple of 8, the cache has heads")
    _loader.no_gradient(k, v, k_pages, v_pages, q, cos, sin)
    if any(x is not None and x.device != k.device for x in (v, k_pages, v_pages, table, lens, q, cos, sin, starts)):
        raise ValueError("all tensors live on one device")
    if q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[1] == 0 or q.shape[2] != D or q.dtype != dt or not _loader.packed(q, 2)):
        raise ValueError("q is [T, heads, D] of the cache's type and device with a contiguous last dimension")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        rot = 2 * cos.shape[-1]
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < width * page or rot > D or rot % 16 != 0:
            raise ValueError("cos and sin are [P, rot / 2] with P >= width * page, rot <= D and rot % 16 == 0")
    if starts is not None:
        if starts.dtype != torch.int32 or starts.shape != (B + 1,) or not _loader.packed(starts, 0):
            raise ValueError("starts is int32 [B + 1] on the cache's device")
    elif (T % B if B else T) != 0:
        raise ValueError("without starts every sequence has the same number of new tokens")
    return paged_append_reference(k, v, k_pages, v_pages, table, lens, q, cos, sin, starts, interleaved)


def paged_attention_reference(q, k_pages, v_pages, table, lens, scale: Optional[float] = None, causal: bool = True,
                              dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sequence by sequence in ``dtype``: (o [B, n, heads, D], log-sum-exp [B, n, heads])."""
    B, n, hq, D = q.shape
    pages, page, hkv, _ = k_pages.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros((B, n, hq, D), dtype=dtype, device=q.device)
    lse = torch.full((B, n, hq), -math.inf, dtype=dtype, device=q.device)
    cap = table.shape[1] * page
    for b in range(B):
        kept = int(lens[b])
        for i in range(n):
            seen = 0 if kept < 0 else min(kept + (i + 1 if causal else 0), cap)
            pos = torch.arange(seen, device=q.device)
            pid = table[b].long()[pos // page]
            ok = (pid >= 0) & (pid < pages)
            pid, slot = pid[ok], (pos % page)[ok]
            if pid.numel() == 0:
                continue
            k = k_pages[pid, slot].to(dtype).permute(1, 2, 0).contiguous()        # [hkv, D, keys]
            v = v_pages[pid, slot].to(dtype).permute(1, 0, 2).contiguous()        # [hkv, keys, D]
            x = torch.matmul(q[b, i].to(dtype).reshape(hkv, hq // hkv, D), k) * scale
            lse[b, i] = torch.logsumexp(x, -1).reshape(hq)
            o[b, i] = torch.matmul(torch.softmax(x, -1), v).reshape(hq, D)
            o[b, i, torch.isneginf(lse[b, i])] = 0.0                              # no score above -inf: nothing seen
    return o, lse


_DEAL: Tuple[Optional[int], int] = (None, 0)
"""(workgroups to deal all tiles out to, least tiles of a part) in place of the rule in csrc/bind/decode_ops.cpp: for tests and
sweeps."""


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                    scale: Optional[float] = None, causal: bool = True, max_len: Optional[int] = None,
                    return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of n new tokens per sequence over the paged cache.  q: [B, n, heads, D] (strides free, D contiguous;
    heads a multiple of kv_heads: query head h reads key head h // (heads / kv_heads)); returns a contiguous [B, n, heads,
    D] tensor of q's type, with ``return_lse`` also the log-sum-exp of the scaled scores, fp32 [B, n, heads].

    ``causal``: token i of a sequence sees the positions up to its own, lens[b] + i (its key is in the cache already:
    ``paged_append`` ran with the same ``lens``).  Not causal: every query sees exactly the lens[b] kept positions
    (cross-attention over encoder tokens held in pages).  A query that sees nothing, or only scores of -inf, gives 0 and a
    log-sum-exp of -inf.
    ``max_len``: an upper bound of the positions any query sees, when the caller knows a tighter one than ``width * page``
    (only used to choose how the work is split; lengths are read on the device).  D is 64 or 128, page % 16 == 0, ``scale``
    (None: D^-1/2) a number of either sign up to 2e38."""
    if q.is_cuda:
        return (_BIND or _bind()).paged_attention(q, k_pages, v_pages, table, lens, scale, causal, max_len, return_lse, *_DEAL,
                                                  _loader.raw_stream(q.get_device()))
    _check_cache(k_pages, v_pages, table, lens)
    if q.dim() != 4 or q.dtype != k_pages.dtype or not _loader.packed(q, 3):
        raise ValueError("q is [B, n, heads, D] of the cache's type with a contiguous last dimension")
    B, n, hq, D = q.shape
    page, hkv, kD = k_pages.shape[1:]
    if table.shape[0] != B or kD != D or hkv == 0 or hq % hkv != 0:
        raise ValueError("q, table and cache disagree: one table row per sequence, D alike, heads a multiple of kv_heads")
    if page % 16 != 0 or page == 0 or D not in (64, 128):
        raise ValueError("page is a multiple of 16, D is 64 or 128")
    if scale is not None and not abs(scale) <= 2e38:
        raise ValueError("scale is a number of at most 2e38")
    _loader.no_gradient(q, k_pages, v_pages)
    if any(x.device != q.device for x in (k_pages, v_pages, table, lens)):
        raise ValueError("all tensors live on one device")
    o, lse = paged_attention_reference(q, k_pages, v_pages, table, lens, scale, causal)
    return (o.to(q.dtype), lse) if return_lse else o.to(q.dtype)
