"""Linear layers with 4-bit weights and group scales, for the few rows of a decode step.  GPU: csrc/kernels/int4_linear.hip
through csrc/bind/decode_ops.cpp; CPU tensors: plain PyTorch fp32 on the dequantized weights (also the oracle).

``quantize_int4`` (from a float weight) or ``pack_int4`` (from codes, scales and zeros made elsewhere) lays a layer's weights
out once; ``linear_int4`` is then called like ``ops.conv.linear_bf16``.  Weight (n, k) is (code - zero) * scale with codes
0 .. 15 and one scale (and zero, 8 if none are given) per row and group of G = 32, 64 or 128 input features."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _loader
from .conv import _act_ref

_ACTS = {"none": 0, "relu": 1, "gelu": 3}
GROUPS = (32, 64, 128)


@dataclass
class Int4Weight:
    """A layer's weights in the kernels' order.  words: int32 [N / 16, K / 128, 64, 4] (sizes rounded up; lane 16 g + r,
    word i holds row r of its 16 and the features 32 i + 8 g .. + 8 of its 128, code 2 p in bits 4 p, code 2 p + 1 in bits
    16 + 4 p); scale: [K / G, N rounded up to 16] bf16 or fp16; zero: uint8 alike, or None (8)."""

    words: torch.Tensor
    scale: torch.Tensor
    zero: Optional[torch.Tensor]
    n: int
    k: int
    group: int

    def to(self, device) -> "Int4Weight":
        return Int4Weight(self.words.to(device), self.scale.to(device), None if self.zero is None else self.zero.to(device),
                          self.n, self.k, self.group)

    def codes(self) -> torch.Tensor:
        """uint8 [N, K]."""
        nt, ks = self.words.shape[:2]
        sh = torch.tensor([4 * (j >> 1) + 16 * (j & 1) for j in range(8)], dtype=torch.int32, device=self.words.device)
        c = ((self.words[..., None] >> sh) & 15).to(torch.uint8)                   # [nt, ks, 64, 4, 8]
        c = c.view(nt, ks, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5)                  # nt, r, ks, i, g, j
        return c.reshape(nt * 16, ks * 128)[: self.n, : self.k].contiguous()

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """[N, K]."""
        c = self.codes().to(dtype).view(self.n, self.k // self.group, self.group)
        z = 8.0 if self.zero is None else self.zero[:, : self.n].t().to(dtype)[..., None]
        return ((c - z) * self.scale[:, : self.n].t().to(dtype)[..., None]).reshape(self.n, self.k)


def pack_int4(packed: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None) -> Int4Weight:
    """packed: uint8 [N, K / 2], feature 2 j in the low and 2 j + 1 in the high four bits of byte j; scale: [N, K / G] bf16 or
    fp16; zero: uint8 [N, K / G] or None (8)."""
    if packed.dim() != 2 or packed.dtype != torch.uint8 or scale.dim() != 2 or scale.shape[0] != packed.shape[0]:
        raise ValueError("packed is uint8 [N, K / 2], scale [N, K / G]")
    N, K = packed.shape[0], 2 * packed.shape[1]
    groups = scale.shape[1]
    G = K // groups if groups else 0
    if N == 0 or G not in GROUPS or G * groups != K:
        raise ValueError("K is a multiple of the group size, which is 32, 64 or 128")
    if scale.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("scales are bf16 or fp16")
    if zero is not None and (zero.shape != scale.shape or zero.dtype != torch.uint8):
        raise ValueError("zero is uint8 of the scales' shape")
    nt, ks = (N + 15) // 16, (K + 127) // 128
    p = torch.zeros((nt * 16, ks * 64), dtype=torch.uint8, device=packed.device)
    p[:N, : K // 2] = packed
    # byte m of a word's four holds features (2 m, 2 m + 1): low nibbles to bits 4 m, high ones to 16 + 4 m
    p = p.view(nt, 16, ks, 4, 4, 4).permute(0, 2, 4, 1, 3, 5)                      # nt, ks, g, r, i, byte
    lo, hi = p & 15, p >> 4
    by = torch.stack((lo[..., 0] | (lo[..., 1] << 4), lo[..., 2] | (lo[..., 3] << 4),
                      hi[..., 0] | (hi[..., 1] << 4), hi[..., 2] | (hi[..., 3] << 4)), -1).contiguous()
    words = by.view(torch.int32).reshape(nt, ks, 64, 4)
    pad = lambda t: torch.nn.functional.pad(t.t(), (0, nt * 16 - N)).contiguous()  # noqa: E731
    return Int4Weight(words, pad(scale), None if zero is None else pad(zero), N, K, G)


def quantize_int4(weight: torch.Tensor, group: int = 128, symmetric: bool = True,
                  scale_dtype: torch.dtype = torch.bfloat16) -> Int4Weight:
    """Round-to-nearest codes of a float weight [N, K].  Symmetric: zero 8, the scale as small as -8 .. 7 allow; otherwise
    the group's range (with 0 in it) on 0 .. 15.  Codes are taken with the scale as it is stored."""
    if weight.dim() != 2 or group not in GROUPS or weight.shape[1] % group != 0:
        raise ValueError("weight is [N, K] with K a multiple of the group size 32, 64 or 128")
    N, K = weight.shape
    w = weight.detach().float().view(N, K // group, group)
    hi, lo = w.amax(-1).clamp(min=0.0), w.amin(-1).clamp(max=0.0)
    s = torch.maximum(hi / 7.0, -lo / 8.0) if symmetric else (hi - lo) / 15.0
    s = s.to(scale_dtype)
    if not bool(torch.isfinite(s).all()):
        raise ValueError("weights are finite and their scales fit scale_dtype")
    s = torch.where(s > 0, s, torch.ones_like(s))                                  # groups of zeros, or of less than a scale can say
    sf = s.float()
    z = torch.full_like(sf, 8.0) if symmetric else (-lo / sf).round().clamp(0, 15)
    c = ((w / sf[..., None]).round() + z[..., None]).clamp(0, 15).to(torch.uint8).view(N, K)
    return pack_int4(c[:, 0::2] | (c[:, 1::2] << 4), s, None if symmetric else z.to(torch.uint8))


def linear_int4_reference(x, w: Int4Weight, bias=None, act: str = "none", res=None) -> torch.Tensor:
    y = x.float() @ w.dequantize().t()
    if bias is not None:
        y = y + bias.float()
    if res is not None:
        y = y + res.float()
    return _act_ref(y, act)


_SHAPE = None
"""(tiles of 16 outputs a wave holds, waves over outputs, waves over K, parts of K over workgroups) in place of the rule in
csrc/bind/decode_ops.cpp: for tests and sweeps."""
_BIND = None


def _bind():
    global _BIND
    _BIND = _loader.bind()
    return _BIND


def linear_int4(x: torch.Tensor, w: Int4Weight, bias: Optional[torch.Tensor] = None, *, act: str = "none",
                res: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = act(x @ W^T + bias (+ res)) in x's type.  x: [..., K] bf16 or fp16, bias: fp32 [N], res: [..., N] of x's type;
    act: none, relu, gelu.  Products are exact and summed in fp32, rounded once.  No gradient: x, scales, bias and res that require
    one are refused outside torch.no_grad(), and so are those with a forward-mode tangent."""
    code = _ACTS.get(act)
    if code is None:
        raise ValueError("act is none, relu or gelu")
    if x.is_cuda:
        return (_BIND or _bind()).linear_int4(x, w.words, w.scale, w.zero, w.n, w.k, w.group, bias, code, res, _SHAPE,
                                              _loader.raw_stream(x.get_device()))
    if x.dim() == 0 or x.shape[-1] != w.k or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("x is [..., K] bf16 or fp16")
    if bias is not None and (bias.shape != (w.n,) or bias.dtype != torch.float32 or not _loader.packed(bias, 0)):
        raise ValueError("bias is fp32 [N]")
    if res is not None and (res.shape[:-1] != x.shape[:-1] or res.shape[-1] != w.n or res.dtype != x.dtype):
        raise ValueError("res is [..., N] of x's type")
    _loader.no_gradient(x, w.scale, bias, res)
    if any(t is not None and t.device != x.device for t in (w.words, bias, res)):
        raise ValueError("all tensors live on one device")
    return linear_int4_reference(x, w, bias, act, res).to(x.dtype)
