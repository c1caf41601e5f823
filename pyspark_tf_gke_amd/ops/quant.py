"""Dense layers with 4-bit weights (csrc/kernels/quant.hip).

``w[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group])`` with codes 0..15, a bf16 scale and
an optional zero point (0..15; 8 where there is none) for every ``group`` (32, 64 or 128) of inputs.

:func:`int4_quantize` makes codes, scales and zero points from a weight matrix, :func:`int4_layout` lays
given ones out for the kernel (once, at load time), :func:`int4_dense_fwd` is the product.  GPU tensors run
the kernel, CPU tensors the fp32 reference.  Inference only: codes have no gradient.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from ._util import hip_on

GROUPS = (32, 64, 128)
_CALL = struct.Struct("=7Q6q")  # Int4Call of quant.hip
ACT = {None: 0, "linear": 0, "relu": 1}


class Int4Weight(NamedTuple):
    """Laid-out weights: tiles uint8 [N/16, K/128, 64, 16], scale bf16 and zero uint8 (or None)
    [N/16, K/128, 16, 128/group], sizes rounded up (padding has scale 0)."""

    tiles: torch.Tensor
    scale: torch.Tensor
    zero: torch.Tensor | None
    n: int
    k: int
    group: int

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.tiles, self.scale, self.zero) if t is not None)


def int4_quantize(w: torch.Tensor, group: int = 128, zero_point: bool = False):
    """(codes uint8 [N, K/2], scale bf16 [N, K/group], zero uint8 [N, K/group] or None) of a weight
    matrix [N, K]; two codes a byte, the even input in the low nibble.

    Symmetric: scale = max|w| / 7, code = round(w / scale) + 8 (1..15).  With zero points the range
    from min(w, 0) to max(w, 0) is mapped on 0..15.  Codes are rounded against the bf16 scale that is
    stored; an all-zero group has scale 0."""
    _check_group(w.shape[1] if w.dim() == 2 else 0, group, w.dim())
    if not torch.isfinite(w).all():
        raise ValueError("int4_quantize: weights must be finite")
    N, K = w.shape
    g = w.detach().float().view(N, K // group, group)
    if zero_point:
        lo, hi = g.amin(2).clamp_max(0.0), g.amax(2).clamp_min(0.0)
        width = hi - lo
        scale = _bf16_up(torch.where(torch.isfinite(width), width / 15.0, hi / 15.0 - lo / 15.0))
        zero = torch.round(_steps(-lo, scale)).clamp_(0, 15)
    else:
        scale = _bf16_up(g.abs().amax(2) / 7.0)
        zero = torch.full_like(scale, 8.0, dtype=torch.float32)
    q = (torch.round(_steps(g, scale[:, :, None])) + zero[:, :, None]).clamp_(0, 15).to(torch.uint8).view(N, K)
    return q[:, 0::2] | (q[:, 1::2] << 4), scale, zero.to(torch.uint8) if zero_point else None


def _steps(v, scale):
    """v / scale, 0 where the scale is; a scale below 2**-128 has no fp32 reciprocal."""
    s = scale.float()
    inv = torch.where(s > 0, 1.0 / s, 0.0)
    return torch.where(torch.isfinite(inv), v * inv, v / s)


def _bf16_up(t):
    """bf16, rounded up: a group's extreme value never falls outside the code range."""
    b = t.to(torch.bfloat16)
    return torch.where(b.float() < t, torch.nextafter(b, torch.full_like(b, float("inf"))), b)


def _check_group(K, group, dim=2):
    if dim != 2:
        raise ValueError("int4: weights must be a matrix [N, K]")
    if group not in GROUPS:
        raise ValueError(f"int4: group must be one of {GROUPS}, got {group}")
    if K < group or K % group:
        raise ValueError(f"int4: {K} inputs do not divide into groups of {group}")


def _check_codes(codes, scale, zero, group):
    if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.shape[0]:
        raise TypeError("int4: codes must be uint8 [N, K/2]")
    N, K = codes.shape[0], codes.shape[1] * 2
    _check_group(K, group)
    if scale.dtype != torch.bfloat16 or tuple(scale.shape) != (N, K // group) or scale.device != codes.device:
        raise ValueError(f"int4: scale must be bfloat16 [{N}, {K // group}] on {codes.device}")
    if zero is not None and (zero.dtype != torch.uint8 or zero.shape != scale.shape or zero.device != codes.device):
        raise ValueError(f"int4: zero must be uint8 [{N}, {K // group}] on {codes.device}")
    return N, K


def int4_layout(codes, scale, zero=None, group: int = 128) -> Int4Weight:
    """Lay codes [N, K/2], scales and zero points out in the kernel's tiles (a new copy)."""
    N, K = _check_codes(codes, scale, zero, group)
    if zero is not None and int(zero.max()) > 15:
        raise ValueError("int4: zero points must lie in 0..15")
    Np, Kp = -(-N // 16) * 16, -(-K // 128) * 128
    if (Np, Kp) != (N, K) or not codes.is_contiguous() or codes.storage_offset() % 4:
        padded = torch.zeros((Np, Kp // 2), dtype=torch.uint8, device=codes.device)
        padded[:N, : K // 2] = codes
        codes = padded
    # a dword of 8 inputs: the even ones' nibbles in its low half, the odd ones' in its high half, rotated
    v = codes.view(torch.int32)
    half = [v & 0x0F0F0F0F, (v >> 4) & 0x0F0F0F0F]
    half = [(h | (h >> 4)) & 0x00FF00FF for h in half]
    half = [(h | (h >> 8)) & 0xFFFF for h in half]
    words = half[0] | (half[1] << 16)
    words = (words << 3) | ((words >> 29) & 7)
    # [nt, n, kt, i, quarter] -> dword i of lane quarter * 16 + n
    words = words.view(Np // 16, 16, Kp // 128, 4, 4).permute(0, 2, 4, 1, 3).contiguous()
    tiles = words.view(torch.uint8).reshape(Np // 16, Kp // 128, 64, 16)

    def group_rows(t):
        if t is None:
            return None
        p = t.contiguous()
        if (Np, Kp) != (N, K):
            p = torch.zeros((Np, Kp // group), dtype=t.dtype, device=t.device)
            p[:N, : K // group] = t
        p = p.view(Np // 16, 16, Kp // 128, 128 // group).permute(0, 2, 1, 3)
        return p.clone(memory_format=torch.contiguous_format)

    return Int4Weight(tiles, group_rows(scale), group_rows(zero), N, K, group)


def int4_codes(w: Int4Weight):
    """(codes, scale, zero) back from the laid-out weights."""
    nt, kt = w.tiles.shape[:2]
    b = w.tiles.view(nt, kt, 64, 4, 4).long()
    words = sum(b[..., j] << (8 * j) for j in range(4))
    words = ((words >> 3) | (words << 29)) & 0xFFFFFFFF  # [nt, kt, lane, dword]
    words = words.view(nt, kt, 4, 16, 4).permute(0, 3, 1, 4, 2)  # [nt, n, kt, i, quarter]
    sh = 4 * (torch.arange(4, device=b.device)[:, None] + 4 * torch.arange(2, device=b.device)[None, :])
    q = ((words[..., None, None] >> sh) & 15).reshape(nt * 16, kt * 128)[: w.n, : w.k].to(torch.uint8)

    def rows(t):
        return None if t is None else t.permute(0, 2, 1, 3).reshape(nt * 16, -1)[: w.n, : w.k // w.group].contiguous()

    return q[:, 0::2] | (q[:, 1::2] << 4), rows(w.scale), rows(w.zero)


def int4_dequantize(w: Int4Weight) -> torch.Tensor:
    """fp32 [N, K]."""
    codes, scale, zero = int4_codes(w)
    q = torch.stack((codes & 15, codes >> 4), 2).view(w.n, w.k // w.group, w.group).float()
    z = 8.0 if zero is None else zero.float()[:, :, None]
    return ((q - z) * scale.float()[:, :, None]).view(w.n, w.k)


_WS: dict = {}


def int4_workspace_floats(batch: int, w: Int4Weight) -> int:
    """Floats of :func:`int4_workspace`."""
    key = (batch, w.n, w.k, w.group)
    v = _WS.get(key)
    if v is None:
        from .. import _native

        n = ctypes.c_long(0)
        _native.check(_native.hip_lib().ptg_int4_ws(batch, w.n, w.k, w.group, ctypes.byref(n)), "ptg_int4_ws")
        if len(_WS) > 4096:
            _WS.clear()
        v = _WS[key] = n.value
    return v


def int4_workspace(batch: int, w: Int4Weight) -> torch.Tensor | None:
    """Scratch of one product of ``batch`` rows (None where it needs none).  Products that may run at the
    same time - on two streams, or in two captured graphs - need one each."""
    if not w.tiles.is_cuda:
        return None
    n = int4_workspace_floats(batch, w)
    return torch.empty(n, dtype=torch.float32, device=w.tiles.device) if n else None


def int4_dense_fwd(x, w: Int4Weight, bias, act, out, workspace=None):
    """out[B, N] = act(x[B, K] @ w^T + bias): x bf16, bias fp32 [N] or None, act None / "linear" /
    "relu" (a NaN stays one), out bf16 or fp32, apart from x.  Infinities and NaN in x give what the formula
    gives.  Sums are fp32; the order of a sum depends on the sizes alone."""
    relu = ACT.get(act)
    if relu is None:
        raise ValueError(f"int4_dense: activation {act!r}")
    tiles, n, k = w.tiles, w.n, w.k
    dev = tiles.device
    groups = tiles.numel() * 2 // w.group
    if tiles.numel() != (n + 15) // 16 * ((k + 127) // 128) * 1024 or w.scale.numel() != groups \
            or w.scale.device != dev or (w.zero is not None and (w.zero.numel() != groups or w.zero.device != dev)):
        raise ValueError(f"int4_dense: the weight is not what int4_layout gives for [{n}, {k}], groups of {w.group}, on "
                         "one device")
    if x.dim() != 2 or x.shape[1] != k or not x.is_contiguous():
        raise ValueError(f"int4_dense: x must be contiguous [batch, {k}]")
    B = x.shape[0]
    if out.shape != (B, n) or not out.is_contiguous() or x.device != dev or out.device != dev:
        raise ValueError(f"int4_dense: out must be contiguous [{B}, {n}], everything on {dev}")
    f32 = out.dtype is torch.float32
    if not f32 and out.dtype is not torch.bfloat16:
        raise TypeError(f"int4_dense: output {out.dtype}")
    if bias is not None and (bias.dtype is not torch.float32 or bias.shape != (n,) or bias.device != dev
                             or not bias.is_contiguous()):
        raise ValueError(f"int4_dense: bias must be a contiguous fp32 [{n}] on {dev}")
    if not tiles.is_cuda:
        y = x.float() @ int4_dequantize(w).t()
        if bias is not None:
            y = y + bias
        out.copy_((torch.relu(y) if relu else y).to(out.dtype))
        return out
    if x.dtype is not torch.bfloat16:
        raise TypeError(f"int4_dense: x must be bfloat16, got {x.dtype}")
    xp, op = x.data_ptr(), out.data_ptr()
    if B and xp < op + B * n * (4 if f32 else 2) and op < xp + B * k * 2:
        raise ValueError("int4_dense: out overlaps x")
    if xp & 15:
        x = x.clone()  # the kernel reads 16 bytes at a time
        xp = x.data_ptr()
    need = int4_workspace_floats(B, w)
    wp = 0
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.float32, device=dev)
        elif workspace.dtype is not torch.float32 or workspace.numel() < need or workspace.device != dev \
                or not workspace.is_contiguous():
            raise ValueError(f"int4_dense: workspace must hold {need} contiguous floats on {dev}")
        wp = workspace.data_ptr()
    hip_on(dev, "ptg_int4_dense",
           _CALL.pack(xp, tiles.data_ptr(), w.scale.data_ptr(), 0 if w.zero is None else w.zero.data_ptr(),
                      0 if bias is None else bias.data_ptr(), op, wp, B, n, k, w.group, relu, f32))
    return out
