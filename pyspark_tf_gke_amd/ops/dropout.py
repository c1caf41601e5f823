"""Dropout drawn from a counter-based generator (csrc/kernels/dropout.hip, rng.h).

The mask is a pure function of ``(seed, step, element index)`` and is never stored: the backward pass
draws it again.  Element ``i`` of the mask takes the ``i & 7``-th 16-bit piece of Philox4x32-10
(Salmon et al., SC11) at counter ``(i >> 3, step)`` under the 64-bit ``seed``; it is dropped when the
piece is below ``round(rate * 65536)``, so the rate is exact to 2**-17, and what is kept is scaled by
the inverse of that exact keep probability.  Dropped elements are 0 whatever the input holds.

``step`` is a host integer or a one-element int64 device tensor that the kernel reads (a captured HIP
graph then draws another mask every replay, see :func:`drop_advance`).

``noise_shape`` (Keras): the shape of the mask, 1 on ONE run of axes that share an entry, e.g. ``(N, 1, 1, C)``
or ``(N, 1)``.  None on an axis is the input's own size there, ``(None, 1, 1, None)`` an entry for each
sample and channel; None in place of the shape draws an entry per element.  GPU tensors run the kernel,
CPU tensors the reference below.
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple

import torch

from ._util import hip_on, on_device, ptr

_M64 = (1 << 64) - 1
_CALL = struct.Struct("=3Q7qd")  # DropCall of dropout.hip


class Drop(NamedTuple):
    """A dropout inside a fused operator: rate, 64-bit seed, step (int or int64 device tensor), and the mask
    index of the tensor's first element (a part of a larger tensor draws that part of its mask)."""

    rate: float
    seed: int
    step: object = 0
    first: int = 0


def threshold(rate: float) -> tuple[int, float]:
    """(threshold of the 16-bit pieces, scale of what is kept)."""
    if not 0.0 <= rate <= 1.0:  # also refuses NaN
        raise ValueError(f"dropout: rate must lie in [0, 1], got {rate}")
    thr = int(round(rate * 65536))
    return thr, 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def _signed(v: int) -> int:
    v = int(v) & _M64
    return v - (1 << 64) if v >> 63 else v


def step_args(step, device) -> tuple:
    """(host step, device step tensor or None), checked."""
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1:
            raise TypeError("dropout: a step tensor must hold one int64")
        if step.device != device:
            raise ValueError(f"dropout: step lives on {step.device}, the data on {device}")
        return 0, step
    return _signed(step), None


def mix_seed(seed: int, stream: int) -> int:
    """A 64-bit seed of its own for each (seed, stream): the SplitMix64 finaliser (Steele, Lea, Flood,
    OOPSLA 2014) over seed + (stream + 1) * golden ratio."""
    z = (int(seed) + (int(stream) + 1) * 0x9E3779B97F4A7C15) & _M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _M64
    return z ^ (z >> 31)


def noise_dims(shape, noise_shape) -> tuple[int, int, int]:
    """(outer, mid, inner) of ``shape`` whose mask is shared over mid."""
    if noise_shape is None:
        return math.prod(shape), 1, 1
    outer, mid, inner = 1, 1, 1
    run = 0  # 0 before, 1 in, 2 behind the shared axes
    again = False
    if len(noise_shape) != len(shape):
        raise ValueError(f"dropout: noise_shape {tuple(noise_shape)} does not broadcast to {tuple(shape)}")
    for s, v in zip(shape, noise_shape):
        if v is None or v == s:
            if run == 1 and s != 1:
                run = 2
            if run == 0:
                outer *= s
            else:
                inner *= s
        elif v == 1:
            again = again or run == 2
            run = 1
            mid *= s
        else:
            raise ValueError(f"dropout: noise_shape {tuple(noise_shape)} does not broadcast to {tuple(shape)}")
    if again:
        raise NotImplementedError(f"dropout: noise_shape {tuple(noise_shape)} shares two separate runs of axes of "
                                  f"{tuple(shape)}")
    return (outer, mid, inner) if mid > 1 else (outer * mid * inner, 1, 1)


def _pieces(blocks, step: int, seed: int):
    """[len(blocks), 8] 16-bit pieces (int64): the host reference of rng.h."""
    lo = 0xFFFFFFFF
    step &= _M64
    seed &= _M64
    c0, c1 = blocks & lo, (blocks >> 32) & lo
    c2 = torch.full_like(blocks, step & lo)
    c3 = torch.full_like(blocks, step >> 32)
    k0, k1 = seed & lo, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # wraps; the masks below read the right bits
        c0, c1, c2, c3 = (((p1 >> 32) & lo) ^ c1 ^ k0, p1 & lo, ((p0 >> 32) & lo) ^ c3 ^ k1, p0 & lo)
        k0, k1 = (k0 + 0x9E3779B9) & lo, (k1 + 0xBB67AE85) & lo
    w = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((w & 0xFFFF, w >> 16), 2).reshape(len(blocks), 8)


def keep_mask(shape, rate: float, seed: int, step, noise_shape=None, first: int = 0) -> torch.Tensor:
    """The bool mask (host reference), of ``shape``, from mask index ``first`` on."""
    thr, _ = threshold(rate)
    outer, mid, inner = noise_dims(shape, noise_shape)
    n = outer * inner
    step = int(step)
    lo = first // 8
    p = _pieces(torch.arange(lo, (first + n + 7) // 8, dtype=torch.int64), step, int(seed))
    p = p.reshape(-1)[first - 8 * lo:first - 8 * lo + n]
    return (p >= thr).view(outer, 1, inner).expand(outer, mid, inner).reshape(tuple(shape))


def _run(name, x, rate, seed, step, out, noise_shape):
    thr, scale = threshold(rate)
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float32:
        raise TypeError(f"{name}: expected bfloat16 or float32, got {dt}")
    if out.dtype is not dt or out.shape != x.shape or out.device != x.device:
        raise ValueError(f"{name}: output must match the input's shape, dtype and device")
    if not x.is_contiguous() or not out.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")
    mid, inner = (1, 1) if noise_shape is None else noise_dims(x.shape, noise_shape)[1:]
    host, dev = step_args(step, x.device)
    if not x.is_cuda:
        keep = keep_mask(x.shape, rate, seed, step, noise_shape)
        out.copy_(torch.where(keep, x.float() * scale, 0.0).to(dt))
        return out
    xp, op, n, f32 = x.data_ptr(), out.data_ptr(), x.numel(), dt is torch.float32
    if xp != op and abs(xp - op) < n * (4 if f32 else 2):
        raise ValueError(f"{name}: input and output overlap")
    hip_on(x.device, "ptg_dropout",
           _CALL.pack(xp, op, 0 if dev is None else dev.data_ptr(), n, f32, thr, _signed(seed), host, mid, inner, scale))
    return out


def dropout_fwd(x, rate: float, seed: int, step, out, noise_shape=None):
    """out = keep ? x * scale : 0, bf16 or fp32, ``out`` may be ``x``."""
    return _run("dropout_fwd", x, rate, seed, step, out, noise_shape)


def dropout_bwd(dy, rate: float, seed: int, step, dx, noise_shape=None):
    """dx = keep ? dy * scale : 0 with the mask of the forward call of the same seed, step and shape."""
    return _run("dropout_bwd", dy, rate, seed, step, dx, noise_shape)


def drop_advance(step):
    """step += 1 for a device-resident step (a kernel, so a captured graph advances it every replay)."""
    if step.dtype != torch.int64 or step.numel() != 1:
        raise TypeError("drop_advance: step must hold one int64")
    if not on_device(step):
        step += 1
        return step
    hip_on(step.device, "ptg_drop_advance", ptr(step))
    return step
