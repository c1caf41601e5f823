"""Residual-block norms (csrc/kernels/norm.h, norm_fwd.hip, norm_bwd.hip).

One pass joins a block's output ``x`` to the residual stream and normalises it for the next block::

    d = dropout(scale * gate * post(x));  h = res + d;  u = pre(h)

over rows of ``C`` columns (the last axis).  Every part is optional: ``post`` / ``pre`` are LayerNorm or
RMSNorm (:class:`Norm`) or None; ``gate`` is None, a vector ``[C]`` (fp32) or a row for each of ``G``
groups of consecutive rows ``[G, C]`` (the tensors' type); ``drop`` a :class:`~.dropout.Drop`; ``res`` the
stream.  Plain LayerNormalization is ``pre`` alone.  ``u`` is taken from the unrounded ``h``.

The backward pass computes ``h`` and the mask again from ``x``, ``res`` and the saved row statistics, so
``h`` need not be kept for it.  Its column sums (affine and gate gradients) are added in a fixed order:
the same inputs give the same bits.  Gradients are written, not accumulated.

Activations are bf16 or fp32, affine vectors and their gradients fp32; statistics and sums are fp32.
GPU tensors run the kernels, CPU tensors the fp32 reference below.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from . import dropout as DR
from ._util import hip_on

KINDS = {"layer": 1, "rms": 2}
MAX_COLS = 8192


# arguments of the C entries: 64 bits each, as FwdCall and BwdCall of norm.h
_FWD = struct.Struct("=11Q13q4d")
_BWD = struct.Struct("=18Q13q2d")


class Norm(NamedTuple):
    """``kind`` "layer" or "rms", ``gamma`` / ``beta`` fp32 [C] or None (1 / 0; an RMSNorm has no beta)."""

    kind: str
    gamma: torch.Tensor | None
    beta: torch.Tensor | None
    eps: float


def block_norm_stats(rows: int, device) -> torch.Tensor:
    """Row statistics a forward pass leaves for the backward: [4, rows] fp32 (mean and 1/std of x, then
    of h; an RMSNorm's mean is 0)."""
    return torch.empty((4, rows), dtype=torch.float32, device=device)


def block_norm_workspace(rows: int, cols: int, groups: int, device) -> torch.Tensor:
    """Scratch of one backward pass (partial column sums).  Passes that may run at the same time - on
    two streams, or in two captured graphs - need one each."""
    if torch.device(device).type != "cuda" or rows == 0:
        return torch.empty(0, dtype=torch.float32, device=device)
    if not 1 <= cols <= MAX_COLS:
        raise ValueError(f"block_norm: rows of 1..{MAX_COLS} columns, got {cols}")
    if groups < 1 or rows % groups:
        raise ValueError(f"block_norm: {rows} rows do not divide into {groups} gate groups")
    return torch.empty(block_norm_workspace_floats(rows, cols, groups), dtype=torch.float32, device=device)


_NO_DROP = (0, 0, 1.0, 0, 0, 0, 0)  # on, threshold, scale, seed, host step, device step's address, first index


def _bad(name, x):
    raise ValueError(f"block_norm: {name} must be contiguous and match x ({tuple(x.shape)}, {x.dtype}, {x.device})")


def _vec(t, C, dev, name):
    if t.dtype is not torch.float32:
        raise TypeError(f"block_norm: {name} must be float32, got {t.dtype}")
    if t.dim() != 1 or t.numel() != C or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"block_norm: {name} must be a contiguous [{C}] vector on the device of x")


def _norm_args(nm, C, dev, name):
    """(kind, gamma pointer, beta pointer, epsilon), checked."""
    if nm is None:
        return 0, 0, 0, 0.0
    kind, g, b, eps = nm
    kind = KINDS.get(kind)
    if kind is None:
        raise ValueError(f"block_norm: {name} kind {nm.kind!r} (layer or rms)")
    if not eps > 0.0:
        raise ValueError(f"block_norm: {name} needs an epsilon > 0, got {nm.eps}")
    if g is not None:
        _vec(g, C, dev, name + ".gamma")
        g = g.data_ptr()
    else:
        g = 0
    if b is not None:
        if kind == 2:
            raise ValueError(f"block_norm: {name}: an RMSNorm has no beta")
        _vec(b, C, dev, name + ".beta")
        b = b.data_ptr()
    else:
        b = 0
    return kind, g, b, eps


def _common(x, gate, drop):
    """(rows, columns, device index, gate mode, rows per gate row, dropout arguments), checked."""
    dt, shape, dev = x.dtype, x.shape, x.get_device()
    if dt is not torch.bfloat16 and dt is not torch.float32:
        raise TypeError(f"block_norm: expected bfloat16 or float32, got {dt}")
    if not shape or shape[-1] < 1:
        raise ValueError("block_norm: x needs at least one column")
    if not x.is_contiguous():
        raise ValueError("block_norm: x must be contiguous")
    C = shape[-1]
    M = x.numel() // C
    if C > MAX_COLS and dev >= 0:
        raise ValueError(f"block_norm: rows of at most {MAX_COLS} columns, got {C}")
    mode, rpg = 0, 1
    if gate is not None:
        if gate.dim() == 1:
            _vec(gate, C, dev, "gate")
            mode, rpg = 1, M or 1
        else:
            if gate.dim() != 2 or gate.shape[1] != C or gate.dtype is not dt or gate.get_device() != dev \
                    or not gate.is_contiguous():
                raise ValueError(f"block_norm: gate must be fp32 [{C}] or {dt} [groups, {C}], contiguous, on the "
                                 "device of x")
            G = gate.shape[0]
            if M and (G == 0 or M % G):
                raise ValueError(f"block_norm: {M} rows do not divide into {G} gate groups")
            mode, rpg = 2, M // G if G else 1
    return M, C, dev, mode, rpg, _drop_args(drop, x.device)


def _drop_args(drop, device):
    if drop is None:
        return _NO_DROP
    thr, ds = DR.threshold(drop.rate)
    host, step = DR.step_args(drop.step, device)
    first = int(drop.first)
    if not 0 <= first < 1 << 62:
        raise ValueError(f"block_norm: a mask begins at an index from 0 on, got {first}")
    return 1, thr, ds, DR._signed(drop.seed), host, 0 if step is None else step.data_ptr(), first


def _like(x, dt, dev, n, strides, t, name):
    """Data pointer of a tensor that must look like x (0 where absent)."""
    if t is None:
        return 0
    if t.dtype is not dt or t.get_device() != dev or t.numel() != n or not t.is_contiguous() \
            or (t.stride() != strides and t.shape != x.shape):
        _bad(name, x)  # contiguous, as many values, equal strides: the same rows
    return t.data_ptr()


def _apart(o, on, size, ins):
    """Output ``o`` may not overlap an input (pointer, name, whether the very same buffer will do).  A value is
    used by the thread that writes its place, and read before; the last lane of an unaligned row reads its
    neighbour's values too, so there the waves of a row meet before they write."""
    for i, name, same in ins:
        if -size < o - i < size and i and not (o == i and same):
            raise ValueError(f"block_norm: {on} overlaps {name}")


def _gate_apart(gate, outs, size):
    lo, hi = gate.data_ptr(), gate.data_ptr() + gate.numel() * gate.element_size()
    for o, on in outs:
        if lo < o + size and o < hi:
            raise ValueError(f"block_norm: {on} overlaps gate")


def _stats_ok(stats, M, dev):
    if stats.dtype is not torch.float32 or stats.shape != (4, M) or stats.get_device() != dev \
            or not stats.is_contiguous():
        raise ValueError(f"block_norm: stats must be a contiguous fp32 [4, {M}] on the device of x")


def block_norm_fwd(x, *, res=None, post=None, gate=None, scale: float = 1.0, drop=None, pre=None, h=None, u=None,
                   stats=None):
    """Writes ``h`` (if given) and ``u`` (with ``pre``); ``stats`` (:func:`block_norm_stats`) for a
    backward pass.  Returns (h, u).  ``h`` may be ``res`` or ``x``; nothing else may overlap an input."""
    M, C, dev, mode, rpg, d = _common(x, gate, drop)
    if (pre is None) != (u is None):
        raise ValueError("block_norm: u goes with pre")
    if h is None and u is None:
        raise ValueError("block_norm: nothing to write (h and u are None)")
    k1, g1, b1, e1 = _norm_args(post, C, dev, "post")
    k2, g2, b2, e2 = _norm_args(pre, C, dev, "pre")
    dt, n, st, xp = x.dtype, M * C, x.stride(), x.data_ptr()
    rp = _like(x, dt, dev, n, st, res, "res")
    hp = _like(x, dt, dev, n, st, h, "h")
    up = _like(x, dt, dev, n, st, u, "u")
    if stats is not None:
        _stats_ok(stats, M, dev)
    f32 = dt is torch.float32
    size = n * (4 if f32 else 2)
    if hp:
        _apart(hp, "h", size, ((xp, "x", True), (rp, "res", True)))
    if up:  # u is written after others have read, and h written before it
        _apart(up, "u", size, ((xp, "x", False), (rp, "res", False), (hp, "h", False)))
    if mode == 2:
        _gate_apart(gate, [(p, n) for p, n in ((hp, "h"), (up, "u")) if p], size)
    if dev < 0:
        hv, uv, st = _ref_fwd(x, res, post, gate, scale, drop, pre, M, C, rpg)
        if h is not None:
            h.copy_(hv.view(x.shape).to(h.dtype))
        if u is not None:
            u.copy_(uv.view(x.shape).to(u.dtype))
        if stats is not None:
            stats.copy_(st)
        return h, u
    gp = 0 if gate is None else gate.data_ptr()
    aligned = not ((C | d[6]) & 7 or (xp | rp | hp | up | (gp if mode == 2 else 0)) & 15)
    hip_on(x.device, "ptg_block_norm_fwd",
           _FWD.pack(xp, rp, gp, hp, up, g1, b1, g2, b2, 0 if stats is None else stats.data_ptr(), d[5], M, C, f32,
                     aligned, k1, k2, mode, rpg, d[0], d[1], d[3], d[4], d[6], e1, e2, scale, d[2]))
    return h, u


def block_norm_bwd(x, stats, *, res=None, post=None, gate=None, scale: float = 1.0, drop=None, pre=None, du=None,
                   dh=None, dx=None, dres=None, dgate=None, dpost=None, dpre=None, workspace=None):
    """Gradients of :func:`block_norm_fwd` (same x, res, post, gate, scale, drop, pre) from ``du`` (with
    ``pre``) and ``dh`` (None: zero).  ``stats`` as that call left them (None where neither norm is there).
    Writes dx and dres (None: skipped), ``dgate`` like ``gate``, and
    ``dpost`` / ``dpre`` = (dgamma, dbeta), fp32 [C] or None where the norm has none.  ``dx`` and ``dres``
    may each be one of x, res, du and dh; nothing else may overlap.  ``workspace``:
    :func:`block_norm_workspace` (None: allocated here)."""
    M, C, dev, mode, rpg, d = _common(x, gate, drop)
    if (pre is None) != (du is None):
        raise ValueError("block_norm: du goes with pre")
    if pre is None and dh is None:
        raise ValueError("block_norm: no gradient comes in (du and dh are None)")
    if dx is None and dres is None and dgate is None and dpost is None and dpre is None:
        raise ValueError("block_norm: no gradient is asked for")
    k1, g1, b1, _ = _norm_args(post, C, dev, "post")
    k2, g2, _, _ = _norm_args(pre, C, dev, "pre")
    dt, n, st, xp = x.dtype, M * C, x.stride(), x.data_ptr()
    rp = _like(x, dt, dev, n, st, res, "res")
    up = _like(x, dt, dev, n, st, du, "du")
    hp = _like(x, dt, dev, n, st, dh, "dh")
    dxp = _like(x, dt, dev, n, st, dx, "dx")
    drp = _like(x, dt, dev, n, st, dres, "dres")
    if stats is not None:
        _stats_ok(stats, M, dev)
    elif k1 or k2:
        raise ValueError("block_norm: the gradients of a norm need the forward pass's stats")
    if dgate is not None and (gate is None or dgate.shape != gate.shape or dgate.dtype is not gate.dtype
                              or dgate.get_device() != dev or not dgate.is_contiguous()):
        raise ValueError("block_norm: dgate must match gate")
    vecs = []
    for g, nm, name in ((dpost, post, "dpost"), (dpre, pre, "dpre")):
        if g is None:
            vecs += (None, None)
            continue
        for t, w, part in ((g[0], nm and nm.gamma, "gamma"), (g[1], nm and nm.beta, "beta")):
            if t is not None:
                if w is None:
                    raise ValueError(f"block_norm: {name} asks for the gradient of an absent {part}")
                _vec(t, C, dev, name)
            vecs.append(t)
    f32 = dt is torch.float32
    size = n * (4 if f32 else 2)
    ins = ((xp, "x", True), (rp, "res", True), (up, "du", True), (hp, "dh", True))
    outs = [(p, n) for p, n in ((dxp, "dx"), (drp, "dres")) if p]
    for p, name in outs:
        _apart(p, name, size, ins)
    if dxp and drp:
        _apart(drp, "dres", size, ((dxp, "dx", False),))
    if mode == 2:
        _gate_apart(gate, outs, size)
        if dgate is not None:
            _gate_apart(dgate, outs + [(p, n) for p, n, _ in ins if p], size)
            _gate_apart(dgate, [(gate.data_ptr(), "gate")], gate.numel() * gate.element_size())
    if M == 0:
        for t in (dgate, *vecs):
            if t is not None:
                t.zero_()
        return dx, dres
    if dev < 0:
        _ref_bwd(x, stats, res, post, gate, scale, drop, pre, du, dh, dx, dres, dgate, vecs, M, C, rpg)
        return dx, dres
    need = block_norm_workspace_floats(M, C, M // rpg if mode == 2 else 1)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.float32, device=x.device)
    elif workspace.dtype is not torch.float32 or workspace.get_device() != dev or workspace.numel() < need \
            or not workspace.is_contiguous():
        raise ValueError(f"block_norm: workspace must hold {need} contiguous floats on the device of x")
    if mode == 2 and dgate is None:
        dgate = torch.empty_like(gate)  # written all the same
    gp = 0 if gate is None else gate.data_ptr()
    dgp = 0 if dgate is None else dgate.data_ptr()
    bits = xp | rp | up | hp | dxp | drp
    if mode == 2:
        bits |= gp | dgp
    v = [0 if t is None else t.data_ptr() for t in vecs]
    hip_on(x.device, "ptg_block_norm_bwd",
           _BWD.pack(xp, rp, gp, up, hp, dxp, drp, g1, b1, g2, 0 if stats is None else stats.data_ptr(), *v, dgp,
                     workspace.data_ptr(), d[5], M, C, f32, not ((C | d[6]) & 7 or bits & 15), k1, k2, mode, rpg,
                     d[0], d[1], d[3], d[4], d[6], scale, d[2]))
    return dx, dres


# ---------------------------------------------------------------------------------------- without norms
# Without a norm the pass is elementwise and takes tensors of any shape: as rows of 1024 columns (four a workgroup
# of the backward pass, two of the forward), and what is left over as one row behind them, whose mask goes on where
# theirs ends.  There is nothing to sum up, so the backward pass takes no workspace.
FLAT_COLS = 1024


def _flat_parts(n):
    """(first element, rows, columns) of the launches"""
    rows, rest = divmod(n, FLAT_COLS)
    return ([(0, rows, FLAT_COLS)] if rows else []) + ([(n - rest, 1, rest)] if rest else [])


def _flat_common(x):
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float32:
        raise TypeError(f"block_norm: expected bfloat16 or float32, got {dt}")
    if not x.is_contiguous():
        raise ValueError("block_norm: x must be contiguous")
    return dt, x.get_device(), x.numel(), x.data_ptr(), x.element_size()


def _flat_like(x, dt, dev, n, t, name):
    if t is None:
        return 0
    if t.dtype is not dt or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        _bad(name, x)
    return t.data_ptr()


def flat_fwd(x, *, res=None, gate=None, scale: float = 1.0, drop=None, h):
    """h = res + dropout(scale * gate * x) over tensors of any shape, as many values in each.  ``h`` may be ``res`` or
    ``x``; nothing else may overlap.  Returns h."""
    dt, dev, n, xp, size = _flat_common(x)
    rp = _flat_like(x, dt, dev, n, res, "res")
    gp = _flat_like(x, dt, dev, n, gate, "gate")
    hp = _flat_like(x, dt, dev, n, h, "h")
    d = _drop_args(drop, x.device)
    _apart(hp, "h", n * size, ((xp, "x", True), (rp, "res", True), (gp, "gate", False)))
    if dev < 0:
        row = lambda t: None if t is None else t.reshape(1, n)  # noqa: E731
        h.copy_(_ref_fwd(row(x), row(res), None, row(gate), scale, drop, None, 1, n, 1)[0].view(h.shape).to(dt))
        return h
    for lo, M, C in _flat_parts(n):
        at = lambda p: p and p + lo * size  # noqa: E731
        aligned = not ((C | d[6]) & 7 or (at(xp) | at(rp) | at(gp) | at(hp)) & 15)
        hip_on(x.device, "ptg_block_norm_fwd",
               _FWD.pack(at(xp), at(rp), at(gp), at(hp), 0, 0, 0, 0, 0, 0, d[5], M, C, size == 4, aligned, 0, 0,
                         2 if gp else 0, 1, d[0], d[1], d[3], d[4], d[6] + lo, 0.0, 0.0, scale, d[2]))
    return h


def flat_bwd(x, *, gate=None, scale: float = 1.0, drop=None, dh, dx=None, dres=None, dgate=None):
    """Gradients of :func:`flat_fwd`, written to those of dx, dres and dgate that are given.  ``dx`` and ``dres`` may
    each be x or dh; nothing else may overlap."""
    dt, dev, n, xp, size = _flat_common(x)
    gp = _flat_like(x, dt, dev, n, gate, "gate")
    hp = _flat_like(x, dt, dev, n, dh, "dh")
    dxp = _flat_like(x, dt, dev, n, dx, "dx")
    drp = _flat_like(x, dt, dev, n, dres, "dres")
    dgp = _flat_like(x, dt, dev, n, dgate, "dgate")
    d = _drop_args(drop, x.device)
    if dh is None:
        raise ValueError("block_norm: no gradient comes in (dh is None)")
    if dx is None and dres is None and dgate is None:
        raise ValueError("block_norm: no gradient is asked for")
    if dgate is not None and gate is None:
        raise ValueError("block_norm: dgate must match gate")
    ins, bytes_ = ((xp, "x", True), (hp, "dh", True), (gp, "gate", False)), n * size
    for p, name in ((dxp, "dx"), (drp, "dres")):
        if p:
            _apart(p, name, bytes_, ins)
    if dxp and drp:
        _apart(drp, "dres", bytes_, ((dxp, "dx", False),))
    if dgp:
        outs = ((dxp, "dx", False), (drp, "dres", False))
        _apart(dgp, "dgate", bytes_, [(p, name, False) for p, name, _ in ins] + list(outs))
    if dev < 0:
        row = lambda t: None if t is None else t.view(1, n)  # noqa: E731
        _ref_bwd(row(x), None, None, None, row(gate), scale, drop, None, None, row(dh), row(dx), row(dres), row(dgate),
                 (None,) * 4, 1, n, 1)
        return
    if gate is not None and dgate is None:
        dgate = torch.empty_like(gate)  # written all the same
        dgp = dgate.data_ptr()
    for lo, M, C in _flat_parts(n):
        at = lambda p: p and p + lo * size  # noqa: E731
        aligned = not ((C | d[6]) & 7 or (at(xp) | at(gp) | at(hp) | at(dxp) | at(drp) | at(dgp)) & 15)
        hip_on(x.device, "ptg_block_norm_bwd",
               _BWD.pack(at(xp), 0, at(gp), 0, at(hp), at(dxp), at(drp), 0, 0, 0, 0, 0, 0, 0, 0, at(dgp), 0, d[5], M, C,
                         size == 4, aligned, 0, 0, 2 if gp else 0, 1, d[0], d[1], d[3], d[4], d[6] + lo, scale, d[2]))


_WS: dict = {}


def block_norm_workspace_floats(rows: int, cols: int, groups: int) -> int:
    """Floats of :func:`block_norm_workspace`."""
    key = (rows, cols, groups)
    v = _WS.get(key)
    if v is None:
        from .. import _native

        n = ctypes.c_long(0)
        _native.check(_native.hip_lib().ptg_block_norm_ws(rows, cols, groups, ctypes.byref(n)), "ptg_block_norm_ws")
        if len(_WS) > 4096:
            _WS.clear()
        v = _WS[key] = n.value
    return v


# ---------------------------------------------------------------------------------------- reference
def _ref_norm(v, nm):
    mean = v.mean(1, keepdim=True) if nm.kind == "layer" else torch.zeros_like(v[:, :1])
    e = v - mean
    rstd = torch.rsqrt((e * e).mean(1, keepdim=True) + nm.eps)
    out = e * rstd
    if nm.gamma is not None:
        out = out * nm.gamma
    if nm.beta is not None:
        out = out + nm.beta
    return out, mean, rstd


def _ref_parts(x, gate, drop, M, C, rpg):
    g = None
    if gate is not None:
        g = gate.float().view(1, C) if gate.dim() == 1 else gate.float().repeat_interleave(rpg, 0)
    keep = ks = None
    if drop is not None:
        _, ks = DR.threshold(drop.rate)
        keep = DR.keep_mask((M, C), drop.rate, drop.seed, drop.step, first=int(drop.first))
    return g, keep, ks


def _ref_fwd(x, res, post, gate, scale, drop, pre, M, C, rpg):
    v = x.reshape(M, C).float()
    st = torch.zeros(4, M)
    st[1] = st[3] = 1.0
    if post is not None:
        v, m, s = _ref_norm(v, post)
        st[0], st[1] = m[:, 0], s[:, 0]
    g, keep, ks = _ref_parts(x, gate, drop, M, C, rpg)
    if g is not None:
        v = v * g
    v = v * scale
    if keep is not None:
        v = torch.where(keep, v * ks, 0.0)
    h = v if res is None else res.reshape(M, C).float() + v
    u = None
    if pre is not None:
        u, m, s = _ref_norm(h, pre)
        st[2], st[3] = m[:, 0], s[:, 0]
    return h, u, st


def _ref_norm_bwd(g, xhat, rstd, nm):
    gg = g if nm.gamma is None else g * nm.gamma
    d = gg - xhat * (gg * xhat).mean(1, keepdim=True)
    if nm.kind == "layer":
        d = d - gg.mean(1, keepdim=True)
    return d * rstd, (g * xhat).sum(0), g.sum(0)


def _ref_bwd(x, stats, res, post, gate, scale, drop, pre, du, dh, dx, dres, dgate, vecs, M, C, rpg):
    def put(t, v):
        if t is not None:
            t.copy_(v.reshape(t.shape).to(t.dtype))

    m1, s1, m2, s2 = (0.0, 1.0, 0.0, 1.0) if stats is None else (stats[k].view(M, 1) for k in range(4))
    n = x.reshape(M, C).float()
    xh = (n - m1) * s1
    if post is not None:
        n = xh * post.gamma if post.gamma is not None else xh
        n = n + post.beta if post.beta is not None else n
    g, keep, ks = _ref_parts(x, gate, drop, M, C, rpg)
    gs = scale if g is None else g * scale
    gh = dh.reshape(M, C).float() if dh is not None else torch.zeros(M, C)
    if pre is not None:
        h = n * gs
        if keep is not None:
            h = torch.where(keep, h * ks, 0.0)
        if res is not None:
            h = h + res.reshape(M, C).float()
        d, dg, db = _ref_norm_bwd(du.reshape(M, C).float(), (h - m2) * s2, s2, pre)
        gh = gh + d
        put(vecs[2], dg)
        put(vecs[3], db)
    put(dres, gh)
    dd = gh if keep is None else torch.where(keep, gh * ks, 0.0)
    if dgate is not None:
        dg = dd * n * scale
        put(dgate, dg.sum(0) if dgate.dim() == 1 else dg.view(-1, rpg, C).sum(1))
    dn = dd * gs
    if post is not None:
        dn, dg, db = _ref_norm_bwd(dn, xh, s1, post)
        put(vecs[0], dg)
        put(vecs[1], db)
    put(dx, dn)
