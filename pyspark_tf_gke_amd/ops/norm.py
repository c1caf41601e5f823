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
from typing import NamedTuple

import torch

from . import dropout as DR
from ._util import hip_on, on_device, ptr

KINDS = {"layer": 1, "rms": 2}
MAX_COLS = 8192


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
    from .. import _native

    if not 1 <= cols <= MAX_COLS:
        raise ValueError(f"block_norm: rows of 1..{MAX_COLS} columns, got {cols}")
    if groups < 1 or rows % groups:
        raise ValueError(f"block_norm: {rows} rows do not divide into {groups} gate groups")
    n = ctypes.c_long(0)
    _native.check(_native.hip_lib().ptg_block_norm_ws(rows, cols, groups, ctypes.byref(n)), "ptg_block_norm_ws")
    return torch.empty(n.value, dtype=torch.float32, device=device)


def _same(t, like, name):
    if t is None:
        return
    if t.dtype != like.dtype or t.shape != like.shape or t.device != like.device:
        raise ValueError(f"block_norm: {name} must match x in shape, dtype and device")
    if not t.is_contiguous():
        raise ValueError(f"block_norm: {name} must be contiguous")


def _vec(t, C, dev, name):
    if t is None:
        return
    if t.dtype != torch.float32:
        raise TypeError(f"block_norm: {name} must be float32, got {t.dtype}")
    if tuple(t.shape) != (C,) or t.device != dev or not t.is_contiguous():
        raise ValueError(f"block_norm: {name} must be a contiguous [{C}] vector on {dev}")


def _check_norm(nm, C, dev, name):
    if nm is None:
        return
    if nm.kind not in KINDS:
        raise ValueError(f"block_norm: {name} kind {nm.kind!r} (layer or rms)")
    if not float(nm.eps) > 0.0:
        raise ValueError(f"block_norm: {name} needs an epsilon > 0, got {nm.eps}")
    if nm.kind == "rms" and nm.beta is not None:
        raise ValueError(f"block_norm: {name}: an RMSNorm has no beta")
    _vec(nm.gamma, C, dev, name + ".gamma")
    _vec(nm.beta, C, dev, name + ".beta")


def _gate_dims(gate, x, M, C):
    """(mode, rows per gate row)."""
    if gate is None:
        return 0, 1
    if gate.dim() == 1:
        _vec(gate, C, x.device, "gate")
        return 1, max(M, 1)
    if gate.dim() != 2 or gate.shape[1] != C or gate.dtype != x.dtype or gate.device != x.device \
            or not gate.is_contiguous():
        raise ValueError(f"block_norm: gate must be fp32 [{C}] or {x.dtype} [groups, {C}], contiguous, on {x.device}")
    G = gate.shape[0]
    if M and (G == 0 or M % G):
        raise ValueError(f"block_norm: {M} rows do not divide into {G} gate groups")
    return 2, M // G if G else 1


def _common(x, res, post, gate, drop, pre):
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"block_norm: expected bfloat16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("block_norm: x needs at least one column")
    if not x.is_contiguous():
        raise ValueError("block_norm: x must be contiguous")
    C = x.shape[-1]
    M = x.numel() // C
    if C > MAX_COLS and x.is_cuda:
        raise ValueError(f"block_norm: rows of at most {MAX_COLS} columns, got {C}")
    _same(res, x, "res")
    _check_norm(post, C, x.device, "post")
    _check_norm(pre, C, x.device, "pre")
    mode, rpg = _gate_dims(gate, x, M, C)
    d = (0, 0, 1.0, 0, 0, None)  # on, threshold, scale, seed, host step, device step
    if drop is not None:
        thr, ds = DR.threshold(drop.rate)
        host, dev = DR.step_args(drop.step, x.device)
        d = (1, thr, ds, DR._signed(drop.seed), host, dev)
    return M, C, mode, rpg, d


def _stats_ok(stats, M, dev):
    if stats.dtype != torch.float32 or tuple(stats.shape) != (4, M) or stats.device != dev or not stats.is_contiguous():
        raise ValueError(f"block_norm: stats must be a contiguous fp32 [4, {M}] on {dev}")


def _aligned(C, *ts) -> int:
    return int(C % 8 == 0 and all(t is None or t.data_ptr() % 16 == 0 for t in ts))


def _nk(nm):
    return 0 if nm is None else KINDS[nm.kind]


def block_norm_fwd(x, *, res=None, post=None, gate=None, scale: float = 1.0, drop=None, pre=None, h=None, u=None,
                   stats=None):
    """Writes ``h`` (if given) and ``u`` (with ``pre``); ``stats`` (:func:`block_norm_stats`) for a
    backward pass.  Returns (h, u).  ``h`` may be ``res``, nothing else may overlap an input."""
    M, C, mode, rpg, d = _common(x, res, post, gate, drop, pre)
    _same(h, x, "h")
    _same(u, x, "u")
    if (pre is None) != (u is None):
        raise ValueError("block_norm: u goes with pre")
    if h is None and u is None:
        raise ValueError("block_norm: nothing to write (h and u are None)")
    if stats is not None:
        _stats_ok(stats, M, x.device)
    _no_overlap({"x": x, "res": res, "gate": gate}, {"h": h, "u": u}, allow=(("res", "h"), ("x", "h")))
    if not on_device(x):
        hv, uv, st = _ref_fwd(x, res, post, gate, scale, drop, pre, M, C, rpg)
        if h is not None:
            h.copy_(hv.view(x.shape).to(h.dtype))
        if u is not None:
            u.copy_(uv.view(x.shape).to(u.dtype))
        if stats is not None:
            stats.copy_(st)
        return h, u
    p, q = post or (None,) * 4, pre or (None,) * 4
    hip_on(x.device, "ptg_block_norm_fwd", ptr(x), ptr(res), ptr(gate), ptr(h), ptr(u), ptr(p[1]), ptr(p[2]), ptr(q[1]),
           ptr(q[2]), ptr(stats), M, C, int(x.dtype == torch.float32),
           _aligned(C, x, res, gate if mode == 2 else None, h, u), _nk(post), float(p[3] or 0.0), _nk(pre),
           float(q[3] or 0.0), mode, rpg, float(scale), *d[:5], ptr(d[5]))
    return h, u


def block_norm_bwd(x, stats, *, res=None, post=None, gate=None, scale: float = 1.0, drop=None, pre=None, du=None,
                   dh=None, dx=None, dres=None, dgate=None, dpost=None, dpre=None, workspace=None):
    """Gradients of :func:`block_norm_fwd` (same x, res, post, gate, scale, drop, pre) from ``du`` (with
    ``pre``) and ``dh`` (None: zero).  Writes dx and dres (None: skipped), ``dgate`` like ``gate``, and
    ``dpost`` / ``dpre`` = (dgamma, dbeta), fp32 [C] or None where the norm has none.  ``dres`` may be
    ``dh``.  ``workspace``: :func:`block_norm_workspace` (None: allocated here)."""
    M, C, mode, rpg, d = _common(x, res, post, gate, drop, pre)
    for t, name in ((du, "du"), (dh, "dh"), (dx, "dx"), (dres, "dres")):
        _same(t, x, name)
    if (pre is None) != (du is None):
        raise ValueError("block_norm: du goes with pre")
    if pre is None and dh is None:
        raise ValueError("block_norm: no gradient comes in (du and dh are None)")
    if dx is None and dres is None and dgate is None and dpost is None and dpre is None:
        raise ValueError("block_norm: no gradient is asked for")
    _stats_ok(stats, M, x.device)
    if dgate is not None:
        if gate is None or dgate.shape != gate.shape or dgate.dtype != gate.dtype or dgate.device != x.device \
                or not dgate.is_contiguous():
            raise ValueError("block_norm: dgate must match gate")
    vecs = []
    for g, nm, name in ((dpost, post, "dpost"), (dpre, pre, "dpre")):
        g = g or (None, None)
        for t, w, part in ((g[0], nm.gamma if nm else None, "gamma"), (g[1], nm.beta if nm else None, "beta")):
            if t is not None and w is None:
                raise ValueError(f"block_norm: {name} asks for the gradient of an absent {part}")
            _vec(t, C, x.device, f"{name}.{part}")
            vecs.append(t)
    _no_overlap({"x": x, "res": res, "gate": gate, "du": du, "dh": dh}, {"dx": dx, "dres": dres, "dgate": dgate},
                allow=(("dh", "dres"), ("du", "dres"), ("du", "dx"), ("dh", "dx"), ("x", "dx"), ("res", "dres"),
                       ("x", "dres"), ("res", "dx")))
    if M == 0:
        for t in (dgate, *vecs):
            if t is not None:
                t.zero_()
        return dx, dres
    if not on_device(x):
        _ref_bwd(x, stats, res, post, gate, scale, drop, pre, du, dh, dx, dres, dgate, vecs, M, C, rpg)
        return dx, dres
    groups = M // rpg if mode == 2 else 1
    need = block_norm_workspace_floats(M, C, groups)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.float32, device=x.device)
    elif workspace.dtype != torch.float32 or workspace.device != x.device or workspace.numel() < need \
            or not workspace.is_contiguous():
        raise ValueError(f"block_norm: workspace must hold {need} contiguous floats on {x.device}")
    p, q = post or (None,) * 4, pre or (None,) * 4
    if mode == 2 and dgate is None:
        mode_b, keep = 2, torch.empty_like(gate)  # the kernel writes it; dropped
    else:
        mode_b, keep = mode, dgate
    hip_on(x.device, "ptg_block_norm_bwd", ptr(x), ptr(res), ptr(gate), ptr(du), ptr(dh), ptr(dx), ptr(dres), ptr(p[1]),
           ptr(p[2]), ptr(q[1]), ptr(stats), *[ptr(t) for t in vecs], ptr(keep), ptr(workspace), M, C,
           int(x.dtype == torch.float32),
           _aligned(C, x, res, gate if mode == 2 else None, du, dh, dx, dres, keep if mode == 2 else None), _nk(post),
           _nk(pre), mode_b, rpg, float(scale), *d[:5], ptr(d[5]))
    return dx, dres


_WS: dict = {}


def block_norm_workspace_floats(rows: int, cols: int, groups: int) -> int:
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


def _no_overlap(ins, outs, allow):
    """Outputs must not overlap inputs or one another; a pair in ``allow`` may be the very same buffer
    (every element is read before it is written, by the same thread)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()

    named = [(n, t) for n, t in ins.items() if t is not None and t.numel()]
    done = []
    for on, o in outs.items():
        if o is None or not o.numel():
            continue
        lo, hi = span(o)
        for n, t in named + done:
            a, b = span(t)
            if lo < b and a < hi and not ((n, on) in allow and (a, b) == (lo, hi)):
                raise ValueError(f"block_norm: {on} overlaps {n}")
        done.append((on, o))


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
        keep = DR.keep_mask((M, C), drop.rate, drop.seed, drop.step)
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

    m1, s1, m2, s2 = (stats[k].view(M, 1) for k in range(4))
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
