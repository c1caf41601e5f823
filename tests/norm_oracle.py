"""float64 oracle of the residual-block norms, with a bound on what fp32 arithmetic may miss.

``bound`` is in units of one fp32 rounding (2**-24): each formula is evaluated a second time on
magnitudes (every term positive, xhat replaced by (|h| + |mean|) * rstd, which also covers the
cancellation in h - mean).  An fp32 evaluation with at most K roundings on any path from an input to the
output stays within K * 2**-24 * bound to first order.
"""
import torch

import rng_oracle as O

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
# roundings on a path: four sums (mean, variance, and two of a gradient) of at most 8 + 6 + 16 additions
# each, and fewer than 40 single operations
K = 4 * 30 + 40


def drop_mask(shape, drop):
    if drop is None:
        return torch.ones(shape, dtype=torch.float64)
    rate, seed, step = drop
    idx = torch.arange(shape[0] * shape[1]).view(shape).numpy()
    return torch.from_numpy(O.keep(idx, rate, seed, step)).double() * O.scale(rate)


def norm(v, kind, gamma, beta, eps):
    mu = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    rstd = 1.0 / torch.sqrt(((v - mu) ** 2).mean(1, keepdim=True) + eps)
    y = (v - mu) * rstd
    y = y if gamma is None else y * gamma
    return (y if beta is None else y + beta), mu, rstd


def forward(x, res, post, gate, scale, mask, pre):
    """post / pre: (kind, gamma, beta, eps) or None -> h, u, extras."""
    M, C = x.shape
    n, m1, r1 = norm(x, *post) if post else (x, None, None)
    g = torch.ones((), dtype=x.dtype)
    if gate is not None:
        g = gate if gate.dim() == 1 else gate.repeat_interleave(M // gate.shape[0], 0)
    h = n * g * scale * mask
    h = h if res is None else h + res
    u, m2, r2 = norm(h, *pre) if pre else (None, None, None)
    return h, u, (n, g, m1, r1, m2, r2)


def run(x, res, post, gate, scale, drop, pre, du=None, dh=None):
    """{name: (exact, bound)} for every output."""
    d = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    leaf = lambda t: None if t is None else d(t).requires_grad_(True)  # noqa: E731
    X, R, G = leaf(x), leaf(res), leaf(gate)
    P = None if post is None else (post[0], leaf(post[1]), leaf(post[2]), post[3])
    Q = None if pre is None else (pre[0], leaf(pre[1]), leaf(pre[2]), pre[3])
    mask = drop_mask(tuple(x.shape), drop)
    h, u, (n, g, m1, r1, m2, r2) = forward(X, R, P, G, scale, mask, Q)
    out = {}
    with torch.no_grad():
        ab = lambda t, one=1.0: one if t is None else t.abs()  # noqa: E731
        A1 = (X.abs() + m1.abs()) * r1 if P else X.abs()
        N = A1 * ab(P[1]) + ab(P[2], 0.0) if P else A1
        S = abs(scale) * g.abs() * mask
        H = S * N + ab(R, 0.0)
        out["h"] = (h.detach(), H)
        if Q:
            # h's own error is seen through the norm as well
            A2 = (H + H.mean(1, keepdim=True)) * r2
            out["u"] = (u.detach(), A2 * ab(Q[1]) + ab(Q[2], 0.0) + A2 * A2.mean(1, keepdim=True) * ab(Q[1]))
    if du is None and dh is None:
        return out
    roots = [(t, d(v)) for t, v in ((u, du), (h, dh)) if v is not None]
    torch.autograd.backward([t for t, _ in roots], [v for _, v in roots])
    with torch.no_grad():
        def nb(gr, A, r, gamma, kind):
            gg = gr * ab(gamma)
            # the last factor: xhat enters twice, each time with A's error
            return r * (gg + gg.mean(1, keepdim=True) + 2 * A * (gg * A).mean(1, keepdim=True))

        DH = d(dh).abs() if dh is not None else torch.zeros_like(h)
        if Q:
            D = d(du).abs()
            DH = DH + nb(D, A2, r2, Q[1], Q[0])
            out["dpre.gamma"] = (ab(None) if Q[1] is None else Q[1].grad, (D * A2).sum(0))
            out["dpre.beta"] = (None if Q[2] is None else Q[2].grad, D.sum(0))
        if R is not None:
            out["dres"] = (R.grad, DH)
        DN = DH * S
        if G is not None:
            GG = DH * mask * abs(scale) * N
            out["dgate"] = (G.grad, GG.sum(0) if G.dim() == 1 else GG.view(G.shape[0], -1, G.shape[1]).sum(1))
        if P:
            out["dpost.gamma"] = (None if P[1] is None else P[1].grad, (DN * A1).sum(0))
            out["dpost.beta"] = (None if P[2] is None else P[2].grad, DN.sum(0))
            DN = nb(DN, A1, r1, P[1], P[0])
        out["dx"] = (X.grad, DN)
    return out


def check(name, got, want, rows):
    exact, bound = want
    k = K + (rows if name.startswith(("dgate", "dpost", "dpre")) else 0)  # column sums add the rows up
    tol = HALF[got.dtype] * exact.abs() * 1.01 + k * 2.0**-24 * bound + 1e-37
    err = (got.double().cpu() - exact).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} x tolerance"
