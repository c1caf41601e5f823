import pytest
import torch

import norm_oracle as NO
from pyspark_tf_gke_amd.ops import dropout as D
from pyspark_tf_gke_amd.ops import norm as N


def make(M, C, post, pre, gate, res, dtype, dev="cpu", seed=0, mean=0.1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0, mu=0.0: torch.randn(*s, generator=g) * std + mu  # noqa: E731
    t = {"x": r(M, C, std=1.5, mu=mean).to(dtype), "res": r(M, C, std=2.0).to(dtype) if res else None}
    mk = lambda k: None if k is None else (k, r(C, std=0.2, mu=1.0), r(C, std=0.2) if k == "layer" else None,  # noqa: E731
                                           1e-3 if k == "layer" else 1e-6)
    t["post"], t["pre"] = mk(post), mk(pre)
    t["gate"] = None if gate is None else r(C, std=0.3, mu=0.5) if gate == 0 else r(gate, C, std=0.3, mu=0.5).to(dtype)
    t["du"] = r(M, C, std=0.5).to(dtype) if pre else None
    t["dh"] = r(M, C, std=0.5).to(dtype)
    mv = lambda v: v.to(dev) if isinstance(v, torch.Tensor) else v  # noqa: E731
    return {k: tuple(mv(e) for e in v) if isinstance(v, tuple) else mv(v) for k, v in t.items()}


def both(t, scale=0.7, drop=None, ws=None):
    """Forward and backward through the operators -> {name: tensor}."""
    e = lambda v: None if v is None else torch.full_like(v, 7.0)  # noqa: E731
    nm = lambda s: None if s is None else N.Norm(*s)  # noqa: E731
    post, pre = nm(t["post"]), nm(t["pre"])
    M, C = t["x"].shape
    h, u = e(t["x"]), e(t["du"])
    st = N.block_norm_stats(M, t["x"].device)
    dr = None if drop is None else D.Drop(*drop)
    kw = dict(res=t["res"], post=post, gate=t["gate"], scale=scale, drop=dr, pre=pre)
    N.block_norm_fwd(t["x"], h=h, u=u, stats=st, **kw)
    dx, dres, dgate = e(t["x"]), e(t["res"]), e(t["gate"])
    pair = lambda s: None if s is None else (e(s[1]), e(s[2]))  # noqa: E731
    dpost, dpre = pair(t["post"]), pair(t["pre"])
    N.block_norm_bwd(t["x"], st, du=t["du"], dh=t["dh"], dx=dx, dres=dres, dgate=dgate, dpost=dpost, dpre=dpre,
                     workspace=ws, **kw)
    out = {"h": h, "u": u, "dx": dx, "dres": dres, "dgate": dgate}
    for name, p in (("dpost", dpost), ("dpre", dpre)):
        if p is not None:
            out[name + ".gamma"], out[name + ".beta"] = p
    return {k: v for k, v in out.items() if v is not None}


def compare(t, got, scale=0.7, drop=None):
    want = NO.run(t["x"], t["res"], t["post"], t["gate"], scale, drop, t["pre"], t["du"], t["dh"])
    for k, v in got.items():
        NO.check(k, v, want[k], t["x"].shape[0])


COMBOS = [(None, "layer", None, False), (None, "rms", 0, True), ("layer", "layer", 0, True), ("rms", "rms", 6, True),
          ("layer", None, 12, True), ("rms", "layer", None, False), (None, None, 0, True), (None, None, None, False)]


@pytest.mark.parametrize("post,pre,gate,res", COMBOS)
@pytest.mark.parametrize("drop", [None, (0.3, 99, 7)])
def test_reference_matches_oracle(post, pre, gate, res, drop):
    t = make(12, 21, post, pre, gate, res, torch.float32)
    compare(t, both(t, drop=drop), drop=drop)


def test_oracle_gradients_match_differences():
    """Central differences of the float64 forward."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    mask = NO.drop_mask((6, 5), (0.3, 5, 2))

    def f(x, res, g1, b1, gate, g2, b2):
        return NO.forward(x, res, ("layer", g1, b1, 1e-3), gate, 0.7, mask, ("rms", g2, b2, 1e-3))[:2]

    assert torch.autograd.gradcheck(f, (r(6, 5), r(6, 5), r(5), r(5), r(3, 5), r(5), r(5)))


def _kw(M=4, C=6):
    x = torch.randn(M, C)
    return x, N.Norm("layer", torch.ones(C), torch.zeros(C), 1e-3)


def test_refusals():
    x, ln = _kw()
    u = torch.empty_like(x)
    st = N.block_norm_stats(4, "cpu")
    ok = dict(pre=ln, u=u, stats=st)
    N.block_norm_fwd(x, **ok)
    bad = [
        (TypeError, x.half(), dict(pre=ln, u=u.half())),
        (ValueError, torch.randn(6, 4).t(), dict(pre=ln, u=torch.empty(4, 6))),
        (ValueError, x, dict(pre=ln)), (ValueError, x, dict(u=u)), (ValueError, x, dict()),
        (ValueError, x, dict(ok, pre=ln._replace(kind="group"))), (ValueError, x, dict(ok, pre=ln._replace(eps=0.0))),
        (ValueError, x, dict(ok, pre=ln._replace(gamma=torch.ones(5)))),
        (TypeError, x, dict(ok, pre=ln._replace(gamma=torch.ones(6).double()))),
        (ValueError, x, dict(ok, pre=ln._replace(kind="rms"))), (ValueError, x, dict(ok, res=torch.randn(3, 6))),
        (ValueError, x, dict(ok, gate=torch.ones(3, 6))), (ValueError, x, dict(ok, gate=torch.ones(5))),
        (ValueError, x, dict(ok, stats=torch.empty(4, 3))), (ValueError, x, dict(ok, u=torch.empty(4, 5))),
        (ValueError, x, dict(ok, drop=D.Drop(1.2, 1))), (ValueError, x, dict(pre=ln, u=x)),
    ]
    for exc, a, kw in bad:
        with pytest.raises(exc):
            N.block_norm_fwd(a, **kw)
    dx = torch.empty_like(x)
    ok = dict(pre=ln, du=x.clone(), dx=dx)
    N.block_norm_bwd(x, st, **ok)
    for kw in (dict(pre=ln, dx=dx), dict(ok, dx=None), dict(ok, dgate=torch.ones(6)), dict(dx=dx),
               dict(ok, dpost=(torch.ones(6), None)), dict(ok, dpre=(torch.ones(5), None)),
               dict(ok, dres=dx), dict(ok, du=x.bfloat16())):
        with pytest.raises(ValueError):
            N.block_norm_bwd(x, st, **kw)
    with pytest.raises(ValueError):
        N.block_norm_bwd(x, torch.empty(4, 5), **ok)


def test_empty():
    x, ln = _kw(0)
    N.block_norm_fwd(x, pre=ln, u=torch.empty_like(x), stats=N.block_norm_stats(0, "cpu"))
    dg = (torch.ones(6), torch.ones(6))
    N.block_norm_bwd(x, N.block_norm_stats(0, "cpu"), pre=ln, du=x.clone(), dx=x.clone(), dpre=dg)
    assert not dg[0].any() and not dg[1].any()
