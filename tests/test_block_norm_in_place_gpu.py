"""Block norm with outputs over its inputs, at widths whose last columns lie in a wave of their own (the last lane reads
8 values, most of them its neighbour's): the bits of the same call with outputs of their own."""
import pytest
import torch

from pyspark_tf_gke_amd.ops import dropout as D
from pyspark_tf_gke_amd.ops import norm as N
from test_block_norm_cpu import both, make

pytestmark = pytest.mark.gpu
WIDTHS = [513, 515, 519, 1027, 1541, 2051, 4097, 5127]


def rows_for(C):
    return 4 * (1 << 20) // C  # several rows a workgroup, whatever the width


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("post,pre", [(None, None), (None, "layer"), ("rms", None), ("layer", "rms")])
@pytest.mark.parametrize("C", WIDTHS)
def test_forward(hip_built, dtype, post, pre, C):
    t = make(rows_for(C), C, post, pre, 0, True, dtype, "cuda", seed=C)
    nm = lambda s: None if s is None else N.Norm(*s)  # noqa: E731
    kw = dict(post=nm(t["post"]), gate=t["gate"], scale=0.7, drop=D.Drop(0.3, 5, 9), pre=nm(t["pre"]))
    u = [None if pre is None else torch.empty_like(t["x"]) for _ in range(3)]
    want = torch.empty_like(t["x"])
    N.block_norm_fwd(t["x"], res=t["res"], h=want, u=u[0], **kw)
    over_res, over_x = t["res"].clone(), t["x"].clone()
    N.block_norm_fwd(t["x"], res=over_res, h=over_res, u=u[1], **kw)
    N.block_norm_fwd(over_x, res=t["res"], h=over_x, u=u[2], **kw)
    assert torch.equal(over_res, want) and torch.equal(over_x, want)
    assert pre is None or (torch.equal(u[1], u[0]) and torch.equal(u[2], u[0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("post,pre", [(None, None), (None, "layer"), ("rms", None), ("layer", "rms")])
@pytest.mark.parametrize("C", WIDTHS)
def test_backward(hip_built, dtype, post, pre, C):
    t = make(rows_for(C), C, post, pre, 0, True, dtype, "cuda", seed=C)
    drop = (0.3, 5, 9)
    want = both(t, drop=drop)
    nm = lambda s: None if s is None else N.Norm(*s)  # noqa: E731
    kw = dict(post=nm(t["post"]), gate=t["gate"], scale=0.7, drop=D.Drop(*drop), pre=nm(t["pre"]))
    st = N.block_norm_stats(len(t["x"]), "cuda")
    u = None if pre is None else torch.empty_like(t["x"])
    N.block_norm_fwd(t["x"], res=t["res"], h=torch.empty_like(t["x"]), u=u, stats=st, **kw)
    kw["res"] = t["res"]
    for dres_over, dx_over in (("dh", "x"), ("x", "dh"), ("du", "res"), ("res", "du")):
        b = {k: None if t[k] is None else t[k].clone() for k in ("x", "res", "du", "dh")}
        dres, dx = b[dres_over], b[dx_over]
        if dres is None or dx is None:
            continue
        N.block_norm_bwd(b["x"], st, du=b["du"], dh=b["dh"], dres=dres, dx=dx, **{**kw, "res": b["res"]})
        assert torch.equal(dres, want["dres"]) and torch.equal(dx, want["dx"]), (dres_over, dx_over)
