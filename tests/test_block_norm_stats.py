"""A block norm's backward pass and the row statistics: refused where a norm needs them, not asked for without one."""
import pytest
import torch

from pyspark_tf_gke_amd.ops import dropout as D
from pyspark_tf_gke_amd.ops import norm as N


@pytest.mark.parametrize("side", ["post", "pre"])
def test_a_norm_needs_them(side):
    x = torch.randn(4, 6)
    kw = {side: N.Norm("layer", None, None, 1e-3), ("du" if side == "pre" else "dh"): x.clone()}
    with pytest.raises(ValueError, match="stats"):
        N.block_norm_bwd(x, None, dx=torch.empty_like(x), **kw)


def no_norm(dev, M, C):
    g = torch.Generator().manual_seed(C)
    x, res, dh, gate = (torch.randn(M, C, generator=g).to(dev) for _ in range(4))
    kw = dict(res=res, gate=gate, scale=0.7, drop=D.Drop(0.3, 5, 2))
    outs = []
    for stats in (N.block_norm_stats(M, dev), None):
        h, dx, dres, dgate = (torch.empty_like(x) for _ in range(4))
        N.block_norm_fwd(x, h=h, stats=stats, **kw)
        N.block_norm_bwd(x, stats, dh=dh, dx=dx, dres=dres, dgate=dgate, **kw)
        outs.append((h, dx, dres, dgate))
    return outs


def test_none_without_a_norm():
    with_stats, without = no_norm("cpu", 5, 24)
    assert all(torch.equal(a, b) for a, b in zip(with_stats, without))


@pytest.mark.gpu
@pytest.mark.parametrize("M,C", [(5, 24), (300, 1027), (7, 2056)])
def test_none_without_a_norm_on_the_gpu(hip_built, M, C):
    with_stats, without = no_norm("cuda", M, C)
    assert all(torch.equal(a, b) for a, b in zip(with_stats, without))
