import pytest
import torch

import norm_oracle as NO
from pyspark_tf_gke_amd.ops import dropout as D
from pyspark_tf_gke_amd.ops import norm as N
from test_block_norm_cpu import COMBOS, both, compare, make

pytestmark = pytest.mark.gpu
DROP = (0.3, 0xABCDEF0123456789, 1 << 33)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("post,pre,gate,res", COMBOS)
@pytest.mark.parametrize("C", [8, 24, 128, 512, 520, 1024, 2048])
def test_aligned(hip_built, dtype, post, pre, gate, res, C):
    t = make(12, C, post, pre, gate, res, dtype, "cuda", seed=C)
    compare(t, both(t, drop=DROP), drop=DROP)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C", [1, 2, 7, 9, 15, 17, 63, 65, 255, 257, 511, 513, 771, 1025, 2047, 4095, 4097, 8191])
def test_odd_columns(hip_built, dtype, C):
    for post, pre, gate, res in (("layer", "layer", 0, True), ("rms", "rms", 3, True), (None, "layer", None, False)):
        t = make(6, C, post, pre, gate, res, dtype, "cuda", seed=C)
        compare(t, both(t, drop=DROP), drop=DROP)


@pytest.mark.parametrize("C", [4096, 8192])
def test_wide(hip_built, C):
    t = make(5, C, "layer", "rms", 0, True, torch.bfloat16, "cuda")
    compare(t, both(t, drop=DROP), drop=DROP)


@pytest.mark.parametrize("M,C", [(1, 64), (3, 2048), (1000, 16), (2049, 40), (5000, 256), (1537, 771), (2100, 1024)])
def test_rows(hip_built, M, C):
    t = make(M, C, "layer", "layer", 0, True, torch.bfloat16, "cuda")
    compare(t, both(t, drop=DROP), drop=DROP)


@pytest.mark.parametrize("G,rpg", [(1, 1), (37, 1), (5, 3), (9, 29), (2, 300), (1, 3000), (700, 40), (3, 1001)])
@pytest.mark.parametrize("C", [16, 200, 768, 1027])
def test_gate_groups(hip_built, G, rpg, C):
    t = make(G * rpg, C, None, "layer", G, True, torch.bfloat16, "cuda")
    compare(t, both(t))


@pytest.mark.parametrize("G,rpg", [(1, 29), (1, 62), (1, 200), (3, 70), (600, 62), (2, 8), (257, 5), (2000, 17)])
@pytest.mark.parametrize("C", [7, 24, 48, 520])
def test_gate_groups_shared_and_own(hip_built, G, rpg, C):
    """Groups whose rows a workgroup's slots share, and groups that a slot goes through alone."""
    t = make(G * rpg, C, "rms", "layer", G, True, torch.float32, "cuda")
    compare(t, both(t, drop=DROP), drop=DROP)


@pytest.mark.parametrize("G,rpg", [(1, 40), (6, 3), (300, 1), (2, 301)])
@pytest.mark.parametrize("C", [2056, 4101, 8192])
@pytest.mark.parametrize("post", [None, "layer"])
def test_gate_groups_wide(hip_built, G, rpg, C, post):
    """Rows of 16 waves: a layer pair and grouped gates of 8192 columns just fit their vectors in LDS."""
    t = make(G * rpg, C, post, "layer", G, True, torch.bfloat16, "cuda")
    compare(t, both(t, drop=DROP), drop=DROP)


@pytest.mark.parametrize("C", [3000, 6144, 8192])
@pytest.mark.parametrize("post,pre", [("layer", "layer"), ("rms", "layer"), (None, "rms"), ("layer", None), (None, None)])
def test_wide_vectors_in_and_out_of_lds(hip_built, C, post, pre):
    t = make(530, C, post, pre, 0, True, torch.float32, "cuda")
    compare(t, both(t, drop=DROP), drop=DROP)


def test_unaligned_bases(hip_built):
    t = make(7, 64, "layer", "rms", 7, True, torch.bfloat16, "cuda")

    def shift(v):
        b = torch.empty(v.numel() + 1, dtype=v.dtype, device=v.device)[1:].view(v.shape)
        return b.copy_(v)

    t = {k: shift(v) if isinstance(v, torch.Tensor) else v for k, v in t.items()}
    compare(t, both(t, drop=DROP), drop=DROP)


def test_offset_rows_keep_their_precision(hip_built):
    """A row mean of 4096 over a standard deviation of 1: a sum of squares around zero would lose the
    variance, the deviations do not."""
    t = make(9, 2048, None, "layer", None, False, torch.float32, "cuda", mean=4096.0)
    compare(t, both(t, scale=1.0), scale=1.0)


def test_constant_rows_and_zero_rows(hip_built):
    x = torch.zeros(4, 640, device="cuda")
    x[1] = 3.25
    u = torch.empty_like(x)
    N.block_norm_fwd(x, pre=N.Norm("layer", None, None, 1e-3), u=u)
    # the sums of 3.25 are exact; 1 / 640 and the product with it are rounded, so the mean is off by at most
    # 2 * 2**-24 * 3.25 (3 with second-order terms), seen through 1 / sqrt(epsilon)
    assert not u[[0, 2, 3]].any() and float(u[1].abs().max()) <= 3 * 2.0**-24 * 3.25 / 1e-3**0.5
    N.block_norm_fwd(x, pre=N.Norm("rms", None, None, 1e-6), u=u)
    assert not u[0].any() and abs(float(u[1, 0]) - 1) < 1e-6


def test_rows_are_independent_of_bad_rows(hip_built):
    """NaN and infinite rows stay in their rows (forward and input gradients)."""
    t = make(10, 300, "layer", "layer", None, True, torch.float32, "cuda")
    good = both(t)
    t["x"][3] = float("nan")
    t["x"][7, 5] = float("inf")
    bad = both(t)
    rows = [0, 1, 2, 4, 5, 6, 8, 9]
    for k in ("h", "u", "dx", "dres"):
        assert torch.equal(good[k][rows], bad[k][rows])
        assert not torch.isfinite(bad[k][3]).any()


def test_same_bits_every_run_and_workspace(hip_built):
    t = make(3000, 384, "layer", "layer", 0, True, torch.bfloat16, "cuda")
    ws = N.block_norm_workspace(3000, 384, 1, "cuda")
    a, b = both(t, drop=DROP, ws=ws), both(t, drop=DROP)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_in_place(hip_built):
    """h over res, dres over dh, dx over x."""
    t = make(50, 96, "rms", "layer", 0, True, torch.bfloat16, "cuda")
    want = both(t)
    post, pre = N.Norm(*t["post"]), N.Norm(*t["pre"])
    st, u, res0 = N.block_norm_stats(50, "cuda"), torch.empty_like(t["x"]), t["res"].clone()
    kw = dict(post=post, gate=t["gate"], scale=0.7, pre=pre)
    N.block_norm_fwd(t["x"], res=t["res"], h=t["res"], u=u, stats=st, **kw)
    assert torch.equal(t["res"], want["h"]) and torch.equal(u, want["u"])
    N.block_norm_bwd(t["x"], st, res=res0, du=t["du"], dh=t["dh"], dres=t["dh"], dx=t["x"], **kw)
    assert torch.equal(t["dh"], want["dres"]) and torch.equal(t["x"], want["dx"])


def test_nothing_beside_the_outputs_is_written(hip_built):
    for C in (72, 77):
        t = make(9, C, None, "layer", None, True, torch.bfloat16, "cuda")
        buf = torch.full((9 * C + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
        u = buf[32:32 + 9 * C].view(9, C)
        N.block_norm_fwd(t["x"], res=t["res"], pre=N.Norm(*t["pre"]), u=u)
        assert (buf[:32] == 7).all() and (buf[32 + 9 * C:] == 7).all()


def test_captured(hip_built):
    """Forward and backward in a captured graph, the mask advancing each replay, on two streams."""
    t = make(400, 160, "layer", "layer", 0, True, torch.bfloat16, "cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    ws = N.block_norm_workspace(400, 160, 1, "cuda")
    both(t, drop=(0.3, 9, step), ws=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        D.drop_advance(step)
        out = both(t, drop=(0.3, 9, step), ws=ws)
    for k in range(1, 4):
        g.replay()
        torch.cuda.synchronize()
        want = both(t, drop=(0.3, 9, k))
        assert all(torch.equal(out[n], want[n]) for n in out)


def test_skipped_gradients(hip_built):
    """Gradients that are not asked for: null destinations."""
    t = make(40, 88, "layer", "layer", 5, True, torch.bfloat16, "cuda")
    want = both(t)
    post, pre = N.Norm(*t["post"]), N.Norm(*t["pre"])
    st, u = N.block_norm_stats(40, "cuda"), torch.empty_like(t["x"])
    kw = dict(res=t["res"], post=post, gate=t["gate"], scale=0.7, pre=pre)
    N.block_norm_fwd(t["x"], u=u, stats=st, **kw)
    dx = torch.empty_like(u)
    N.block_norm_bwd(t["x"], st, du=t["du"], dh=t["dh"], dx=dx, **kw)
    assert torch.equal(dx, want["dx"]) and torch.equal(u, want["u"])
    dg = torch.empty(88, device="cuda")
    N.block_norm_bwd(t["x"], st, du=t["du"], dh=t["dh"], dpost=(None, dg), **kw)
    assert torch.equal(dg, want["dpost.beta"])


def test_refusals(hip_built):
    x = torch.zeros(4, 8200, device="cuda")
    with pytest.raises(ValueError):
        N.block_norm_fwd(x, pre=N.Norm("layer", None, None, 1e-3), u=torch.empty_like(x))
    x = torch.zeros(4, 64, device="cuda")
    ln = N.Norm("layer", torch.ones(64), None, 1e-3)
    with pytest.raises(ValueError):  # gamma on the host
        N.block_norm_fwd(x, pre=ln, u=torch.empty_like(x))
    ln = N.Norm("layer", None, None, 1e-3)
    st = N.block_norm_stats(4, "cuda")
    with pytest.raises(ValueError):
        N.block_norm_bwd(x, st, pre=ln, du=x.clone(), dx=torch.empty_like(x), workspace=torch.empty(3, device="cuda"))


_ = NO
