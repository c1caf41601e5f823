import pytest
import torch

from pyspark_tf_gke_amd.ops import quant as Q
from test_int4_cpu import codes_for

pytestmark = pytest.mark.gpu


def weights64(codes, scale, zero, group):
    N, K = codes.shape[0], codes.shape[1] * 2
    q = torch.stack((codes & 15, codes >> 4), 2).view(N, K // group, group).double()
    z = 8.0 if zero is None else zero.double()[:, :, None]
    return ((q - z) * scale.double()[:, :, None]).view(N, K)


SHAPES = [(1, 1, 32, 32), (1, 16, 128, 128), (3, 17, 160, 32), (5, 33, 320, 64), (16, 100, 1024, 128),
          (17, 48, 2048, 64), (1, 2048, 20480, 128), (2, 7, 4096, 32), (33, 130, 1280, 128), (64, 64, 512, 64),
          (65, 50, 1056, 32), (130, 300, 2560, 128), (256, 64, 640, 64), (300, 272, 1152, 128), (1, 5000, 256, 64),
          (70, 530, 3040, 32), (40, 256, 20480, 64), (129, 1000, 4160, 64), (33, 2, 32, 32), (70, 8200, 1056, 32),
          (64, 8192, 1280, 128), (255, 3100, 960, 64), (1, 1 << 21, 32, 32)]


@pytest.mark.parametrize("B,N,K,group", SHAPES)
@pytest.mark.parametrize("zero", [False, True])
def test_exact_on_small_integers(hip_built, B, N, K, group, zero):
    """Integer inputs and power-of-two scales: every partial sum is a multiple of 1/8 below 2**21, so
    fp32 holds it exactly in any order and the fp32 output must be equal."""
    codes, scale, z, _ = codes_for(N, K, group, zero, seed=B + N, dev="cuda")
    w = Q.int4_layout(codes, scale, z, group)
    g = torch.Generator().manual_seed(K)
    x = torch.randint(-1, 2, (B, K), generator=g).to(torch.bfloat16).cuda()
    b = torch.randint(-3, 4, (N,), generator=g).float().cuda()
    out = torch.full((B, N), 7.0, device="cuda")
    Q.int4_dense_fwd(x, w, b, "relu", out)
    want = torch.relu(x.double() @ weights64(codes, scale, z, group).t() + b.double())
    assert torch.equal(out.double(), want)
    o16 = torch.empty(B, N, device="cuda", dtype=torch.bfloat16)
    Q.int4_dense_fwd(x, w, None, "linear", o16, workspace=Q.int4_workspace(B, w))
    assert torch.equal(o16, (x.double() @ weights64(codes, scale, z, group).t()).to(torch.bfloat16))


@pytest.mark.parametrize("B,N,K,group,zero", [(1, 2048, 20480, 128, False), (16, 512, 4096, 64, True),
                                               (200, 256, 2048, 32, True)])
def test_random_values(hip_built, B, N, K, group, zero):
    codes, scale, z, _ = codes_for(N, K, group, zero, dev="cuda", pow2=False)
    w = Q.int4_layout(codes, scale, z, group)
    x = torch.randn(B, K, device="cuda").to(torch.bfloat16)
    out = torch.empty(B, N, device="cuda")
    Q.int4_dense_fwd(x, w, None, None, out)
    w64 = weights64(codes, scale, z, group)
    want = x.double() @ w64.t()
    # products are exact; every sum is at most 55 * scale * |x| a term ((16 + z) and (16 + u) parts);
    # roundings: 2 * group inside a group, one for each group and a few joins
    mag = x.double().abs() @ (scale.double() * 55).repeat_interleave(group, 1).t()
    tol = (2 * group + K // group + 40) * 2.0**-24 * mag
    assert ((out.double() - want).abs() <= tol).all()
    # errors of many roundings add up at random: far below that worst case
    assert float(((out.double() - want).pow(2).mean() / want.pow(2).mean()).sqrt()) < 2.0**-16


def test_rows_do_not_mix_and_nothing_else_is_written(hip_built):
    codes, scale, z, _ = codes_for(37, 512, 128, True, dev="cuda")
    w = Q.int4_layout(codes, scale, z, 128)
    x = torch.randint(-1, 2, (20, 512), device="cuda").to(torch.bfloat16)
    buf = torch.full((20 * 37 + 64,), 7.0, device="cuda")
    out = buf[32:32 + 20 * 37].view(20, 37)
    Q.int4_dense_fwd(x, w, None, None, out)
    good = out.clone()
    assert (buf[:32] == 7).all() and (buf[32 + 20 * 37:] == 7).all()
    x[5] = float("nan")
    Q.int4_dense_fwd(x, w, None, None, out)
    rows = [r for r in range(20) if r != 5]
    assert torch.equal(out[rows], good[rows]) and torch.isnan(out[5]).all()
    one = torch.empty(1, 37, device="cuda")
    Q.int4_dense_fwd(x[7:8], w, None, None, one)  # a view that starts inside a batch
    assert torch.equal(one[0], good[7])
    Q.int4_dense_fwd(x[:0], w, None, None, out[:0])


@pytest.mark.parametrize("B,N,K,group", [(3, 20, 160, 32), (66, 20, 160, 32), (40, 300, 1088, 64), (12, 20, 192, 64)])
def test_padding_reads_nothing_of_a_neighbour(hip_built, B, N, K, group):
    """K % 128 != 0: the tile's rest lies over the next row, here all NaN; the last row's over NaN too."""
    codes, scale, z, _ = codes_for(N, K, group, True, dev="cuda")
    w = Q.int4_layout(codes, scale, z, group)
    buf = torch.full((2 * B + 1, K), float("nan"), device="cuda", dtype=torch.bfloat16)
    x = torch.randint(-1, 2, (B, K), device="cuda").to(torch.bfloat16)
    buf[:B] = x
    buf[1:B:2] = float("nan")
    out = torch.empty(B, N, device="cuda")
    Q.int4_dense_fwd(buf[:B], w, None, None, out)
    want = x.double() @ weights64(codes, scale, z, group).t()
    assert torch.equal(out[0::2].double(), want[0::2]) and torch.isnan(out[1::2]).all()


@pytest.mark.parametrize("B,N,K,group", [(1, 40, 4096, 128), (16, 33, 256, 32), (30, 20, 512, 64), (70, 300, 8192, 128)])
@pytest.mark.parametrize("zero", [False, True])
def test_infinities_and_large_inputs(hip_built, B, N, K, group, zero):
    """Row 0 has one infinity, row 1 two of one sign, row 2 a NaN, row 3 values near the largest number that
    cancel: the outputs are those of the formula, and ReLU keeps a NaN."""
    codes, scale, z, _ = codes_for(N, K, group, zero, dev="cuda")
    w = Q.int4_layout(codes, scale, z, group)
    x = torch.randint(-1, 2, (B, K), device="cuda").to(torch.bfloat16)
    x[0, 5] = float("inf")
    if B > 3:
        x[1, 3], x[1, K - 1] = float("-inf"), float("-inf")
        x[2, 7] = float("nan")
        x[3] = 0
        x[3, 0] = 2.0**125
    out, pos = torch.empty(B, N, device="cuda"), torch.empty(B, N, device="cuda")
    Q.int4_dense_fwd(x, w, None, None, out)
    Q.int4_dense_fwd(x, w, None, "relu", pos)
    w64 = weights64(codes, scale, z, group)
    want = (x.double()[:, None] * w64[None]).sum(2).float()  # single terms, no offset
    assert torch.isinf(want[0]).any()
    assert torch.equal(torch.nan_to_num(out, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(pos, nan=7.0), torch.nan_to_num(torch.relu(want), nan=7.0))


@pytest.mark.parametrize("B", [4, 20, 70])
def test_unaligned_input(hip_built, B):
    codes, scale, z, _ = codes_for(40, 256, 64, True, dev="cuda")
    w = Q.int4_layout(codes, scale, z, 64)
    b = torch.randint(-1, 2, (B * 256 + 1,), device="cuda").to(torch.bfloat16)
    x = b[1:].view(B, 256)
    out, want = torch.empty(B, 40, device="cuda"), torch.empty(B, 40, device="cuda")
    Q.int4_dense_fwd(x, w, None, None, out)
    Q.int4_dense_fwd(x.clone(), w, None, None, want)
    assert torch.equal(out, want)


def test_captured_and_two_streams(hip_built):
    """One weight used by two streams at once and by a captured graph, each with its own workspace."""
    codes, scale, z, _ = codes_for(512, 8192, 128, False, dev="cuda")
    w = Q.int4_layout(codes, scale, z, 128)
    xs = [torch.randint(-1, 2, (4, 8192), device="cuda").to(torch.bfloat16) for _ in range(2)]
    want = [torch.empty(4, 512, device="cuda") for _ in range(2)]
    for x, o in zip(xs, want):
        Q.int4_dense_fwd(x, w, None, None, o)
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty(4, 512, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, x, o in zip(st, xs, outs):
            with torch.cuda.stream(s):
                Q.int4_dense_fwd(x, w, None, None, o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    ws, sx, so = Q.int4_workspace(4, w), xs[0].clone(), torch.empty(4, 512, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Q.int4_dense_fwd(sx, w, None, None, so, workspace=ws)
    for k in (1, 0, 1):
        sx.copy_(xs[k])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(so, want[k])


def test_refusals(hip_built):
    codes, scale, z, _ = codes_for(512, 8192, 128, False, dev="cuda")
    w = Q.int4_layout(codes, scale, z, 128)
    x, out = torch.zeros(1, 8192, device="cuda"), torch.empty(1, 512, device="cuda")
    with pytest.raises(TypeError):
        Q.int4_dense_fwd(x, w, None, None, out)
    x = x.bfloat16()
    with pytest.raises(ValueError):
        Q.int4_dense_fwd(x.cpu(), w, None, None, out)
    if Q.int4_workspace(1, w) is not None:
        with pytest.raises(ValueError):
            Q.int4_dense_fwd(x, w, None, None, out, workspace=torch.empty(5, device="cuda"))
    both = torch.zeros(8192 + 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps"):
        Q.int4_dense_fwd(both[:8192].view(1, 8192), w, None, None, both[4096:4608].view(1, 512))
