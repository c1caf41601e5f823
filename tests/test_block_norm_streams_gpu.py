"""Block norms at the same time: on two streams, and in two captured graphs, with a workspace each."""
import pytest
import torch

from pyspark_tf_gke_amd.ops import norm as N
from test_block_norm_cpu import both, make

pytestmark = pytest.mark.gpu
SIZES = [(3000, 384), (401, 1027), (5000, 64)]


def case(k, M, C):
    t = make(M, C, "layer", "layer", 0, True, torch.bfloat16, "cuda", seed=k)
    drop = (0.3, 9 + k, 5)
    return t, drop, both(t, drop=drop)


@pytest.mark.parametrize("M,C", SIZES)
def test_two_streams(hip_built, M, C):
    cases = [case(k, M, C) for k in range(2)]
    ws = [N.block_norm_workspace(M, C, 1, "cuda") for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (t, drop, _), w, s in zip(cases, ws, streams):
            with torch.cuda.stream(s):
                got.append(both(t, drop=drop, ws=w))
        torch.cuda.synchronize()
        for (_, _, want), g in zip(cases, got):
            assert all(torch.equal(g[n], want[n]) for n in want)


@pytest.mark.parametrize("M,C", SIZES)
def test_two_captured_graphs(hip_built, M, C):
    cases = [case(k, M, C) for k in range(2)]
    ws = [N.block_norm_workspace(M, C, 1, "cuda") for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for (t, drop, _), w in zip(cases, ws):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both(t, drop=drop, ws=w))
    for _ in range(4):
        for o in outs:
            for v in o.values():
                v.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (t, drop, want), o, w in zip(cases, outs, ws):
            assert all(torch.equal(o[n], want[n]) for n in want)
            eager = both(t, drop=drop, ws=w)  # between the replays
            assert all(torch.equal(eager[n], want[n]) for n in want)
