"""Data-parallel training of residual blocks (2 gloo ranks): the gradients of every parameter are summed, also of
those that a fused block boundary holds from both sides of a gate computed in between."""
import pytest

from test_distributed_cpu import _results, _run_ranks

BODY = """
import json, torch, numpy as np
from pyspark_tf_gke_amd import nn
from pyspark_tf_gke_amd.distribute import MultiWorkerMirroredStrategy
from pyspark_tf_gke_amd.nn import layers as L
from pyspark_tf_gke_amd.parallel import comm

def model(st):
    L.reset_name_counters()
    inp = nn.Input(shape=(24,))
    h = nn.Dense(72, activation="relu", name="stem")(inp)
    y = nn.LayerNormalization(name="post")(nn.Dense(72, name="a")(h))
    y = nn.Multiply(name="gate")([y, nn.Dense(72, name="cond")(inp)])  # declared behind the norm, computed before the block
    u = nn.RMSNormalization(name="pre")(nn.Add(name="add")([h, y]))
    with st.scope():
        m = nn.Model(inp, nn.Dense(2, name="head")(u))
        m.build(device="cpu")
    m.compile(optimizer=nn.optimizers.SGD(0.5), loss="mse")
    return m

shard = bool(SHARD)
st = MultiWorkerMirroredStrategy(device="cpu", sharded_update=shard, bucket_mb=1e-3)
reduce = comm.all_reduce_
comm.all_reduce_ = lambda t, async_op=False: reduce(t)  # at once: takes what the gradients are at its launch
r = np.random.default_rng(0)
X = torch.from_numpy(r.standard_normal((16, 24)).astype(np.float32))
Y = torch.from_numpy(r.standard_normal((16, 2)).astype(np.float32))
m = model(st)
w0 = {p.name: p.data.clone() for p in m.store.params}
want = {}
ref = model(type("S", (), {"scope": lambda self: __import__("contextlib").nullcontext()})())
for k in (0, 8):
    ref.store.zero_grad()
    ref.store.flat_grad.zero_()
    out = ref._run_forward(X[k:k + 8], True)
    ref._run_backward(ref._loss_grad(out, Y[k:k + 8], torch.zeros(8)))
    for p in ref.store.params:
        want[p.name] = want.get(p.name, 0) + 0.5 * p.grad.clone()
lo = 8 * st.rank
m.train_step_fast(X[lo:lo + 8], Y[lo:lo + 8], m._stats_buf())
st.synchronize_master(m)
diff = {p.name: float((w0[p.name] - p.data - 0.5 * want[p.name]).norm() / want[p.name].norm()) for p in m.store.params}
print("RESULT", json.dumps(diff), flush=True)
"""


@pytest.mark.parametrize("sharded", [False, True])
def test_gate_computed_behind_the_norm_of_its_block(sharded):
    r = _run_ranks(BODY.replace("SHARD", str(int(sharded))), extra_env={"PTG_HOST_FP32": "1"})
    assert r.returncode == 0, r.stdout + r.stderr
    res = _results(r.stdout)
    # fp32 sums of 8 samples in another order, and w - w0 rounded at w's size
    assert len(res) == 2 and all(v < 1e-4 for d in res.values() for v in d.values()), res
