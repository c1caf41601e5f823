"""Cases, plain forms and exact values of the residual-block and small-weight operators.

Three operators are covered, by the ``"op"`` of a case:

* ``dropout``: y = keep ? x / p : 0 with the mask drawn from a counter-based generator, forward or
  backward (the same map on the output gradient), per element or shared over an axis (``noise_shape``).
* ``block``: d = dropout(scale * gate * post(x)); h = res + d; u = pre(h), post / pre being LayerNorm,
  RMSNorm or absent; inference (forward only) or training (forward, then every gradient).
* ``int4``: y = act(x @ dequant(w)^T + b) with 4-bit weights, a scale and optionally a zero point per
  group of inputs of each output.

Random bits: element i of a mask takes the (i & 7)-th 16-bit piece of Philox4x32-10 (Salmon, Moraes,
Dror, Shaw, SC11) at counter (i >> 3, step), both 64 bits wide, under the 64-bit seed as the key.  It is
kept when that piece is at least round(rate * 65536), and scaled by the inverse of the exact keep
probability.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_DEV = "cuda"


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _drop_case(name, dtype, shape, rate, direction, noise="", device_step=False):
    """shape / noise as "a,b,c" texts; noise "" draws a bit per element."""
    return {"name": name, "op": "dropout", "dtype": dtype, "shape": shape, "rate": rate, "dir": direction,
            "noise": noise, "device_step": device_step}


def _block_case(name, dtype, rows, cols, post, pre, gate, groups, res, scale, rate, train):
    """gate: "none", "vec" (one gate row for all rows) or "group" (``groups`` gate rows, each for
    rows / groups consecutive rows)."""
    return {"name": name, "op": "block", "dtype": dtype, "rows": rows, "cols": cols, "post": post, "pre": pre,
            "gate": gate, "groups": groups, "res": res, "scale": scale, "rate": rate, "train": train}


def _int4_case(name, batch, n, k, group, zero, act):
    return {"name": name, "op": "int4", "batch": batch, "n": n, "k": k, "group": group, "zero": zero, "act": act}


def listed():
    return [
        # the Dense(2048) activations of a batch of 32: the smallest call, launch latency counts
        _drop_case("drop-dense-b32", "bf16", "32,2048", 0.5, "fwd", device_step=True),
        # fp32 gradient of a narrow layer, sizes that divide by nothing
        _drop_case("drop-ragged-f32", "f32", "1031,2053", 0.1, "bwd"),
        # whole channels of image features dropped together (one bit per sample and channel)
        _drop_case("drop-channels", "bf16", "256,64,80,16", 0.2, "fwd", noise="256,1,1,16"),
        # pooled first-layer output of the image regressor at batch 256, every element its own bit
        _drop_case("drop-features", "bf16", "256,128,160,8", 0.25, "bwd"),
        # one row at a time while answering: post- and pre-norm around a gated residual join
        _block_case("block-one-row", "bf16", 1, 2048, "rms", "rms", "vec", 1, True, 0.5, 0.0, False),
        # an ordinary training step of a residual block boundary with everything in it
        _block_case("block-train", "bf16", 4096, 1024, "layer", "layer", "vec", 1, True, 0.7071, 0.1, True),
        # the largest activations that a wide residual tower trains on
        _block_case("block-train-large", "bf16", 32768, 2048, "none", "rms", "vec", 1, True, 1.0, 0.1, True),
        # LayerNorm alone over the 64 channels of 56 x 56 image features at batch 128
        _block_case("norm-features", "bf16", 401408, 64, "none", "layer", "none", 1, False, 1.0, 0.0, True),
        # fp32, odd sizes, a gate row for each sample's 29 rows, post-norm only
        _block_case("block-ragged-f32", "f32", 1537, 771, "layer", "none", "group", 53, True, 1.0, 0.25, True),
        # one image through the image regressor's Dense(2048) on 16 x 20 x 64 features
        _int4_case("int4-one-row", 1, 2048, 20480, 128, False, "relu"),
        # sixteen rows at a time through a wide layer, small groups with zero points
        _int4_case("int4-rows16", 16, 8192, 8192, 64, True, "linear"),
        # predict over a batch of 256 images through the same Dense(2048)
        _int4_case("int4-batch256", 256, 2048, 20480, 128, False, "relu"),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dropout", "block", "int4"])
    if op == "dropout":
        total = _logu(rng, 1, 1 << 24)
        inner = _logu(rng, 1, min(total, 4096))
        noise = ""
        if rng.random() < 0.3:  # one bit per sample and channel
            mid = max(1, _logu(rng, 1, max(1, total // inner)))
            outer = max(1, total // (inner * mid))
            shape, noise = f"{outer},{mid},{inner}", f"{outer},1,{inner}"
        else:
            shape = f"{max(1, total // inner)},{inner}"
        return {"op": op, "dtype": rng.choice(["bf16", "f32"]), "shape": shape,
                "rate": round(rng.uniform(0.0, 0.9), 3), "dir": rng.choice(["fwd", "bwd"]), "noise": noise,
                "device_step": rng.random() < 0.5}
    if op == "block":
        cols = _logu(rng, 8, 8192)
        if rng.random() < 0.6:
            cols = -(-cols // 8) * 8
        rows = _logu(rng, 1, max(1, min(100000, (1 << 25) // cols)))
        post, pre = rng.choice([("none", "layer"), ("none", "rms"), ("layer", "layer"), ("rms", "rms"),
                                ("layer", "none"), ("rms", "layer")])
        gate = rng.choice(["none", "vec", "group"])
        groups = 1
        if gate == "group":
            groups = rng.choice([1, rows, max(1, _logu(rng, 1, rows))])
            rows = groups * max(1, rows // groups)
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "f32"]), "rows": rows, "cols": cols, "post": post,
                "pre": pre, "gate": gate, "groups": groups, "res": rng.random() < 0.8,
                "scale": rng.choice([1.0, 0.5, 0.7071]), "rate": rng.choice([0.0, 0.1, 0.3]),
                "train": rng.random() < 0.7}
    group = rng.choice([32, 64, 128])
    k = -(-_logu(rng, group, 20480) // group) * group
    n = _logu(rng, 1, min(8192, max(1, (1 << 26) // k)))
    return {"op": op, "batch": _logu(rng, 1, 256), "n": n, "k": k, "group": group, "zero": rng.random() < 0.5,
            "act": rng.choice(["linear", "relu"])}


def _ints(text):
    return tuple(int(v) for v in text.split(","))


def work(case):
    if case["op"] == "dropout":
        n = math.prod(_ints(case["shape"]))
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * n * size, "flops": n}
    if case["op"] == "block":
        n = case["rows"] * case["cols"]
        size = 2 if case["dtype"] == "bf16" else 4
        ch = 4 * case["cols"]
        branch = case["res"] or case["gate"] != "none" or case["post"] != "none" or case["rate"] > 0 \
            or case["scale"] != 1.0
        vecs = sum(2 if s == "layer" else 1 if s == "rms" else 0 for s in (case["post"], case["pre"]))
        gate = {"none": 0, "vec": ch, "group": case["groups"] * case["cols"] * size}[case["gate"]]
        reads, writes = 1 + case["res"], int(branch) + (case["pre"] != "none")
        passes = reads + writes
        extra = vecs * ch + gate
        if case["train"]:  # the gradients of h and u come in, those of x and res go out
            passes += writes + reads + 1 + case["res"]
            extra += vecs * ch * 2 + gate * 2
        return {"bytes": passes * n * size + extra, "flops": n * (40 if case["train"] else 15)}
    b, n, k = case["batch"], case["n"], case["k"]
    groups = n * (k // case["group"])
    return {"bytes": n * k // 2 + groups * (3 if case["zero"] else 2) + 2 * b * (n + k) + 4 * n,
            "flops": 2 * b * n * k}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _ctr(seed):
    """A mask's (seed, step) from a case seed: 64 and 40 bits."""
    g = torch.Generator().manual_seed(seed * 2 + 1)
    v = torch.randint(0, 1 << 32, (3,), generator=g).tolist()
    return (v[0] << 32) | v[1], (v[2] << 8) | 1


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        t = torch.randn(shape, device=_DEV, dtype=torch.float32, generator=gen)
        return t.mul_(std).add_(mean).to(dtype)

    st = {"case": case}
    st["seed"], st["step"] = _ctr(seed)
    if case["op"] == "dropout":
        shape, dt = _ints(case["shape"]), _DT[case["dtype"]]
        st["x"] = normal(*shape, dtype=dt)
        st["out"] = torch.empty_like(st["x"])
        st["noise"] = _ints(case["noise"]) if case["noise"] else None
        if case["device_step"]:
            st["step_dev"] = torch.tensor([st["step"]], dtype=torch.int64, device=_DEV)
    elif case["op"] == "block":
        m, c, dt = case["rows"], case["cols"], _DT[case["dtype"]]
        st["x"] = normal(m, c, dtype=dt, std=1.5, mean=0.1)
        st["res"] = normal(m, c, dtype=dt, std=2.0) if case["res"] else None
        for side in ("post", "pre"):
            st[side] = None
            if case[side] != "none":
                st[side] = (normal(c, std=0.2, mean=1.0), normal(c, std=0.2) if case[side] == "layer" else None)
        st["gate"] = None
        if case["gate"] == "vec":
            st["gate"] = normal(c, std=0.3, mean=0.5)
        elif case["gate"] == "group":
            st["gate"] = normal(case["groups"], c, dtype=dt, std=0.3, mean=0.5)
        branch = case["res"] or st["gate"] is not None or st["post"] is not None or case["rate"] > 0 \
            or case["scale"] != 1.0
        st["branch"] = branch
        like = lambda t: None if t is None else torch.empty_like(t)  # noqa: E731
        st["h"] = like(st["x"]) if branch else None
        st["u"] = like(st["x"]) if st["pre"] is not None else None
        if case["train"]:
            st["dh"] = normal(m, c, dtype=dt, std=0.5) if branch else None
            st["du"] = normal(m, c, dtype=dt, std=0.5) if st["pre"] is not None else None
            st["dx"], st["dres"], st["dgate"] = like(st["x"]), like(st["res"]), like(st["gate"])
            for side in ("post", "pre"):
                st["d" + side] = None if st[side] is None else tuple(like(t) for t in st[side])
        if own:
            from pyspark_tf_gke_amd.ops import norm as NM

            st["stats"] = NM.block_norm_stats(m, _DEV) if case["train"] else None
            st["ws"] = NM.block_norm_workspace(m, c, case["groups"], _DEV) if case["train"] else None
    else:
        b, n, k, g = case["batch"], case["n"], case["k"], case["group"]
        st["x"] = normal(b, k, dtype=torch.bfloat16)
        q = normal(n, k, std=2.5, mean=8.0).round_().clamp_(0, 15).to(torch.uint8)
        st["codes"] = q[:, 0::2] | (q[:, 1::2] << 4)  # two inputs a byte, the even one low
        st["scale"] = normal(n, k // g, std=0.004, mean=0.02).to(torch.bfloat16)
        st["zero"] = torch.randint(5, 12, (n, k // g), device=_DEV, generator=gen).to(torch.uint8) \
            if case["zero"] else None
        st["bias"] = normal(n, std=0.1)
        st["out"] = torch.empty((b, n), dtype=torch.bfloat16, device=_DEV)
        if own:
            from pyspark_tf_gke_amd.ops import quant as Q

            st["w"] = Q.int4_layout(st["codes"], st["scale"], st["zero"], g)
            st["ws"] = Q.int4_workspace(b, st["w"])
    return st


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
_LOW = 0xFFFFFFFF


def _random16(n, seed, step):
    """The first n 16-bit pieces, as an int64 tensor."""
    g = torch.arange((n + 7) // 8, dtype=torch.int64, device=_DEV)
    c0, c1 = g & _LOW, (g >> 32) & _LOW
    c2, c3 = torch.full_like(g, step & _LOW), torch.full_like(g, (step >> 32) & _LOW)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        # a 64-bit product wraps into the sign, its upper half comes back with the mask
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW)
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]


def _keep(shape, rate, seed, step, noise=None):
    """(keep mask broadcastable to shape, scale of what is kept)."""
    noise = noise or tuple(shape)
    thr = int(round(rate * 65536))
    keep = (_random16(math.prod(noise), seed, step) >= thr).view(noise)
    return keep, 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def _norm(v, kind, params):
    """(normalised and affine v, xhat, rstd) along the rows, fp32."""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS[kind])
    xhat = v * rstd
    out = xhat * params[0]
    return (out + params[1] if params[1] is not None else out), xhat, rstd


def _norm_grad(g, kind, params, xhat, rstd):
    """(d input, d gamma, d beta) of _norm."""
    gg = g * params[0]
    dv = gg - xhat * (gg * xhat).mean(1, keepdim=True)
    if kind == "layer":
        dv = dv - gg.mean(1, keepdim=True)
    return dv * rstd, (g * xhat).sum(0), g.sum(0) if params[1] is not None else None


_EPS = {"layer": 1e-3, "rms": 1e-6}


def _plain_block(st):
    c = st["case"]
    dt = st["x"].dtype
    m, groups = c["rows"], c["groups"]
    x = st["x"].float()
    n, xh1, rs1 = _norm(x, c["post"], st["post"]) if st["post"] is not None else (x, None, None)
    gate = st["gate"]
    if gate is not None:
        gate = gate.float()
        gate = gate.repeat_interleave(m // groups, 0) if gate.dim() == 2 else gate
    d = n * c["scale"] if gate is None else n * gate * c["scale"]
    mask = None
    if c["rate"] > 0:
        keep, k = _keep(x.shape, c["rate"], st["seed"], st["step"])
        mask = keep.float() * k
        d = d * mask
    h = d if st["res"] is None else d + st["res"].float()
    out = {"h": h.to(dt) if st["branch"] else None}
    u = xh2 = rs2 = None
    if st["pre"] is not None:
        u, xh2, rs2 = _norm(h, c["pre"], st["pre"])
    out["u"] = None if u is None else u.to(dt)
    if not c["train"]:
        return out
    dh = st["dh"].float() if st["dh"] is not None else torch.zeros_like(h)
    if st["pre"] is not None:
        dv, dg, db = _norm_grad(st["du"].float(), c["pre"], st["pre"], xh2, rs2)
        dh = dh + dv
        out["dpre"] = (dg, db)
    out["dres"] = dh.to(dt) if st["res"] is not None else None
    dd = dh if mask is None else dh * mask
    if gate is not None:
        dg = dd * n * c["scale"]
        out["dgate"] = dg.sum(0) if st["gate"].dim() == 1 else dg.view(groups, m // groups, -1).sum(1).to(dt)
        dn = dd * gate * c["scale"]
    else:
        dn = dd * c["scale"]
    if st["post"] is not None:
        dn, dg, db = _norm_grad(dn, c["post"], st["post"], xh1, rs1)
        out["dpost"] = (dg, db)
    out["dx"] = dn.to(dt)
    return out


def _dequant(st, dtype):
    c = st["case"]
    q = torch.stack((st["codes"] & 15, st["codes"] >> 4), 2).view(c["n"], c["k"] // c["group"], c["group"]).to(dtype)
    z = st["zero"].to(dtype)[:, :, None] if st["zero"] is not None else 8.0
    return ((q - z) * st["scale"].to(dtype)[:, :, None]).view(c["n"], c["k"])


def _plain(st):
    c = st["case"]
    if c["op"] == "dropout":
        keep, k = _keep(st["x"].shape, c["rate"], st["seed"], st["step"], st["noise"])
        return torch.where(keep, st["x"].float() * k, 0.0).to(st["x"].dtype)
    if c["op"] == "block":
        return _plain_block(st)
    y = st["x"].float() @ _dequant(st, torch.float32).t() + st["bias"]
    return (torch.relu(y) if c["act"] == "relu" else y).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------
# the framework's operators
# ------------------------------------------------------------------------------------------------
def _own(st):
    c = st["case"]
    if c["op"] == "dropout":
        from pyspark_tf_gke_amd.ops import dropout as DR

        fn = DR.dropout_fwd if c["dir"] == "fwd" else DR.dropout_bwd
        return fn(st["x"], c["rate"], st["seed"], st.get("step_dev", st["step"]), st["out"], st["noise"])
    if c["op"] == "int4":
        from pyspark_tf_gke_amd.ops import quant as Q

        return Q.int4_dense_fwd(st["x"], st["w"], st["bias"], c["act"], st["out"], workspace=st["ws"])
    from pyspark_tf_gke_amd.ops import dropout as DR
    from pyspark_tf_gke_amd.ops import norm as NM

    sides = {s: None if st[s] is None else NM.Norm(c[s], st[s][0], st[s][1], _EPS[c[s]]) for s in ("post", "pre")}
    drop = DR.Drop(c["rate"], st["seed"], st["step"]) if c["rate"] > 0 else None
    NM.block_norm_fwd(st["x"], res=st["res"], gate=st["gate"], scale=c["scale"], drop=drop, h=st["h"], u=st["u"],
                      stats=st["stats"], **sides)
    out = {"h": st["h"], "u": st["u"]}
    if not c["train"]:
        return out
    NM.block_norm_bwd(st["x"], st["stats"], res=st["res"], gate=st["gate"], scale=c["scale"], drop=drop, du=st["du"],
                      dh=st["dh"], dx=st["dx"], dres=st["dres"], dgate=st["dgate"], dpost=st["dpost"],
                      dpre=st["dpre"], workspace=st["ws"], **sides)
    return _block_out(st, out, st["dpre"], st["dres"], st["dgate"], st["dpost"], st["dx"])


def _block_out(st, out, dpre, dres, dgate, dpost, dx):
    if st["pre"] is not None:
        out["dpre"] = dpre
    out["dres"] = dres
    if st["gate"] is not None:
        out["dgate"] = dgate
    if st["post"] is not None:
        out["dpost"] = dpost
    out["dx"] = dx
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------
# exact values, 64 bits
# ------------------------------------------------------------------------------------------------
def _mul32(a, k):
    """(upper, lower) 32 bits of a * k from 16-bit limbs, a an int64 tensor below 2**32."""
    al, ah, kl, kh = a & 0xFFFF, a >> 16, k & 0xFFFF, k >> 16
    ll, lh, hl, hh = al * kl, al * kh, ah * kl, ah * kh
    mid = (ll >> 16) + (lh & 0xFFFF) + (hl & 0xFFFF)
    return hh + (lh >> 16) + (hl >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (ll & 0xFFFF)


def _exact_mask(numel, rate, seed, step):
    """0 or 1/p of each element, float64."""
    blocks = torch.arange(-(-numel // 8), dtype=torch.int64, device=_DEV)
    x = [blocks % 2**32, blocks // 2**32, torch.zeros_like(blocks) + step % 2**32,
         torch.zeros_like(blocks) + step // 2**32]
    for r in range(10):
        ka, kb = (seed % 2**32 + r * 0x9E3779B9) % 2**32, (seed // 2**32 + r * 0xBB67AE85) % 2**32
        ha, la = _mul32(x[0], 0xD2511F53)
        hb, lb = _mul32(x[2], 0xCD9E8D57)
        x = [hb ^ x[1] ^ ka, lb, ha ^ x[3] ^ kb, la]
    bits = torch.empty((blocks.numel(), 8), dtype=torch.int64, device=_DEV)
    for j in range(8):
        bits[:, j] = (x[j // 2] // 65536 ** (j % 2)) % 65536
    drop = round(rate * 65536)
    inv = 65536 / (65536 - drop) if drop < 65536 else 0.0
    return (bits.view(-1)[:numel] >= drop).double() * inv


def _exact_norm(v, kind, gamma, beta):
    mu = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    y = (v - mu) / torch.sqrt(((v - mu) ** 2).mean(1, keepdim=True) + _EPS[kind]) * gamma
    return y if beta is None else y + beta


def _exact_block(case, st):
    leaf = lambda t: None if t is None else t.double().requires_grad_(case["train"])  # noqa: E731
    x, res, gate = leaf(st["x"]), leaf(st["res"]), leaf(st["gate"])
    post = None if st["post"] is None else tuple(leaf(t) for t in st["post"])
    pre = None if st["pre"] is None else tuple(leaf(t) for t in st["pre"])
    d = x if post is None else _exact_norm(x, case["post"], *post)
    if gate is not None:
        per = case["rows"] // case["groups"]
        d = (d.view(case["groups"], per, -1) * gate.view(-1, 1, case["cols"])).view(x.shape) if gate.dim() == 2 \
            else d * gate
    d = d * case["scale"]
    if case["rate"] > 0:
        d = d * _exact_mask(d.numel(), case["rate"], st["seed"], st["step"]).view(d.shape)
    h = d if res is None else res + d
    u = None if pre is None else _exact_norm(h, case["pre"], *pre)
    out = {"h": h.detach() if st["branch"] else None, "u": None if u is None else u.detach()}
    if not case["train"]:
        return out
    roots = [(t, st[g].double()) for t, g in ((h, "dh"), (u, "du")) if st[g] is not None]
    torch.autograd.backward([t for t, _ in roots], [g for _, g in roots])
    grad = lambda t: None if t is None else t.grad  # noqa: E731
    pair = lambda p: None if p is None else tuple(grad(t) for t in p)  # noqa: E731
    return _block_out(st, out, pair(pre), grad(res), grad(gate), pair(post), grad(x))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dropout":
        noise = st["noise"] or tuple(st["x"].shape)
        mask = _exact_mask(math.prod(noise), case["rate"], st["seed"], st["step"]).view(noise)
        return st["x"].double() * mask
    if case["op"] == "block":
        return _exact_block(case, st)
    n, k, g = case["n"], case["k"], case["group"]
    w = torch.empty((n, k), dtype=torch.float64, device=_DEV)
    w[:, 0::2] = (st["codes"] % 16).double()
    w[:, 1::2] = (st["codes"] // 16).double()
    w = w.view(n, k // g, g)
    w -= 8.0 if st["zero"] is None else st["zero"].double().unsqueeze(2)
    w *= st["scale"].double().unsqueeze(2)
    y = torch.matmul(st["x"].double(), w.view(n, k).t()) + st["bias"].double()
    return y.clamp_min(0.0) if case["act"] == "relu" else y
