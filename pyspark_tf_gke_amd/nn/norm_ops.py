"""Device ops of the Dropout, LayerNormalization / RMSNormalization, LayerScale, Multiply and Rescaling
layers (:mod:`..ops.dropout`, :mod:`..ops.norm`).

A residual block boundary ``[norm] -> [LayerScale | Multiply(gate)] -> [Rescaling] -> [Dropout] ->
Add(stream) -> [norm]`` lowers to ONE :class:`BlockOp`: a forward pass that reads the block's output and
the stream and writes the new stream and the next block's normalised input, and a backward pass that
draws the dropout mask again instead of reading one.  Any part alone is the same op with the others absent.
"""
from __future__ import annotations

import torch

from ..ops import dropout as DR
from ..ops import norm as NM
from . import engine as E
from . import layers as L


class DropState:
    """The training step that a model's dropout masks are drawn at: one int64 on the device, shared by
    the model's dropout ops and advanced by the first of them in every training forward pass (a kernel,
    so a captured step draws new masks every replay).  The backward pass reads the same step."""

    def __init__(self):
        self.step = None
        self.start = 0

    def tensor(self, device):
        if self.step is None or self.step.device != torch.device(device):
            self.step = torch.full((1,), self.start, dtype=torch.int64, device=device)
        return self.step

    def get(self) -> int:
        return self.start if self.step is None else int(self.step)

    def set(self, value: int) -> None:
        self.start = int(value)
        if self.step is not None:
            self.step.fill_(self.start)

    def advance(self, device) -> None:
        DR.drop_advance(self.tensor(device))


def drop_state(ops):
    """The DropState of a plan's ops (None: no dropout)."""
    for op in ops:
        s = getattr(getattr(op, "inner", getattr(op, "op", op)), "drop_state", None)
        if s is not None:
            return s
    return None


def bind_drop_state(ops) -> None:
    """Give a plan's dropout ops one DropState; the first of them advances it."""
    st = None
    for op in ops:
        op = getattr(op, "inner", getattr(op, "op", op))
        if getattr(op, "drop", None) is not None:
            op.leads = st is None
            st = st or DropState()
            op.drop_state = st


def _drop_now(op, dev):
    """The dropout of this training pass (data-parallel ranks draw different masks), or None."""
    if op.drop is None:
        return None
    if op.leads:
        op.drop_state.advance(dev)
    if op.drop.rate == 0.0:
        return None
    if op.seed is None:
        from ..parallel import comm

        op.seed = DR.mix_seed(op.drop.seed_value(), comm.rank())
    return DR.Drop(op.drop.rate, op.seed, op.drop_state.tensor(dev))


def _float(x, ws, key, dtype=None):
    """x contiguous in ``dtype`` (None: fp32 stays, everything else becomes bf16)."""
    if dtype is None:
        dtype = torch.float32 if x.dtype == torch.float32 else torch.bfloat16
    if x.dtype == dtype:
        return x.contiguous()
    if dtype == torch.bfloat16:
        return E._bf16(x, ws, key).contiguous()
    out = ws.get(key, x.shape, dtype, x.device)
    out.copy_(x)
    return out


class DropoutOp(E.Op):
    drop_state = seed = None
    leads = False

    def __init__(self, layer: L.Dropout):
        super().__init__()
        self.drop = layer
        self.name = layer.name

    def forward(self, x, ws, training):
        self._d = _drop_now(self, x.device) if training else None
        if self._d is None:
            return x
        x = _float(x, ws, self.name + "/x16")
        y = ws.get(self.name + "/y", x.shape, x.dtype, x.device)
        self._shape = x.shape  # the mask goes by it
        return DR.dropout_fwd(x, self._d.rate, self._d.seed, self._d.step, y, self.drop.noise_shape)

    def backward(self, dy, ws):
        if self._d is None or self.first:
            return dy
        if dy.numel() != self._shape.numel():
            raise ValueError(f"{self.name}: a gradient of shape {tuple(dy.shape)} for an output of {tuple(self._shape)}")
        dy = _float(dy, ws, self.name + "/dy16").reshape(self._shape)
        dx = ws.get(self.name + "/dx", dy.shape, dy.dtype, dy.device)
        return DR.dropout_bwd(dy, self._d.rate, self._d.seed, self._d.step, dx, self.drop.noise_shape)


class BlockOp:
    """``forward([x] + [gate] + [res])`` -> [h][u] (those that are wanted); ``backward`` takes their
    gradients (None where nothing came back) and returns those of the inputs."""

    first = False
    drop_state = seed = None
    leads = False

    def __init__(self, name, post=None, gate=None, gate_input=False, scale=1.0, drop=None, res=False, pre=None,
                 want_h=True):
        self.name = name
        self.post, self.gate, self.gate_input, self.scale = post, gate, gate_input, float(scale)
        self.drop, self.res, self.pre, self.want_h = drop, res, pre, want_h
        self.params = [p for l in (post, gate, pre) if l is not None for p in l.params]
        for p in self.params:
            p.overwrite_grad = True  # the backward pass writes whole gradients
        if not want_h and pre is None:
            raise ValueError(f"{name}: no output")

    @staticmethod
    def _norm(layer):
        if layer is None:
            return None
        beta = getattr(layer, "beta", None)
        return NM.Norm(layer.norm_kind, None if layer.gamma is None else layer.gamma.data,
                       None if beta is None else beta.data, layer.epsilon)

    def _prep_input(self, x, ws):
        return _float(x, ws, self.name + "/x16")

    def forward(self, xs, ws, training):
        dt = torch.float32 if all(t.dtype == torch.float32 for t in xs) else torch.bfloat16
        names = ["/x16"] + (["/gate16"] if self.gate_input else []) + (["/res16"] if self.res else [])
        xs = [_float(t, ws, self.name + n, dt) for t, n in zip(xs, names)]
        x = xs[0]
        dt, dev = x.dtype, x.device
        gate = xs[1].reshape(-1, x.shape[-1]) if self.gate_input else \
            self.gate.gamma.data if self.gate is not None else None
        res = xs[-1] if self.res else None
        d = _drop_now(self, dev) if training else None
        h = ws.get(self.name + "/h", x.shape, dt, dev) if self.want_h else None
        u = ws.get(self.name + "/u", x.shape, dt, dev) if self.pre is not None else None
        st = None
        if training and (self.post is not None or self.pre is not None):
            st = ws.get(self.name + "/stats", (4, x.numel() // x.shape[-1]), torch.float32, dev)
        self._kw = dict(res=res, post=self._norm(self.post), gate=gate, scale=self.scale, drop=d,
                        pre=self._norm(self.pre))
        self._x, self._st, self._gshape = x, st, xs[1].shape if self.gate_input else None
        if self._wide(x):
            NM.flat_fwd(x, res=res, gate=gate, scale=self.scale, drop=d, h=h)
        else:
            NM.block_norm_fwd(x, h=h, u=u, stats=st, **self._kw)
        return [t for t in (h, u) if t is not None]

    # Rows above the kernels' width, without a norm or a gate vector: elementwise.
    def _wide(self, x) -> bool:
        return x.shape[-1] > NM.MAX_COLS and self.post is None and self.pre is None and self.gate is None \
            and (not self.gate_input or self._kw["gate"].numel() == x.numel())

    def _grads(self, layer):
        if layer is None:
            return None
        beta = getattr(layer, "beta", None)
        return (None if layer.gamma is None else layer.gamma.grad, None if beta is None else beta.grad)

    def backward(self, gs, ws, existing=None):
        x, st, kw = self._x, self._st, self._kw
        n_in = 1 + self.gate_input + self.res
        if self.first and not self.params:
            return [None] * n_in
        gs = list(gs)
        dh = gs.pop(0) if self.want_h else None
        du = gs.pop(0) if self.pre is not None else None
        dt, dev = x.dtype, x.device
        dh = None if dh is None else _float(dh, ws, self.name + "/dh16", dt).reshape(x.shape)
        if self.pre is not None and du is None:
            du = ws.get(self.name + "/du0", x.shape, dt, dev)  # the normalised output led nowhere
            du.zero_()
        du = None if du is None else _float(du, ws, self.name + "/du16", dt).reshape(x.shape)
        dx = None if self.first else ws.get(self.name + "/dx", x.shape, dt, dev)
        dres = ws.get(self.name + "/dres", x.shape, dt, dev) if self.res and not self.first else None
        dgate = None
        if self.gate_input:
            dgate = ws.get(self.name + "/dgate", kw["gate"].shape, dt, dev)
        elif self.gate is not None:
            dgate = self.gate.gamma.grad
        if self._wide(x):
            NM.flat_bwd(x, gate=kw["gate"], scale=self.scale, drop=kw["drop"], dh=dh, dx=dx, dres=dres, dgate=dgate)
        else:
            wsp = None
            if x.is_cuda:
                C = x.shape[-1]
                G = kw["gate"].shape[0] if self.gate_input else 1
                floats = NM.block_norm_workspace_floats(x.numel() // C, C, G)
                wsp = ws.get(self.name + "/colsums", (floats,), torch.float32, dev)
            NM.block_norm_bwd(x, st, du=du, dh=dh, dx=dx, dres=dres, dgate=dgate, dpost=self._grads(self.post),
                              dpre=self._grads(self.pre), workspace=wsp, **kw)
        return [dx] + ([dgate.view(self._gshape)] if self.gate_input else []) + ([dres] if self.res else [])


class SeqBlockOp(E.Op):
    """A single-input :class:`BlockOp` in the Sequential engine (and behind a graph Adapter)."""

    def __init__(self, op: BlockOp):
        super().__init__()
        self.op = op
        self.params = op.params
        self.name = op.name

    def forward(self, x, ws, training):
        self.op.first = self.first
        return self.op.forward([x], ws, training)[0]

    def backward(self, dy, ws):
        return self.op.backward([dy], ws)[0]


class BlockNode:
    """Graph node of a :class:`BlockOp`: one or two outputs (the stream h, the normalised u)."""

    def __init__(self, op: BlockOp, inputs, outputs):
        self.op, self.inputs, self.outputs = op, inputs, outputs
        self.output = outputs[-1]
        self.params = op.params
        self.name = op.name

    @property
    def first(self):
        return self.op.first

    @first.setter
    def first(self, v):
        self.op.first = v

    def forward(self, xs, ws, training):
        return self.op.forward(xs, ws, training)

    def backward(self, gs, ws, existing):
        return self.op.backward(gs, ws, existing)

    def _prep_input(self, x, ws):
        return self.op._prep_input(x, ws)


def bare(op) -> bool:
    """A Dropout, Rescaling or Multiply op (no weights): what reads the model's input through it alone is as good
    as first."""
    op = getattr(op, "inner", getattr(op, "op", op))
    return isinstance(op, (DropoutOp, SeqBlockOp, BlockOp)) and not op.params


def is_norm(layer) -> bool:
    return isinstance(layer, (L.LayerNormalization, L.RMSNormalization))


class Chain:
    """The parts of a block boundary collected one layer after another; :meth:`take` refuses what does not
    fit behind what is there (a norm only in front, one gate, one dropout)."""

    def __init__(self):
        self.post = self.gate = self.drop = None
        self.gate_input = False
        self.scale = 1.0
        self.layers = []

    def take(self, layer) -> bool:
        if is_norm(layer):
            ok = not self.layers
            self.post = layer if ok else self.post
        elif isinstance(layer, (L.LayerScale, L.Multiply)):
            ok = self.gate is None and not self.gate_input
            if ok and isinstance(layer, L.Multiply):
                self.gate_input = True
            elif ok:
                self.gate = layer
        elif isinstance(layer, L.Rescaling):
            ok = True
            self.scale *= layer.scale
        elif isinstance(layer, L.Dropout):
            ok = self.drop is None and layer.noise_shape is None
            self.drop = layer if ok else self.drop
        else:
            ok = False
        if ok:
            self.layers.append(layer)
        return ok

    def op(self, res=False, pre=None, want_h=True):
        post = self.post
        if len(self.layers) == 1 and post is not None and not res and pre is None:
            post, pre, want_h = None, post, False  # a norm alone: no stream to write
        return BlockOp(self.layers[0].name if self.layers else pre.name, post, self.gate, self.gate_input, self.scale,
                       self.drop, res, pre, want_h)
