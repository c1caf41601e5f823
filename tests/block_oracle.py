"""float64 autograd oracle of models with dropout, row norms, gates and residual scales (test helper)."""
import numpy as np
import torch
import torch.nn.functional as F

import rng_oracle as O
from pyspark_tf_gke_amd.nn import layers as L
from pyspark_tf_gke_amd.ops import dropout as D


def _mask(l, shape, step):
    noise = l.noise_shape
    full = tuple(s if v is None else v for v, s in zip(noise, shape)) if noise else tuple(shape)
    seed = D.mix_seed(l.seed_value(), 0)
    return torch.from_numpy(O.keep(O.shared_index(tuple(shape), full), l.rate, seed, step)).double() * O.scale(l.rate)


def _norm(l, a, params):
    if isinstance(l, L.LayerNormalization):
        a = a - a.mean(-1, keepdim=True)
    y = a / torch.sqrt((a * a).mean(-1, keepdim=True) + l.epsilon)
    g = params.get(f"{l.name}/gamma", params.get(f"{l.name}/scale"))
    y = y if g is None else y * g
    return y + params[f"{l.name}/beta"] if f"{l.name}/beta" in params else y


def apply_layer(l, ins, params, step, training):
    a = ins[0]
    if isinstance(l, L.Dense):
        z = a @ params[f"{l.name}/kernel"].t()
        z.retain_grad()
        l._oracle = (a, z)
        v = z + params[f"{l.name}/bias"]
        return torch.relu(v) if l.activation == "relu" else v
    if isinstance(l, (L.LayerNormalization, L.RMSNormalization)):
        return _norm(l, a, params)
    if isinstance(l, L.Dropout):
        return a * _mask(l, a.shape, step) if training else a
    if isinstance(l, L.LayerScale):
        return a * params[f"{l.name}/gamma"]
    if isinstance(l, L.Rescaling):
        return a * l.scale
    if isinstance(l, L.Multiply):
        g = ins[1]
        return a * (g if g.dim() == a.dim() else g.view(g.shape[0], *([1] * (a.dim() - 2)), g.shape[1]))
    if isinstance(l, L.Add):
        return ins[0] + ins[1]
    if isinstance(l, L.Flatten):
        return a.reshape(a.shape[0], -1)
    if isinstance(l, L.GlobalAveragePooling2D):
        return a.mean((1, 2))
    if isinstance(l, L.Conv2D):
        w = params[f"{l.name}/kernel"][..., : l.cin].permute(0, 3, 1, 2)
        v = F.conv2d(a.permute(0, 3, 1, 2), w, params.get(f"{l.name}/bias"), padding=l.pad_amount())
        v = v.permute(0, 2, 3, 1)
        return torch.relu(v) if l.activation == "relu" else v
    raise NotImplementedError(type(l).__name__)


def run(model, x, y, step, training=True, spread=None):
    """(output, loss, {parameter: gradient}) in float64 (mean squared error).  ``spread`` (a dict): takes, for
    every parameter of a model of [batch, C] tensors, the root of the sum of the squares of the samples'
    contributions to its gradient."""
    params = {p.name: p.data.detach().double().cpu().clone() for p in model.store.params}
    if spread is not None:  # a copy of each vector for each sample
        params = {k: v.expand(len(x), -1).clone() if v.dim() == 1 else v for k, v in params.items()}
    for v in params.values():
        v.requires_grad_(True)
    x = torch.as_tensor(np.asarray(x)).double()
    if hasattr(model, "nodes"):
        vals = {}
        for t in model.nodes:
            vals[id(t)] = x if isinstance(t.layer, L.Input) else \
                apply_layer(t.layer, [vals[id(i)] for i in t.inputs], params, step, training)
        out = vals[id(model.nodes[-1])]
    else:
        out = x
        for l in model.layers:
            out = apply_layer(l, [out], params, step, training)
    loss = ((out - torch.as_tensor(np.asarray(y)).double()) ** 2).mean()
    loss.backward()
    grads = {k: v.grad for k, v in params.items() if v.grad is not None}
    if spread is not None:
        for p in model.store.params:
            if len(p.shape) == 1 and p.name in grads:
                spread[p.name] = grads[p.name].pow(2).sum(0).sqrt()
                grads[p.name] = grads[p.name].sum(0)
        for l in model.layers:
            if isinstance(l, L.Dense):
                a, z = l._oracle
                spread[f"{l.name}/kernel"] = ((z.grad ** 2).t() @ (a.detach() ** 2)).sqrt()
    return out.detach(), float(loss.detach()), grads
