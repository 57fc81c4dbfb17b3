"""Float64 values of the operators that are one node each (tensor-compiler-webgpu_amd/js/src/ir/operators.js) —
TEST INFRASTRUCTURE ONLY. The reference has none of them, so nothing of its pins these: they restate the formulas, and
their gradients are checked against differences of their values (tests/test_operators.py).

Each function takes a node ({op, inputs, attrs, shape}), its operands' values (flat) and shapes, and gives the node's
value, flat. What each is: see the node rules' own comment; rows that a loss leaves out count as 0, whatever they hold.
"""
from __future__ import annotations

from typing import List

import numpy as np


def turned(attrs, x_shape, positions, p_shape):
    """cos and sin of every row's angles, broadcastable to x's axes but the last, then the pairs."""
    axis, r = attrs["axis"], len(x_shape)
    f, axes = np.asarray(attrs["frequencies"], dtype=np.float64), np.asarray(attrs["axes"], dtype=int)
    many = attrs["positionAxes"] > 1
    p = positions.reshape(p_shape if many else list(p_shape) + [1])
    angle = p[..., axes] * f if len(f) else np.zeros(p.shape[:-1] + (0,))
    shape = [1] * (r - 1) + [len(f)]
    shape[axis] = x_shape[axis]
    if p.ndim == 3:
        shape[0] = x_shape[0]
    angle = angle.reshape(shape)
    return np.cos(angle), np.sin(angle)


def pair_dims(attrs, dh):
    R = len(attrs["frequencies"])
    if attrs["pairs"] == "adjacent":
        return np.arange(0, 2 * R, 2), np.arange(1, 2 * R, 2)
    return np.arange(R), np.arange(R, 2 * R)


def turn(attrs, v, cos, sin):
    a, b = pair_dims(attrs, v.shape[-1])
    out = v.copy()
    out[..., a] = v[..., a] * cos - v[..., b] * sin
    out[..., b] = v[..., b] * cos + v[..., a] * sin
    return out


def rotary(node, args: List[np.ndarray], shapes):
    x = args[0].reshape(shapes[0])
    cos, sin = turned(node["attrs"], shapes[0], args[1], shapes[1])
    if len(args) == 3:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + node["attrs"]["eps"]) * args[2]
    return turn(node["attrs"], x, cos, sin).reshape(-1)


def rotary_grad(node, args, shapes):
    attrs = node["attrs"]
    x, dy = args[0].reshape(shapes[0]), args[-1].reshape(shapes[0])
    cos, sin = turned(attrs, shapes[0], args[1], shapes[1])
    dn = turn(attrs, dy, cos, -sin)
    if len(args) == 3:
        return dn.reshape(-1)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + attrs["eps"])
    h = x * r
    if attrs["part"] == "dgain":
        return (dn * h).reshape(-1, shapes[0][-1]).sum(0)
    g = dn * args[2]
    return (r * (g - h * (g * h).mean(-1, keepdims=True))).reshape(-1)


def loss_parts(args, shapes):
    """(h with the rows left out as 0, W, kept, target, logits - maximum, sum of exponentials)."""
    V = shapes[1][1]
    t = args[2]
    kept = (t >= 0) & (t < V) & (t == np.floor(t))
    h = np.where(kept[:, None], args[0].reshape(shapes[0]), 0.0)
    W = args[1].reshape(shapes[1])
    z = h @ W
    if len(shapes) > 3 and len(shapes[3]) == 1 and shapes[3][0] == V:
        z = z + args[3]
    z = z - z.max(1, keepdims=True)
    return h, W, kept, np.where(kept, t, 0).astype(int), z, np.exp(z).sum(1)


def linear_cross_entropy(node, args, shapes):
    _, _, kept, t, z, s = loss_parts(args, shapes)
    return np.where(kept, np.log(s) - z[np.arange(len(t)), t], 0.0)


def linear_cross_entropy_grad(node, args, shapes):
    # Without a bias the fourth operand is the losses' gradient: never mistaken for one, even where N equals V.
    head = 4 if len(args) == 5 else 3
    h, W, kept, t, z, s = loss_parts(args[:head], shapes[:head])
    g = np.exp(z) / s[:, None]
    g[np.arange(len(t)), t] -= 1
    g = np.where(kept[:, None], g * np.where(kept, args[-1], 0.0)[:, None], 0.0)
    part = node["attrs"]["part"]
    return (g @ W.T if part == "dh" else h.T @ g if part == "dW" else g.sum(0)).reshape(-1)


def orthogonalize(node, args, shapes):
    a, b, c = node["attrs"]["coefficients"]
    x = args[0].reshape([-1] + list(shapes[0][-2:]))
    x = x / (np.sqrt((x * x).sum((1, 2), keepdims=True)) + node["attrs"]["eps"])
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(0, 2, 1) if tall else x
    for _ in range(node["attrs"]["steps"]):
        A = x @ x.transpose(0, 2, 1)
        x = a * x + (b * A + c * (A @ A)) @ x
    return (x.transpose(0, 2, 1) if tall else x).reshape(-1)


KERNELS = {"rotary": rotary, "rotaryGrad": rotary_grad, "linearCrossEntropy": linear_cross_entropy,
           "linearCrossEntropyGrad": linear_cross_entropy_grad, "orthogonalize": orthogonalize}
