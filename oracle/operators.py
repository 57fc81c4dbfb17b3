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


def embedding(node, args, shapes):
    t, table = args[0], args[1].reshape(shapes[1])
    kept = (t >= 0) & (t < len(table)) & (t == np.floor(t))
    return np.where(kept[:, None], table[np.where(kept, t, 0).astype(int)] * node["attrs"]["scale"], 0.0).reshape(-1)


def embedding_grad(node, args, shapes):
    rows, d = node["attrs"]["rows"], shapes[1][-1]
    t, dy = args[0], args[1].reshape(-1, shapes[1][-1])
    kept = np.flatnonzero((t >= 0) & (t < rows) & (t == np.floor(t)))
    out = np.zeros((rows, d))
    np.add.at(out, t[kept].astype(int), dy[kept])
    return (out * node["attrs"]["scale"]).reshape(-1)


def residual_operands(node, args, shapes):
    """Operands by name, rows as [N, d] (a gate of [d] broadcasts)."""
    a = node["attrs"]
    grad = node["op"] == "residualNormGrad"
    names = ["x", "y"] + [n for n, on in (("gain", a["pre"]), ("bias", a["bias"] and not grad), ("postGain", a["post"]), ("postBias", a["postBias"]), ("gate", a["gate"])) if on]
    names += a["has"] if grad else []
    d = shapes[0][-1]
    return {n: v.reshape(-1, d) for n, v in zip(names, args)}


def normalised(attrs, v):
    """(1 / deviation, the rows over it)."""
    c = v - v.mean(1, keepdims=True) if attrs["norm"] == "layer" else v
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True) + attrs["eps"])
    return r, c * r


def residual_rows(node, v):
    a = node["attrs"]
    p = normalised(a, v["y"])[1] * v["postGain"] + v.get("postBias", 0.0) if a["post"] else v["y"]
    return p, a["residual"] * v["x"] + v.get("gate", 1.0) * p


def residual_norm(node, args, shapes):
    v = residual_operands(node, args, shapes)
    h = residual_rows(node, v)[1]
    return (h if node["attrs"]["part"] == "h" else normalised(node["attrs"], h)[1] * v["gain"] + v.get("bias", 0.0)).reshape(-1)


def residual_norm_grad(node, args, shapes):
    a, v = node["attrs"], residual_operands(node, args, shapes)
    p, h = residual_rows(node, v)

    def back(r, hat, g):
        return r * (g - hat * (g * hat).mean(1, keepdims=True) - (g.mean(1, keepdims=True) if a["norm"] == "layer" else 0.0))

    dh, part = v.get("dh", 0.0), a["part"]
    if "dn" in v:
        r, hat = normalised(a, h)
        if part in ("dgain", "dbias"):
            return (v["dn"] * hat if part == "dgain" else v["dn"]).sum(0)
        dh = dh + back(r, hat, v["dn"] * v["gain"])
    if part == "dx":
        return (a["residual"] * dh).reshape(-1)
    if part == "dgate":
        return (dh * p).reshape(-1) if v["gate"].shape == p.shape and len(shapes[list(v).index("gate")]) == len(shapes[0]) else (dh * p).sum(0)
    dp = dh * v.get("gate", 1.0)
    if not a["post"]:
        return dp.reshape(-1)
    r, hat = normalised(a, v["y"])
    return {"dpostGain": lambda: (dp * hat).sum(0), "dpostBias": lambda: dp.sum(0), "dy": lambda: back(r, hat, dp * v["postGain"]).reshape(-1)}[part]()


def window_sees(node, args, shapes):
    """[B, T, S]: whether a query sees a key."""
    a = node["attrs"]
    (B, T), S = shapes[0][:2], shapes[1][1]
    length = np.full(B, S)
    if len(shapes) in (4, 7):
        length = np.floor(np.clip(np.nan_to_num(args[3], nan=0.0, posinf=S, neginf=0.0), 0, S)).astype(int)
    at = np.arange(T)[None, :] + (0 if a["queries"] == "first" else length[:, None] - T)
    at, j, length = at[:, :, None], np.arange(S)[None, None], length[:, None, None]
    near = (at - j < a["window"]) if a["window"] else True
    return (j <= at) & (near | (j < a["sinks"])) & (at >= 0) & (at < length)


def window_values(node, args, shapes):
    """(sees, q, k, v, scores) as [B, H, rows, ...] with what nothing sees as 0."""
    sees = window_sees(node, args, shapes)
    R = shapes[0][2] // shapes[1][2]
    q, k, v = (args[i].reshape(shapes[i]).transpose(0, 2, 1, 3) for i in range(3))
    q = np.where(sees.any(2)[:, None, :, None], q, 0.0)
    k, v = (np.repeat(np.where(sees.any(1)[:, None, :, None], x, 0.0), R, 1) for x in (k, v))
    return sees[:, None], q, k, v, node["attrs"]["scale"] * (q @ k.transpose(0, 1, 3, 2))


def window_attention(node, args, shapes):
    sees, q, k, v, s = window_values(node, args, shapes)
    with np.errstate(all="ignore"):
        s = np.where(sees, s, -np.inf)
        top = np.where(sees.any(3), s.max(3), 0.0)
        e = np.where(sees, np.exp(s - top[..., None]), 0.0)
        total = e.sum(3)
        if node["attrs"]["part"] == "lse":
            return (np.log(total) + top).transpose(0, 2, 1).reshape(-1)
        p = e / np.where(total == 0, 1.0, total)[..., None]
    return (p @ v).transpose(0, 2, 1, 3).reshape(-1)


def window_attention_grad(node, args, shapes):
    sees, q, k, v, s = window_values(node, args, shapes)
    some = sees.any(3)[..., None]
    o, dy = (np.where(some, args[i].reshape(shapes[0]).transpose(0, 2, 1, 3), 0.0) for i in (-3, -1))
    lse = args[-2].reshape(shapes[-2]).transpose(0, 2, 1)[..., None]
    with np.errstate(all="ignore"):
        p = np.where(sees, np.exp(s - np.where(some, lse, 0.0)), 0.0)
    ds = p * (dy @ v.transpose(0, 1, 3, 2) - (dy * o).sum(3, keepdims=True)) * node["attrs"]["scale"]
    part = node["attrs"]["part"]
    if part == "dq":
        return (ds @ k).transpose(0, 2, 1, 3).reshape(-1)
    g = ds.transpose(0, 1, 3, 2) @ q if part == "dk" else p.transpose(0, 1, 3, 2) @ dy
    B, S, HK, dh = shapes[1]
    return g.reshape(B, HK, -1, S, dh).sum(2).transpose(0, 2, 1, 3).reshape(-1)


KERNELS = {"rotary": rotary, "rotaryGrad": rotary_grad, "linearCrossEntropy": linear_cross_entropy,
           "linearCrossEntropyGrad": linear_cross_entropy_grad, "orthogonalize": orthogonalize, "embedding": embedding,
           "embeddingGrad": embedding_grad, "residualNorm": residual_norm, "residualNormGrad": residual_norm_grad,
           "windowAttention": window_attention, "windowAttentionGrad": window_attention_grad}
