"""Inputs of the test graphs of embedding, residualNorm and windowAttention, and how far a float32 evaluation of each may be
from its float64 value, element by element.

Errors are carried through each formula beside its values (`Off`): a float32 operation rounds by at most U = 2^-24 of its
result (hardware reciprocal roots and exponentials: one step, 2U), a sum of terms added at most `deep` deep rounds by deep·U of
their magnitudes. The attention's products may be of pairs of halves, as operator_checks.py says: pair_sum(K) of a
product's magnitude, and a floor of 2^-50 of its operands' largest values a term.
"""
import numpy as np

from oracle import operators
from operator_checks import FLOOR, U, pair_sum

ROW_FLOOR = 2.0 ** -39


def inputs_of(case, graph, seed):
    """float32 inputs by name, with what the operators meet in earnest: tokens that are no row over rows that hold no numbers, rows of
    zeros, of one value and far from zero, keys that no query sees, sequences of no key, queries that stand outside their sequence."""
    rng = np.random.default_rng(seed)
    shapes = {n["attrs"]["name"]: n["shape"] for n in graph["nodes"] if n["op"] == "input"}
    v = {k: rng.standard_normal(s).astype(np.float32) for k, s in shapes.items()}
    if case["family"] == "embedding":
        V, N = case["V"], int(np.prod(case["tokens"]))
        t = np.floor(V ** rng.random(N)).clip(1, V) - 1            # few tokens often, and the last row
        t[: N // 3] = rng.integers(0, V, N // 3)
        if N > 2:
            t[-1] = V - 1
        if case.get("one") is not None:
            t[rng.random(N) < 0.9] = case["one"]
        left = rng.random(N) < 0.1
        t[left] = rng.choice([-1.0, V, 0.5, np.nan, 1e30, -np.inf], size=left.sum())
        v["tokens"] = t.astype(np.float32).reshape(shapes["tokens"])
        if "d0" in v:
            v["d0"].reshape(N, -1)[left] = rng.choice([np.nan, np.inf, 1e38], size=left.sum())[:, None]
    if case["family"] == "residual":
        for k in shapes:
            if k not in ("x", "y", "d0", "d1"):
                v[k] = (0.3 * v[k] + (1 if k.endswith("ain") else 0)).astype(np.float32)
        x, y = (v[k].reshape(-1, case["x"][-1]) for k in "xy")
        y += np.float32(0.5)
        if len(x) > 4:
            x[0] = y[0] = 0
            y[1] = 3
            x[2] *= np.float32(1e4)
            y[2] *= np.float32(1e-4)
            x[3] += 100
    if case["family"] == "window":
        B, T = case["q"][:2]
        S = case["k"][1]
        v["q"] *= np.float32(1.5)
        if case.get("lengths"):
            lengths = rng.integers(1, S + 1, B).astype(np.float32)
            some = [S, 0, 1 + (S > 1), S + 3.5, np.nan, -2, S / 2 + 0.25]
            lengths[: len(some)] = some[: B]
            v["lengths"] = lengths
        node = next(n for n in graph["nodes"] if n["op"] == "windowAttention")
        sees = operators.window_sees(node, [None, None, None, v.get("lengths")], [graph["nodes"][i]["shape"] for i in node["inputs"]])
        unseen, blind = ~sees.any(1), ~sees.any(2)
        for k in "kv":
            v[k][unseen] = rng.choice([np.nan, np.inf, 1e38], size=unseen.sum())[:, None, None]
        v["q"][blind] = np.nan
        if "d0" in v:
            v["d0"][blind] = np.nan
    return v


class Off:
    """Values and how far their float32 evaluation may be from them."""

    def __init__(self, v, e=0.0):
        self.v, self.e = np.asarray(v, dtype=np.float64), np.broadcast_to(np.asarray(e, dtype=np.float64), np.shape(v))

    def rounded(self, steps=1.0):
        return Off(self.v, self.e + steps * U * (np.abs(self.v) + self.e))

    def __add__(self, o):
        o = o if isinstance(o, Off) else Off(o)
        return Off(self.v + o.v, self.e + o.e).rounded()

    def __sub__(self, o):
        return self + Off(-o.v, o.e)

    def __mul__(self, o):
        o = o if isinstance(o, Off) else Off(o)
        return Off(self.v * o.v, self.e * np.abs(o.v) + o.e * np.abs(self.v) + self.e * o.e).rounded()

    def sum(self, axis, deep):
        v, e = self.v.sum(axis, keepdims=True), self.e.sum(axis, keepdims=True)
        return Off(v, e + deep * U * (np.abs(self.v) + self.e).sum(axis, keepdims=True))


ROW = 16 + 6 + 16          # additions that a term of a row's sum goes through: a lane's, its wavefront's, the wavefronts'


def embedding_allowed(node, args, shapes):
    # The scale itself is rounded, then the product.
    if node["op"] == "embedding":
        return 2.01 * U * np.abs(operators.embedding(node, args, shapes))
    t, dy = args
    n = max(1, len(t))
    kept = (t >= 0) & (t < node["attrs"]["rows"]) & (t == np.floor(t))
    most = np.bincount(t[kept].astype(int), minlength=1).max() if kept.any() else 1
    mass = operators.embedding_grad(dict(node, attrs=dict(node["attrs"], scale=abs(node["attrs"]["scale"]))), [t, np.abs(dy)], shapes)
    return (min(n, most) + 3) * U * mass


def residual_off(node, args, shapes):
    a, v = node["attrs"], operators.residual_operands(node, args, shapes)
    d = shapes[0][-1]

    def mean(x):
        return x.sum(1, ROW) * (1.0 / d)

    def normalised(x):
        if a["norm"] == "layer":
            m = mean(x)
            x = x - Off(np.broadcast_to(m.v, x.v.shape), np.broadcast_to(m.e, x.v.shape))
        s = mean(x * x)
        s = Off(s.v + a["eps"], s.e).rounded(2)
        r = 1 / np.sqrt(s.v)
        # (Squares add up to no less than 0 in float32 too: a root is of eps at least, of eps rounded.)
        low = 1 / np.sqrt(np.maximum(s.v - s.e, max(a["eps"] * (1 - 4 * U), 1e-300)))
        r = Off(r, low - r).rounded(3)
        return r, x * r

    def back(r, hat, g):
        m = mean(g * hat)
        out = g - hat * m
        return r * (out - mean(g)) if a["norm"] == "layer" else r * out

    y = Off(v["y"])
    ry, p = None, y
    if a["post"]:
        ry, hat = normalised(y)
        p = hat * v["postGain"]
        if "postBias" in v:
            p = p + v["postBias"]
    rho = Off(a["residual"], U * abs(a["residual"]))
    h = rho * v["x"] + (p * v["gate"] if a["gate"] else p)
    if node["op"] == "residualNorm":
        if a["part"] == "h":
            return h
        n = normalised(h)[1] * v["gain"]
        return n + v["bias"] if "bias" in v else n
    part = a["part"]
    # A column's sum: a workgroup's rows (their count over its share of them, 512 workgroups), its 16 lane groups, then the partial sums: a 32nd of
    # them a thread, eights and fours of threads.
    N = len(v["x"])
    deep = N / 512 + 16 + min(512, N) / 32 + 8 + 4
    dh = Off(v["dh"]) if "dh" in v else None
    if "dn" in v:
        r, hat = normalised(h)
        if part in ("dgain", "dbias"):
            return (Off(v["dn"]) * hat if part == "dgain" else Off(v["dn"])).sum(0, deep)
        through = back(r, hat, Off(v["dn"]) * v["gain"])
        dh = through if dh is None else dh + through
    if part == "dx":
        return rho * dh
    if part == "dgate":
        full = len(shapes[list(v).index("gate")]) == len(shapes[0]) and v["gate"].shape == v["x"].shape
        return dh * p if full else (dh * p).sum(0, deep)
    dp = dh * v["gate"] if a["gate"] else dh
    if not a["post"]:
        return dp
    ry, hat = normalised(y)
    return {"dpostGain": lambda: (dp * hat).sum(0, deep), "dpostBias": lambda: dp.sum(0, deep), "dy": lambda: back(ry, hat, dp * v["postGain"])}[part]()


def residual_allowed(node, args, shapes):
    off = residual_off(node, args, shapes)
    np.testing.assert_allclose(off.v.reshape(-1), operators.KERNELS[node["op"]](node, args, shapes), rtol=1e-9, atol=1e-9)
    return off.e.reshape(-1)


def window_allowed(node, args, shapes):
    sees, q, k, v, s = operators.window_values(node, args, shapes)
    scale, dh, S = abs(node["attrs"]["scale"]), shapes[0][3], shapes[1][1]
    T, R = shapes[0][1], shapes[0][2] // shapes[1][2]
    mt = lambda x: np.abs(x).transpose(0, 1, 3, 2)
    top = lambda x: np.abs(x).max(initial=0.0)
    rows = lambda x, y: 2 * dh * ROW_FLOOR * np.abs(x).max(3, keepdims=True) * np.abs(y).max(3)[:, :, None]
    seen = np.where(sees, np.abs(s), 0.0)
    es = scale * (pair_sum(dh) * (np.abs(q) @ mt(k)) + rows(q, k)) + 6 * U * seen
    some = sees.any(3)[..., None]
    with np.errstate(all="ignore"):
        if node["op"] == "windowAttention":
            m = np.where(some, np.where(sees, s, -np.inf).max(3, keepdims=True), 0.0)
            # The running maximum may be any earlier one's: exponents up to the scores' spread, rounded twice.
            spread = np.where(some, m - np.where(sees, s, np.inf).min(3, keepdims=True), 0.0)
            rel = es + 4 * U * (np.where(sees, m - s, 0.0) + spread) + (S / 16 + 32) * U
            e = np.where(sees, np.exp(s - m), 0.0)
            p = e / np.where(some, e.sum(3, keepdims=True), 1.0)
            mean = (p * rel).sum(3, keepdims=True)
            if node["attrs"]["part"] == "lse":
                lse = np.where(some, m + np.log(np.where(some, e.sum(3, keepdims=True), 1.0)), 0.0)
                return (mean + 4 * U * (np.abs(lse) + np.abs(m)) + 4 * U)[..., 0].transpose(0, 2, 1).reshape(-1)
            off = (p * (rel + mean)) @ np.abs(v) + (pair_sum(S) + 8 * U) * (p @ np.abs(v)) + S * FLOOR * top(v)
            return off.transpose(0, 2, 1, 3).reshape(-1)
        o, dy = (np.where(some, args[i].reshape(shapes[0]).transpose(0, 2, 1, 3), 0.0) for i in (-3, -1))
        lse = np.where(some, args[-2].reshape(shapes[-2]).transpose(0, 2, 1)[..., None], 0.0)
        p = np.where(sees, np.exp(s - lse), 0.0)
        rel = es + 4 * U * (seen + np.abs(lse)) + 4 * U
        part = node["attrs"]["part"]
        if part == "dv":
            mass, off = p, p * rel
            a, K = dy, T * R
        else:
            dp, D = dy @ v.transpose(0, 1, 3, 2), (dy * o).sum(3, keepdims=True)
            edp = pair_sum(dh) * (np.abs(dy) @ mt(v)) + rows(dy, v) + (dh + 16) * U * (np.abs(dy) * np.abs(o)).sum(3, keepdims=True)
            mass = p * np.abs(dp - D)
            off = mass * (rel + 4 * U) + p * (edp + 2 * U * (np.abs(dp) + np.abs(D)))
            a, K = (k, S) if part == "dq" else (q, T * R)
        factor = 1.0 if part == "dv" else scale
        if part == "dq":
            g = factor * (off @ np.abs(a) + (pair_sum(K) + 8 * U) * (mass @ np.abs(a)) + K * FLOOR * top(mass) * top(a))
            return g.transpose(0, 2, 1, 3).reshape(-1)
        g = factor * (off.transpose(0, 1, 3, 2) @ np.abs(a) + (pair_sum(K) + 8 * U) * (mass.transpose(0, 1, 3, 2) @ np.abs(a)) + K * FLOOR * top(mass) * top(a))
    B, _, HK, _ = shapes[1]
    return g.reshape(B, HK, -1, S, dh).sum(2).transpose(0, 2, 1, 3).reshape(-1)


ALLOWED = {"embedding": embedding_allowed, "embeddingGrad": embedding_allowed, "residualNorm": residual_allowed, "residualNormGrad": residual_allowed,
           "windowAttention": window_allowed, "windowAttentionGrad": window_allowed}
