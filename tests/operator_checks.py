"""Inputs of the operators' test graphs, and how far a float32 evaluation of each may be from its float64 value, element
by element, by arithmetic on the kernels' roundings (u: half a float32 step, 2^-24, relative).

Products are of pairs of halves: an operand is off by 2^-23 of itself (its remainder's rounding), the term left out is at
most 2^-22 of a product, so a product is off by 2^-21 of its magnitude at most; a sum of K of them rounds K times (and a
few more, where partial sums are joined). A pair's floor, 2^-36 where its operand's largest value is 2^14 or more, adds
2^-50 of that largest value an element.
"""
import numpy as np

from oracle import operators

U = 2.0 ** -24
FLOOR = 2.0 ** -50


def pair_sum(K):
    return 2.0 ** -21 + (K + 16) * U


def plain(x):
    """Values for a JSON request: what JSON has no number for as text (Float32Array.from reads both)."""
    return [float(v) if np.isfinite(v) else ("NaN" if np.isnan(v) else "Infinity" if v > 0 else "-Infinity") for v in np.asarray(x).reshape(-1)]


def inputs_of(case, graph, seed):
    """float32 inputs by name, with what the operators meet in earnest: rows of zeros, far positions, targets that are no class over
    rows that hold no numbers, classes masked by a bias of -inf."""
    rng = np.random.default_rng(seed)
    shapes = {n["attrs"]["name"]: n["shape"] for n in graph["nodes"] if n["op"] == "input"}
    v = {k: rng.standard_normal(s).astype(np.float32) for k, s in shapes.items()}
    if case["family"] == "rotary":
        for k in v:
            if k.startswith("x"):
                v[k].reshape(-1, v[k].shape[-1])[0] = 0          # a row of zeros
                v[k] *= 3
            if k.startswith("g"):
                v[k] = (1 + 0.1 * v[k]).astype(np.float32)
        T = shapes["at"]
        v["at"] = (rng.integers(0, 1 << 20, size=T) + (rng.random(T) < 0.2) * 0.5).astype(np.float32)
    if case["family"] == "loss":
        N, V = case["N"], case["V"]
        t = rng.integers(0, V, size=N).astype(np.float32)
        v["W"] *= np.float32(1.5 / np.sqrt(case["d"]))
        left = rng.random(N) < 0.2
        if N >= 5:
            left[:5] = [False, True, True, True, True]
            t[left] = rng.choice([-1.0, V, 0.5, np.nan, 1e30, -0.5], size=left.sum())
            v["h"][left] = rng.choice([np.nan, np.inf, 1e38, 0], size=left.sum())[:, None]
        v["t"] = t
        if case.get("bias") and V >= 100:
            v["b"][rng.permutation(np.setdiff1d(np.arange(V), t[np.isfinite(t)].clip(0, V - 1)))[: V // 10]] = -np.inf
        if "d0" in v:
            v["d0"] = (v["d0"] / N).astype(np.float32)
            if N >= 5:
                v["d0"][1:5] = [np.nan, np.inf, 1e30, 0]
    return v


def rotary_allowed(node, args, shapes):
    """Forward and gradients: n (or dn) off by its factors' roundings, the sum over the head's among them (half of it in the
    root), sine and cosine off by 4u, the rotation's two products and their sum."""
    attrs, dh = node["attrs"], shapes[0][-1]
    x = args[0].reshape(shapes[0])
    gain = args[2] if len(args) == (3 if node["op"] == "rotary" else 4) else None
    a, b = operators.pair_dims(attrs, dh)

    def paired(v):
        out = np.abs(v)
        out[..., a], out[..., b] = np.abs(v[..., a]) + np.abs(v[..., b]), np.abs(v[..., a]) + np.abs(v[..., b])
        return out

    eps = attrs.get("eps", 0.0)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps) if gain is not None else np.ones(x.shape[:-1] + (1,))
    if node["op"] == "rotary":
        return (dh / 2 + 16) * U * paired(x * r * (gain if gain is not None else 1)).reshape(-1)
    dn, h = paired(args[-1].reshape(shapes[0])), np.abs(x * r)
    if gain is None:
        return 16 * U * dn.reshape(-1)
    if attrs["part"] == "dgain":
        # A lane adds up at most 8 rows here, then 256 lanes of a workgroup, 64 workgroups' sums and 16 of those are added in turn.
        adds = min(x.size // dh, 8 + 256 + 64 + 16)
        return (adds + dh + 32) * U * (dn * h).reshape(-1, dh).sum(0)
    g = dn * np.abs(gain)
    return ((2 * dh + 40) * U * r * (g + h * (g * h).mean(-1, keepdims=True))).reshape(-1)


def loss_allowed(node, args, shapes, pieces=1):
    grad = node["op"].endswith("Grad")
    head = len(args) - (1 if grad else 0)
    h, W, kept, t, z, s = operators.loss_parts(args[:head], shapes[:head])
    (N, d), V = h.shape, W.shape[1]
    mass = np.abs(h) @ np.abs(W)
    bias = np.where(np.isfinite(args[3]), np.abs(args[3]), 0) if head == 4 else np.zeros(V)
    ez = pair_sum(d) * mass + 2 * d * FLOOR * np.abs(h).max() * np.abs(W).max() + 4 * U * (mass + bias)
    e = ez.max(1)                                     # of the row's maximum, and of every logit
    adds = 64 + V / 512                               # the deepest chain of additions to a sum of exponentials
    depth = np.where(np.isfinite(z), -z, 0)           # distance from the maximum
    rel = 2 * e[:, None] + (8 + depth) * U            # of an exponential
    p = np.exp(z) / s[:, None]
    rel_s = (p * rel).sum(1) + adds * U
    if not grad:
        zt = -z[np.arange(N), t]
        return np.where(kept, 2 * e + rel_s + 4 * U * (np.abs(zt) + np.log(s)) + 2.0 ** -21, 0.0)
    w = np.where(kept, args[-1], 0.0)
    hot = np.zeros_like(p)
    hot[np.arange(N), t] = 1
    g = np.abs(w[:, None] * (p - hot))
    eg = np.abs(w)[:, None] * (p * (rel + rel_s[:, None] + 8 * U) + 2 * U * hot) + 2.0 ** -22 * g + FLOOR * np.abs(w).max()
    eg = np.where(kept[:, None], eg, 0)
    part = node["attrs"]["part"]
    if part == "dbias":
        return eg.sum(0) + (N + pieces) * U * g.sum(0)
    top = np.abs(w).max() * FLOOR
    if part == "dh":
        return np.where(kept[:, None], eg @ np.abs(W).T + pair_sum(V) * (g @ np.abs(W).T) + V * top * np.abs(W).max(), 0).reshape(-1)
    return (np.abs(h).T @ eg + (pair_sum(N) + pieces * U) * (np.abs(h).T @ g) + N * top * np.abs(h).max()).reshape(-1)


def orthogonalize_allowed(node, args, shapes):
    """Frobenius-norm bound of one matrix's error, times how much each later step can enlarge it: a step is an odd
    polynomial p of the singular values, whose change in the Frobenius norm is at most the largest |p'| over their interval times its
    argument's. A step's own roundings, in norms (|XY| <= |X|·|Y| for the absolute products too): pair_sum(K) a product and 2^-21 a pair kept."""
    a, b, c = node["attrs"]["coefficients"]
    steps = node["attrs"]["steps"]
    x = args[0].reshape([-1] + list(shapes[0][-2:]))
    allowed = []
    for m in x:
        if m.shape[0] > m.shape[1]:
            m = m.T
        s, l = m.shape
        norm = np.linalg.norm(m) + node["attrs"]["eps"]
        m = m / norm
        err = 4 * U * np.linalg.norm(m) + 2.0 ** -22 * np.linalg.norm(m) + s * l * FLOOR
        for _ in range(steps):
            top = np.linalg.norm(m, 2)
            grid = np.linspace(0, top, 2001)
            slope = np.abs(a + 3 * b * grid ** 2 + 5 * c * grid ** 4).max() * 1.01
            A = m @ m.T
            fro, fa, am = np.linalg.norm(m), np.linalg.norm(A), np.linalg.norm(np.abs(m))
            eA = pair_sum(l) * np.linalg.norm(np.abs(m) @ np.abs(m).T) + 2.0 ** -21 * fa
            B = b * A + c * A @ A
            absA = np.abs(A)
            eB = (abs(b) + 2 * abs(c) * np.linalg.norm(A, 2)) * eA + abs(c) * pair_sum(s) * np.linalg.norm(absA @ absA) \
                + (2.0 ** -21 + 8 * U) * np.linalg.norm(abs(b) * absA + abs(c) * absA @ absA)
            own = eB * top + pair_sum(s) * np.linalg.norm(np.abs(B) @ np.abs(m)) + (2.0 ** -21 + 8 * U) * (abs(a) * fro + np.linalg.norm(np.abs(B) @ np.abs(m))) + s * l * FLOOR
            err = slope * err + own
            m = a * m + B @ m
            del am
        allowed.append(err)
    return np.array(allowed)
