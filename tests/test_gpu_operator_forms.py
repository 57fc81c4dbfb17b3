"""Forms, tiles and ranges of the operators that test_gpu_operators.py's sizes do not take, on the GPU in both lowerings,
against float64 within what their roundings allow."""
import numpy as np
import pytest

from oracle import interp
import operator_checks as checks
import operator_forms
from test_gpu_operators import check

pytestmark = pytest.mark.gpu


def check_forms(tool, directory, names):
    cases = operator_forms.forms(tool, names)
    inputs = [checks.inputs_of(c["case"], c["graph"], 300 + k) for k, c in enumerate(cases)]
    for c, v, entry, b in operator_forms.run(tool, directory, cases, inputs):
        check(c, v, entry, b)


def test_coefficients_near_zero(tool, tmp_path):
    """b and c of 0, and next to it: the products' scales are as far apart as they get."""
    check_forms(tool, tmp_path, ["linear", "nearly-linear"])


def far_inputs(c, seed):
    """Rows of h and cotangents of unit size; every class a finite bias, every twelfth target no class."""
    rng = np.random.default_rng(seed)
    N, d, V = (c["case"][k] for k in ("N", "d", "V"))
    v = {n["attrs"]["name"]: rng.standard_normal(n["shape"]).astype(np.float32) for n in c["graph"]["nodes"] if n["op"] == "input"}
    v["W"] *= np.float32(1.5 / np.sqrt(d))
    v["t"] = rng.integers(0, V, N).astype(np.float32)
    v["t"][::12] = -1
    return v


def outputs(c, entry, b):
    at = {o: i for i, o in enumerate(entry["origin"])}
    return {n: b.arr(entry["gpuPerf"][str(at[k])]) for n, k in zip(c["names"], c["keep"])}


def row_allowed(args, shapes, part):
    """operator_checks.loss_allowed, a pair's floor 2^-50 of a row's own largest values: of z, that of its h and W's; of G, its
    cotangent's. Of dW, whose operands share the scale of the largest |w|·|h|: twice that (a cotangent's scale is a power of two)."""
    h, W, kept, t, z, s = checks.operators.loss_parts(args[:4], shapes[:4])
    (N, d), V, U, FLOOR = h.shape, W.shape[1], checks.U, checks.FLOOR
    rows = np.arange(N)
    mass = np.abs(h) @ np.abs(W)
    hm, wm = np.abs(h).max(1, keepdims=True), np.abs(W).max()
    e = (checks.pair_sum(d) * mass + 2 * d * FLOOR * hm * wm + 4 * U * (mass + np.abs(args[3]))).max(1)
    p = np.exp(z) / s[:, None]
    rel = 2 * e[:, None] + (8 - z) * U
    rel_s = (p * rel).sum(1) + (64 + V / 512) * U
    if part == "loss":
        return np.where(kept, 2 * e + rel_s + 4 * U * (np.abs(z[rows, t]) + np.log(s)) + 2.0 ** -21, 0)
    w = np.where(kept, args[4], 0.0)
    hot = np.zeros_like(p)
    hot[rows, t] = 1
    g = np.abs(w[:, None] * (p - hot))
    eg = np.abs(w)[:, None] * (p * (rel + rel_s[:, None] + 8 * U) + 2 * U * hot + FLOOR) + 2.0 ** -22 * g
    eg = np.where(kept[:, None], eg, 0)
    if part == "dh":
        return (eg @ np.abs(W).T + checks.pair_sum(V) * (g @ np.abs(W).T) + V * FLOOR * np.abs(w)[:, None] * wm).reshape(-1)
    if part == "db":
        return eg.sum(0) + (N + 8) * U * g.sum(0)
    return (np.abs(h).T @ eg + (checks.pair_sum(N) + 8 * U) * (np.abs(h).T @ g) + 2 * N * FLOOR * (np.abs(w) * hm[:, 0]).max()).reshape(-1)


@pytest.mark.parametrize("name", ["far-rows", "far-rows-pieces"])
def test_rows_of_a_loss_hang_on_nothing_that_other_rows_hold(tool, tmp_path, name):
    """One row of h of 1e30 times the others', and cotangents from 1e-30 to 1e20: the other rows' losses and shares of dh are bit for bit
    what they are without; rows and cotangents of all sizes at once are within their own roundings."""
    c = operator_forms.forms(tool, [name])[0]
    N, d = c["case"]["N"], c["case"]["d"]
    base = far_inputs(c, 41)
    rng = np.random.default_rng(42)
    big, small, apart, weights = (dict(base) for _ in range(4))
    big["h"] = base["h"].copy()
    big["h"][[5, 100]] *= np.float32(1e30)
    small["h"] = base["h"] * np.float32(1e-30)
    small["h"][7] = base["h"][7]
    weights["d0"] = base["d0"].copy()
    weights["d0"][[9, 101]] *= np.float32(1e20)
    apart["h"] = (base["h"] * 10.0 ** rng.choice([-12, -6, -1, 0, 0.7], (N, 1))).astype(np.float32)
    apart["d0"] = (base["d0"] * 10.0 ** rng.integers(-12, 4, N)).astype(np.float32)
    runs = dict(zip(["base", "big", "small", "weights", "apart"], operator_forms.run(tool, tmp_path, [dict(c, name=n) for n in ("base", "big", "small", "weights", "apart")],
                                                                                  [base, big, small, weights, apart])))
    got = {k: outputs(c, e, b) for k, (_, _, e, b) in runs.items()}
    for k, rows in (("big", [5, 100]), ("weights", [9, 101])):
        rest = np.setdiff1d(np.arange(N), rows)
        for n in ("loss", "dh"):
            x, y = got[k][n].reshape(N, -1)[rest], got["base"][n].reshape(N, -1)[rest]
            same = np.array_equal(x.view(np.uint32), y.view(np.uint32))
            assert same, (k, n, np.abs(x - y).max())
    assert got["small"]["loss"][7] == got["base"]["loss"][7]
    nodes = c["graph"]["nodes"]
    args = ["h", "W", "t", "b", "d0"]
    shapes = [next(n["shape"] for n in nodes if n["op"] == "input" and n["attrs"]["name"] == a) for a in args]
    for k, v in (("base", base), ("apart", apart), ("small", small), ("weights", weights)):
        want = interp.evaluate(c["graph"], {n: x.astype(np.float64) for n, x in v.items()})
        for n, at in zip(c["names"], c["keep"]):
            off, allowed = np.abs(got[k][n] - want[at]), row_allowed([v[a].astype(np.float64).reshape(-1) for a in args], shapes, n)
            worst = (off / np.maximum(allowed, 1e-300)).max()
            assert worst <= 1, (k, n, worst)
            print(f"{name} {k} {n}: {worst:.3f} of what is allowed")
