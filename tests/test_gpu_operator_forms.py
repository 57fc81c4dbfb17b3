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
        for i, n in enumerate(entry["fused"]["nodes"]):
            if n["op"].startswith("linear"):
                near_float(c["name"], n, i, entry, b)


def near_float(name, n, i, entry, b):
    """A loss's node within eight times what float32 is off, and 2^-20, in norms: a pair's roundings are four of a float's, and a product of
    pairs leaves out as much again. (The bound by elements counts a long sum's roundings as if all went one way.)"""
    args = [b.arr(entry["gpuFused"][str(j)]) for j in n["inputs"]]
    with np.errstate(all="ignore"):
        want = interp.kernel(n, [a.astype(np.float64) for a in args], entry["fused"])
        single = interp.kernel(n, args, entry["fused"])
    x = b.arr(entry["gpuFused"][str(i)]).astype(np.float64)
    finite = np.isfinite(want)
    assert single.dtype == np.float32 and np.array_equal(finite, np.isfinite(x))
    off, by_float, size = (np.linalg.norm(v[finite]) for v in (x - want, single - want, want))
    print(f"{name} {n['op']} {n['attrs'].get('part', '')}: off by {off / size:.1e}, float32 by {by_float / size:.1e}")
    assert off <= 8 * by_float + 2.0 ** -20 * size, (name, n["attrs"], off / size, by_float / size)


def test_coefficients_near_zero(tool, tmp_path):
    """b and c of 0, and next to it: the products' scales are as far apart as they get."""
    check_forms(tool, tmp_path, ["linear", "nearly-linear"])


@pytest.mark.parametrize("names", [
    ["tall-logits", "tall-logits-pieces", "tall-values"], ["large-split"], ["large-whole"], ["large-pieces"],
    ["half", "half-tall"], ["square-tall-tiles", "square-tall-tiles-tall"], ["square-wide-tiles", "square-wide-tiles-tall"],
    ["square-tiles", "square-tiles-tall"], ["square-split"], ["stack-twins", "stack-twins-odd", "eight"]], ids=lambda n: n[0])
def test_large_tiles_and_split_sums(tool, tmp_path, names):
    """The loss by 256 x 128 and 128 x 256 tiles, in pieces and with K split; orthogonalize by its upper tiles, by 128 x 128 ones and X by each larger
    one, with leftover tiles split; equal stacks side by side. test_operator_forms.py has the kernels that each of them takes."""
    check_forms(tool, tmp_path, names)


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


def row_allowed(args, shapes, part, ew=0.0):
    """operator_checks.loss_allowed, a pair's floor 2^-50 of a row's own largest values: of z, that of its h and W's; of G, its
    cotangent's. Of dW, whose operands share the scale of the largest |w|·|h|: twice that (a cotangent's scale is a power of two). ew: how far the cotangents are off already."""
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
    eg = np.where(kept[:, None], eg + 1.001 * np.reshape(ew, (-1, 1)) * np.abs(p - hot), 0)
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


def test_losses_that_decide_their_own_cotangents_end_to_end(tool, tmp_path):
    """The squared losses and their gradients against float64 of the inputs: the losses' errors go into the cotangents 2·loss·d0."""
    c = operator_forms.forms(tool, ["tall-after"])[0]
    v = far_inputs(c, 43)
    _, _, entry, b = operator_forms.run(tool, tmp_path, [c], [v])[0]
    got = outputs(c, entry, b)
    want = interp.evaluate(c["graph"], {n: x.astype(np.float64) for n, x in v.items()})
    wants = {n: want[k] for n, k in zip(c["names"], c["keep"])}
    nodes, args = c["graph"]["nodes"], ["h", "W", "t", "b", "d0"]
    shapes = [next(n["shape"] for n in nodes if n["op"] == "input" and n["attrs"]["name"] == a) for a in args]
    values = [v[a].astype(np.float64).reshape(-1) for a in args]
    e = row_allowed(values, shapes, "loss")
    loss, d0 = np.sqrt(wants["loss"]), values[4]
    values[4] = 2 * loss * d0
    ew = np.abs(d0) * (2 * e + 4 * checks.U * loss)
    for n in c["names"]:
        allowed = 2 * loss * e + e * e + 2 * checks.U * wants[n] if n == "loss" else row_allowed(values, shapes, n, ew)
        worst = (np.abs(got[n] - wants[n]) / np.maximum(allowed, 1e-300)).max()
        assert worst <= 1, (n, worst)
        print(f"tall-after {n}: {worst:.3f} of what is allowed")


def test_an_update_orthogonalised_twice_end_to_end(tool, tmp_path):
    """Against float64 of the inputs: the first result's error, at most twice as large against its norm after the division by it, grows by at most
    the polynomial's largest slope a step."""
    c = operator_forms.forms(tool, ["twice"])[0]
    v = checks.inputs_of(c["case"], c["graph"], 44)
    _, _, entry, b = operator_forms.run(tool, tmp_path, [c], [v])[0]
    got = outputs(c, entry, b)
    want = interp.evaluate(c["graph"], {n: x.astype(np.float64) for n, x in v.items()})
    for name, at in zip(c["names"], c["keep"]):
        node = c["graph"]["nodes"][at]
        first = node["inputs"][0]
        x = c["graph"]["nodes"][first]["inputs"][0]
        shape = [node["shape"]]
        e = checks.orthogonalize_allowed(c["graph"]["nodes"][first], [want[x]], shape)[0]
        p, top, slope = node["attrs"]["coefficients"], 1.0, 1.0
        for _ in range(node["attrs"]["steps"]):
            s = np.linspace(0, top, 4001)
            slope *= np.abs(p[0] + 3 * p[1] * s ** 2 + 5 * p[2] * s ** 4).max() * 1.01
            top = np.abs(s * (p[0] + s ** 2 * (p[1] + s ** 2 * p[2]))).max()
        allowed = slope * 2.01 * e / np.linalg.norm(want[first]) + checks.orthogonalize_allowed(node, [want[first]], shape)[0]
        off = np.linalg.norm(got[name] - want[at])
        assert off <= allowed, (name, off, allowed)
        print(f"{name} twice: {off / allowed:.3f} of what is allowed, which is {allowed / np.linalg.norm(want[at]):.1e} of the result")
