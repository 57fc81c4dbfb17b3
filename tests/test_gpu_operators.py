"""The operators that are one node each (rotary, linearCrossEntropy, orthogonalize and their gradients) on the GPU, in
both lowerings, against float64 (oracle/operators.py) within what their roundings allow (operator_checks.py): sizes from
one element on, none of them whole tiles, tokens before and after heads, several position axes, rows that the
loss leaves out, masked classes, several pieces, gradients of some operands only, stacked matrices and matrices side by side.
Padding past every buffer stays as it was, and the perf lowering, which runs an operator's parts as one launch, gives the
plain lowering's bits."""
import numpy as np
import pytest

from oracle import interp
import operator_checks as checks

pytestmark = pytest.mark.gpu

OPERATORS = {"rotary", "rotaryGrad", "linearCrossEntropy", "linearCrossEntropyGrad", "orthogonalize"}
ALLOWED = {"rotary": checks.rotary_allowed, "rotaryGrad": checks.rotary_allowed, "linearCrossEntropy": checks.loss_allowed,
           "linearCrossEntropyGrad": checks.loss_allowed}


def run(tool, directory, family):
    import tcmi_bridge
    cases = tool("operator-graphs", {"family": family})
    reqs, inputs = [], {}
    for k, c in enumerate(cases):
        inputs[c["name"]] = checks.inputs_of(c["case"], c["graph"], 100 + k)
        reqs.append({"name": c["name"], "graph": c["graph"], "keep": c["keep"], "perf": True, "tuning": c["case"].get("tuning"),
                     "inputs": {n: checks.plain(x) for n, x in inputs[c["name"]].items()}})
    print(f"gpu step: gpu-graphs, {len(reqs)} {family} graphs", flush=True)
    tool("gpu-graphs", {"graphs": reqs}, out=str(directory), timeout=300)
    b = tcmi_bridge.Bundle(directory)
    got = {c["name"]: c for c in b.cases}
    return [(c, inputs[c["name"]], got[c["name"]], b) for c in cases]


def check(c, inputs, entry, b):
    assert all(entry["canaryFused"]) and entry["canaryPerf"], c["name"]
    graph = entry["fused"]
    used = {k: v.astype(np.float64) for k, v in inputs.items()}
    with np.errstate(all="ignore"):
        values = interp.evaluate(graph, used)
        for i, n in enumerate(graph["nodes"]):
            if n["op"] not in OPERATORS:
                continue
            x = b.arr(entry["gpuFused"][str(i)]).astype(np.float64)
            # Node by node: its operands as the GPU had them.
            args = [b.arr(entry["gpuFused"][str(j)]).astype(np.float64) for j in n["inputs"]]
            shapes = [graph["nodes"][j]["shape"] for j in n["inputs"]]
            want = interp.kernel(n, args, graph)
            if n["op"] == "orthogonalize":
                size = shapes[0][-1] * shapes[0][-2]
                off = np.linalg.norm((x - want).reshape(-1, size), axis=1)
                # The bound by norms, and eight times what the same steps are off in float32: a pair's roundings are four of a
                # float's, and a product of pairs leaves out as much again.
                single = interp.kernel(n, [args[0].astype(np.float32)], graph).astype(np.float64)
                by_float = np.linalg.norm((single - want).reshape(-1, size), axis=1)
                allowed = np.minimum(checks.orthogonalize_allowed(n, args, shapes), 8 * by_float + 2.0 ** -20 * np.linalg.norm(want.reshape(-1, size), axis=1))
            else:
                off, allowed = np.abs(x - want), ALLOWED[n["op"]](n, args, shapes)
                both = (x == want) | (np.isnan(x) & np.isnan(want))
                off = np.where(both, 0, off)
            bad = ~(off <= allowed)
            assert not bad.any(), (c["name"], n["op"], n["attrs"].get("part"), np.flatnonzero(bad)[:5], off[bad][:5], allowed[bad][:5])
            worst = np.max(off / np.maximum(allowed, 1e-300)) if off.size else 0
            print(f"{c['name']} {n['op']} {n['attrs'].get('part', '')}: {worst:.3f} of what is allowed")
    for k, h in entry["gpuPerf"].items():
        perf, plain = b.arr(h), b.arr(entry["gpuFused"][k])
        same = np.array_equal(perf.view(np.uint32), plain.view(np.uint32))
        assert same, (c["name"], graph["nodes"][int(k)]["op"], np.flatnonzero(perf.view(np.uint32) != plain.view(np.uint32))[:5])
    del values


@pytest.mark.parametrize("family", ["rotary", "loss", "orthogonalize"])
def test_operators_match_float64(family, tmp_path, tool):
    for c, inputs, entry, b in run(tool, tmp_path, family):
        check(c, inputs, entry, b)


# Few rows, few classes, and many of both.
SHAPES = [(9, 16, 200), (70, 16, 40), (100, 16, 300)]


@pytest.mark.parametrize("N, d, V", SHAPES)
def test_targets_that_are_masked_and_rows_without_numbers(tool, tmp_path, N, d, V):
    """A target whose class has a bias of -inf: an infinite loss, and gradients as the formula's. A row whose h is infinite or NaN: its own loss
    and share of dh are no numbers, the other rows' are what they were. Products of at most 300 terms of magnitudes below 8, each off by
    2^-21 + 300 / 2^24 at most: 1e-4 in all."""
    import tcmi_bridge
    case = {"name": "masked", "family": "loss", "N": N, "d": d, "V": V, "bias": True, "gradient": True}
    c = tool("operator-graphs", {"cases": [case]})[0]
    rng = np.random.default_rng(5)
    v = {n["attrs"]["name"]: rng.standard_normal(n["shape"]).astype(np.float32) for n in c["graph"]["nodes"] if n["op"] == "input"}
    v["W"] *= np.float32(0.3)
    v["t"] = rng.integers(0, V, N).astype(np.float32)
    v["t"][3] = 7
    v["t"][v["t"] == 11] = 12
    v["b"][[7, 11]] = -np.inf
    v["t"][4:] = np.where(v["t"][4:] == 7, 8, v["t"][4:])
    bad = dict(v, h=v["h"].copy())
    bad["h"][5, 2], bad["h"][6] = np.inf, np.nan
    print(f"gpu step: gpu-graphs, masked targets {N} x {d} x {V}", flush=True)
    reqs = [{"name": name, "graph": c["graph"], "keep": c["keep"], "perf": True, "inputs": {k: checks.plain(x) for k, x in x.items()}}
            for name, x in (("masked", v), ("bad", bad))]
    tool("gpu-graphs", {"graphs": reqs}, out=str(tmp_path), timeout=300)
    b = tcmi_bridge.Bundle(tmp_path)
    with np.errstate(all="ignore"):
        want = interp.evaluate(c["graph"], {k: x.astype(np.float64) for k, x in v.items()})
    got = {}
    for e in b.cases:
        at = {o: i for i, o in enumerate(e["origin"])}
        got[e["name"]] = {n: b.arr(e["gpuPerf"][str(at[k])]).astype(np.float64) for n, k in zip(c["names"], c["keep"])}
    for n, k in zip(c["names"], c["keep"]):
        np.testing.assert_allclose(got["masked"][n], want[k], rtol=1e-4, atol=1e-4, err_msg=n)
    assert np.isinf(want[c["keep"][0]][3]) and np.isfinite(got["masked"]["dW"]).all()
    rest = np.setdiff1d(np.arange(N), [5, 6])
    assert not np.isfinite(got["bad"]["loss"][[5, 6]]).any()
    # Up to the scale of h's pairs, which those rows' values no longer decide.
    np.testing.assert_allclose(got["bad"]["loss"][rest], got["masked"]["loss"][rest], rtol=1e-5, atol=1e-5)
    np.testing.assert_allclose(got["bad"]["dh"].reshape(N, d)[rest], got["masked"]["dh"].reshape(N, d)[rest], rtol=1e-5, atol=1e-5)
    assert not np.isfinite(got["bad"]["dh"].reshape(N, d)[[5, 6]]).any()
