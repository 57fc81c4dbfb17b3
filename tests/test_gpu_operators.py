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
