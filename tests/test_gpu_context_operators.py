"""embedding, residualNorm and windowAttention and their gradients on the GPU, in both lowerings, against float64
(oracle/operators.py) within what their roundings allow (context_checks.py): sizes from one element on, tokens that are no row, rows
of one value, windows and sinks that end inside a tile, sequences of no key, queries outside their sequence, shared heads, gradients of some
operands only. Padding past every buffer stays as it was, and the perf lowering, which runs a node's parts as one launch,
gives the plain lowering's bits."""
import numpy as np
import pytest

from oracle import interp
import context_checks as checks

pytestmark = pytest.mark.gpu


def run(tool, directory, cases, inputs):
    import tcmi_bridge
    import operator_forms
    reqs = [{"name": c["name"], "graph": c["graph"], "keep": c["keep"], "perf": True, "inputs": {n: operator_forms.text(x) for n, x in v.items()}}
            for c, v in zip(cases, inputs)]
    print("gpu step: gpu-graphs " + ", ".join(c["name"] for c in cases), flush=True)
    tool("gpu-graphs", {"graphs": reqs}, out=str(directory), timeout=300)
    b = tcmi_bridge.Bundle(directory)
    got = {c["name"]: c for c in b.cases}
    return [(c, got[c["name"]], b) for c in cases]


def check(c, entry, b):
    assert all(entry["canaryFused"]) and entry["canaryPerf"], c["name"]
    graph = entry["fused"]
    with np.errstate(all="ignore"):
        for i, n in enumerate(graph["nodes"]):
            if n["op"] not in checks.ALLOWED:
                continue
            # Node by node: its operands as the GPU had them.
            x = b.arr(entry["gpuFused"][str(i)]).astype(np.float64)
            args = [b.arr(entry["gpuFused"][str(j)]).astype(np.float64) for j in n["inputs"]]
            shapes = [graph["nodes"][j]["shape"] for j in n["inputs"]]
            want = interp.kernel(n, args, graph)
            off, allowed = np.where((x == want) | (np.isnan(x) & np.isnan(want)), 0, np.abs(x - want)), checks.ALLOWED[n["op"]](n, args, shapes)
            bad = ~(off <= allowed)
            assert not bad.any(), (c["name"], n["op"], n["attrs"].get("part"), bad.sum(), np.flatnonzero(bad)[:5], x[bad][:5], want[bad][:5], off[bad][:5], allowed[bad][:5])
            print(f"{c['name']} {n['op']} {n['attrs'].get('part', '')}: {np.max(off / np.maximum(allowed, 1e-300), initial=0):.3f} of what is allowed")
    for k, h in entry["gpuPerf"].items():
        perf, plain = b.arr(h), b.arr(entry["gpuFused"][k])
        same = np.array_equal(perf.view(np.uint32), plain.view(np.uint32))
        assert same, (c["name"], graph["nodes"][int(k)]["op"], np.flatnonzero(perf.view(np.uint32) != plain.view(np.uint32))[:5])


@pytest.mark.parametrize("family", ["embedding", "residual", "window"])
def test_operators_match_float64(family, tmp_path, tool):
    cases = tool("operator-graphs", {"context": True, "family": family})
    inputs = [checks.inputs_of(c["case"], c["graph"], 100 + k) for k, c in enumerate(cases)]
    for c, entry, b in run(tool, tmp_path, cases, inputs):
        check(c, entry, b)
