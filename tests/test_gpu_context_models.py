"""Training steps that run the operators for long contexts and large vocabularies together, on the GPU: token indices, sliding-window
attention with shared key heads, norms joined to the residual sums, rotary positions, class targets. The trainer (perf lowering, a node's parts
as one launch; captured and replayed; in the arena; over two streams) gives the checked path's bits over several steps, each
operator's nodes are within what their roundings allow of float64 on the GPU's own operands, and the first loss is float64's."""
import numpy as np
import pytest

from oracle import interp
from test_gpu_context_operators import check
from test_gpu_operators import check as check_operators

pytestmark = pytest.mark.gpu

FULL = {"tokens": "indices", "targets": "classes", "positions": "rotary", "qkNorm": True, "attention": "window", "window": 9, "sinks": 2, "kvHeads": 2,
        "norms": "joined", "postNorm": True, "gates": True, "residual": 0.9, "embedScale": 8}
SIZES = {"T": 32, "d": 64, "H": 4, "dh": 16, "L": 2, "ff": 160}
LONG = dict(SIZES, T=300, window=270)


@pytest.mark.parametrize("sizes, graph, arena, streams", [(SIZES, False, False, 1), (SIZES, True, False, 1), (SIZES, True, True, 1), (SIZES, False, False, 2),
                                                          (LONG, True, True, 1), (LONG, False, False, 2)])
def test_trainer_is_the_checked_path_bit_for_bit(tool, sizes, graph, arena, streams):
    req = {"model": "transformer", "B": 3, "V": 301, "opt": "muon", "cfg": dict(FULL, **sizes), "graph": graph, "arena": arena, "streams": streams, "steps": 4,
           "consistency": True, "consistencySteps": 4}
    print(f"gpu step: gpu-train {req}", flush=True)
    r = tool("gpu-train", req, timeout=300)
    assert r["identical"], r["losses"]
    assert np.isfinite(r["losses"]).all() and len(r["losses"]) == 4


@pytest.mark.parametrize("sizes", [SIZES, LONG], ids=["short", "long"])
def test_a_step_of_all_operators_matches_float64(tool, tmp_path, sizes):
    import tcmi_bridge
    req = {"model": "transformer", "B": 2, "V": 150, "opt": "adam", "cfg": dict(FULL, **sizes)}
    tool("step-graph", req, out=str(tmp_path / "step"))
    b = tcmi_bridge.Bundle(tmp_path / "step")
    c = b.cases[0]
    inputs = {k: b.arr(v) for k, v in c["inputs"].items()}
    # Padding at the ends of the sequences, in tokens and targets.
    pad = np.arange(len(inputs["x"])) % sizes["T"] >= sizes["T"] - 3
    inputs["x"], inputs["y"] = (np.where(pad, np.float32(-1), inputs[k]) for k in "xy")
    keep = [c["loss"]] + list(c["outputs"].values())
    print("gpu step: gpu-graphs, a training step of all operators", flush=True)
    tool("gpu-graphs", {"graphs": [{"name": "step", "graph": c["graph"], "keep": keep, "perf": True,
                                    "inputs": {k: v.tolist() for k, v in inputs.items()}}]}, out=str(tmp_path / "gpu"), timeout=300)
    g = tcmi_bridge.Bundle(tmp_path / "gpu")
    entry = g.cases[0]
    check({"name": "step"}, entry, g)
    check_operators({"name": "step"}, inputs, entry, g)
    want = interp.evaluate(c["graph"], {k: v.astype(np.float64) for k, v in inputs.items()})
    at = {o: i for i, o in enumerate(entry["origin"])}
    loss = g.arr(entry["gpuFused"][str(at[c["loss"]])])[0]
    # Two layers of products of at most 300 terms, each off by (300 + 16) / 2^24 = 2e-5 of its magnitudes at most, and
    # logits below 1 in magnitude: losses near log 150.
    assert abs(loss - want[c["loss"]][0]) < 1e-4
