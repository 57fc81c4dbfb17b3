"""Training steps that run the operators together, on the GPU: rotary queries and keys with their norms before the
attention, class-index targets, orthogonalised updates. The trainer (perf lowering, parts of an operator as one launch,
equal matrices as one dispatch; captured and replayed; in the arena) gives the checked path's bits over several steps, each
operator's nodes are within what their roundings allow of float64 on the GPU's own operands, and the first loss is float64's."""
import numpy as np
import pytest

from oracle import interp
from test_gpu_operators import check

pytestmark = pytest.mark.gpu

MODERN = {"positions": "rotary", "qkNorm": True, "targets": "classes"}
SIZES = {"T": 32, "d": 64, "H": 4, "dh": 16, "L": 2, "ff": 160}


@pytest.mark.parametrize("attention, graph, arena, streams", [(False, False, False, 1), (True, True, False, 1), (True, True, True, 1), (True, False, False, 2)])
def test_trainer_is_the_checked_path_bit_for_bit(tool, attention, graph, arena, streams):
    """Over several streams every launch runs by itself, an operator's parts too."""
    req = {"model": "transformer", "B": 5, "V": 301, "opt": "muon", "cfg": dict(SIZES, **MODERN), "attention": attention, "graph": graph, "arena": arena,
           "streams": streams, "steps": 4, "consistency": True, "consistencySteps": 4}
    print(f"gpu step: gpu-train {req}", flush=True)
    r = tool("gpu-train", req, timeout=300)
    assert r["identical"], r["losses"]
    assert np.isfinite(r["losses"]).all() and len(r["losses"]) == 4


def test_a_step_of_all_operators_matches_float64(tool, tmp_path):
    import tcmi_bridge
    req = {"model": "transformer", "B": 3, "V": 150, "opt": "muon", "cfg": dict(SIZES, **MODERN)}
    tool("step-graph", req, out=str(tmp_path / "step"))
    b = tcmi_bridge.Bundle(tmp_path / "step")
    c = b.cases[0]
    inputs = {k: b.arr(v) for k, v in c["inputs"].items()}
    # Some targets that are no class: padding.
    inputs["y"] = np.where(np.arange(len(inputs["y"])) % 7 == 3, np.float32(-1), inputs["y"])
    keep = [c["loss"]] + list(c["outputs"].values())
    print("gpu step: gpu-graphs, a training step of all operators", flush=True)
    tool("gpu-graphs", {"graphs": [{"name": "step", "graph": c["graph"], "keep": keep, "perf": True,
                                    "inputs": {k: v.tolist() for k, v in inputs.items()}}]}, out=str(tmp_path / "gpu"), timeout=300)
    g = tcmi_bridge.Bundle(tmp_path / "gpu")
    entry = g.cases[0]
    check({"name": "step"}, inputs, entry, g)
    want = interp.evaluate(c["graph"], {k: v.astype(np.float64) for k, v in inputs.items()})
    at = {o: i for i, o in enumerate(entry["origin"])}
    loss = g.arr(entry["gpuFused"][str(at[c["loss"]])])[0]
    # Two layers of products of at most 160 terms, each off by (160 + 16) / 2^24 = 1e-5 of its magnitudes at most, and
    # logits below 1 in magnitude: losses near log 150.
    assert abs(loss - want[c["loss"]][0]) < 1e-4


def test_a_forward_pass_keeps_no_logits(tool, tmp_path):
    """The loss alone, of the config-5 model with class targets at batch 2: no gradient launches, within float64's loss."""
    import tcmi_bridge
    req = {"model": "transformer", "B": 2, "V": 96, "cfg": MODERN}
    tool("forward-graph", req, out=str(tmp_path / "forward"))
    b = tcmi_bridge.Bundle(tmp_path / "forward")
    c = b.cases[0]
    inputs = {k: b.arr(v) for k, v in c["inputs"].items()}
    print("gpu step: gpu-graphs, a forward pass", flush=True)
    tool("gpu-graphs", {"graphs": [{"name": "forward", "graph": c["graph"], "keep": [c["loss"]], "perf": True, "attention": True,
                                    "inputs": {k: v.tolist() for k, v in inputs.items()}}]}, out=str(tmp_path / "gpu"), timeout=300)
    g = tcmi_bridge.Bundle(tmp_path / "gpu")
    entry = g.cases[0]
    check({"name": "forward"}, inputs, entry, g)
    assert entry["kinds"].count("linear-cross-entropy") == 1 and entry["kinds"].count("rotary") == 8
    want = interp.evaluate(c["graph"], {k: v.astype(np.float64) for k, v in inputs.items()})
    loss = next(iter(entry["gpuPerf"].values()))
    assert abs(g.arr(loss)[0] - want[c["loss"]][0]) < 1e-4
