"""Training steps built with the operators that are one node each (rotary queries and keys with their norms, class-index
targets, orthogonalised updates), in float64 without a GPU: a step on class indices is the step on one-hot targets, a
head's norm and rotation are what they say, and muon's update is its formula on the gradient that its momentum holds."""
import numpy as np
import pytest

from oracle import interp

SMALL = {"T": 8, "d": 16, "H": 2, "dh": 8, "L": 2, "ff": 32}


def step(tool, tmp_path, name, **req):
    import tcmi_bridge
    d = tmp_path / name
    tool("step-graph", dict({"model": "transformer", "B": 3, "V": 13}, **req), out=str(d))
    b = tcmi_bridge.Bundle(d)
    c = b.cases[0]
    inputs = {k: b.arr(v).astype(np.float64) for k, v in c["inputs"].items()}
    return c, inputs, interp.evaluate(c["graph"], inputs)


@pytest.mark.parametrize("opt", ["sgd", "adam"])
def test_class_targets_train_as_one_hot_targets_do(tool, tmp_path, opt):
    a, _, x = step(tool, tmp_path, "onehot", cfg=SMALL, opt=opt)
    b, _, y = step(tool, tmp_path, "classes", cfg=dict(SMALL, targets="classes"), opt=opt)
    assert a["names"] == b["names"] and b["logits"] is None
    assert abs(x[a["loss"]][0] - y[b["loss"]][0]) < 1e-12
    for n in a["outputs"]:
        np.testing.assert_allclose(y[b["outputs"][n]], x[a["outputs"][n]], rtol=1e-9, atol=1e-12, err_msg=n)


def test_rotary_positions_take_the_place_of_learned_ones(tool, tmp_path):
    c, inputs, v = step(tool, tmp_path, "rotary", cfg=dict(SMALL, positions="rotary", qkNorm=True))
    assert "pos" not in c["names"] and "b1.qg" in c["names"] and "b1.kg" in c["names"]
    nodes = c["graph"]["nodes"]
    turned = [i for i, n in enumerate(nodes) if n["op"] == "rotary"]
    assert len(turned) == 2 * SMALL["L"]
    for i in turned:
        x = v[nodes[i]["inputs"][0]].reshape(3, SMALL["T"], SMALL["H"], SMALL["dh"])
        y = v[i].reshape(x.shape)
        # The first token is only normalised; every token's norm is the root of the head's size.
        n = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-5)
        np.testing.assert_allclose(y[:, 0], n[:, 0], atol=1e-12)
        np.testing.assert_allclose((y ** 2).sum(-1), (n ** 2).sum(-1), rtol=1e-10)
        # Scores between tokens of one distance turn by one angle: the pair (0, 4) turns by a radian a token.
        z = (y[..., 0] + 1j * y[..., 4]) / (n[..., 0] + 1j * n[..., 4])
        np.testing.assert_allclose(z, np.broadcast_to(np.exp(1j * np.arange(SMALL["T"]))[:, None], z.shape), atol=1e-9)


def test_muon_orthogonalises_the_blocks_matrices_and_leaves_the_rest_to_adam(tool, tmp_path):
    opt = {"kind": "muon", "lr": 0.03, "momentum": 0.9, "adam": {"kind": "adam", "lr": 1e-3, "beta1": 0.9, "beta2": 0.99, "eps": 1e-8, "weightDecay": 0}}
    c, inputs, v = step(tool, tmp_path, "muon", cfg=SMALL, opt=opt)
    a, _, x = step(tool, tmp_path, "adam", cfg=SMALL, opt=opt["adam"])
    nodes, d, ff = c["graph"]["nodes"], SMALL["d"], SMALL["ff"]
    hidden = [n for n in c["names"] if n.startswith("b") and n.split(".")[1] in ("wq", "wk", "wv", "wo", "w1", "w2")]
    assert len(hidden) == 6 * SMALL["L"] and sum(n["op"] == "orthogonalize" for n in nodes) == len(hidden)
    for n in c["names"]:
        if n not in hidden:
            np.testing.assert_allclose(v[c["outputs"][n]], x[a["outputs"][n]], rtol=1e-12, atol=1e-14, err_msg=n)
            continue
        g = v[c["outputs"][n + ".m"]].reshape(nodes[c["stepInputs"][n]]["shape"])      # the momentum starts at 0
        m = g * 1.9
        m = m / (np.linalg.norm(m) + 1e-7)
        m = m.T if m.shape[0] > m.shape[1] else m
        for _ in range(5):
            s = m @ m.T
            m = 3.4445 * m + (-4.7750 * s + 2.0315 * s @ s) @ m
        m = m.T if g.shape[0] > g.shape[1] else m
        want = inputs[n].reshape(g.shape) - 0.03 * np.sqrt(max(1, g.shape[0] / g.shape[1])) * m
        np.testing.assert_allclose(v[c["outputs"][n]].reshape(g.shape), want, rtol=1e-9, atol=1e-10, err_msg=n)
    assert d != ff


def test_an_unknown_optimizer_is_refused(tool, tmp_path):
    import tcmi_bridge
    with pytest.raises(tcmi_bridge.ToolError, match="unknown optimizer"):
        step(tool, tmp_path, "x", cfg=SMALL, opt="none")


MODERN = {"positions": "rotary", "qkNorm": True, "targets": "classes"}
STEPS = [{"model": "transformer", "B": 4, "opt": "muon", "cfg": MODERN}, {"model": "transformer", "B": 4, "opt": "muon", "cfg": MODERN, "attention": True},
         {"model": "transformer", "B": 40, "V": 301, "cfg": dict(MODERN, **SMALL)}]


def test_a_steps_joint_launches_hold_their_own_parts(tool):
    for r in tool("batch-check", {"models": STEPS}):
        assert r["check"]["ok"], r
        assert r["check"]["saved"] > 50


def test_an_arena_keeps_a_steps_values_until_their_last_use(tool):
    for r in tool("arena-check", {"models": STEPS}):
        assert r["check"]["ok"], r
        assert r["peak"] <= r["bytes"] <= r["peak"] * 1.03 + 4096
