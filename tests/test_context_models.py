"""Training steps built with the operators for long contexts and large vocabularies (token indices, sliding-window attention with
shared key heads, norms joined to the residual sums), in float64 without a GPU: without a window, a gate or a branch's norm each is the
step that it takes the place of, and a step of all of them has the gradients that differences give."""
import numpy as np
import pytest

from oracle import interp
from test_operator_models import SMALL, step

ALL = {"tokens": "indices", "targets": "classes", "positions": "rotary", "qkNorm": True, "attention": "window", "norms": "joined"}
FULL = dict(ALL, window=3, sinks=1, kvHeads=1, postNorm=True, gates=True, residual=0.8, embedScale=4)


@pytest.mark.parametrize("option", [{"tokens": "indices"}, {"attention": "window"}, {"norms": "joined"},
                                    {"attention": "window", "window": SMALL["T"], "sinks": 2}, {"tokens": "indices", "attention": "window", "norms": "joined"}])
def test_an_option_alone_trains_as_what_it_takes_the_place_of(tool, tmp_path, option):
    a, _, x = step(tool, tmp_path, "plain", cfg=SMALL, opt="adam")
    b, _, y = step(tool, tmp_path, "option", cfg=dict(SMALL, **option), opt="adam")
    assert a["names"] == b["names"]
    # (A masked score is -1e4 less there and none here: the same in float64.)
    assert abs(x[a["loss"]][0] - y[b["loss"]][0]) < 1e-10
    for n in a["outputs"]:
        np.testing.assert_allclose(y[b["outputs"][n]], x[a["outputs"][n]], rtol=1e-7, atol=1e-11, err_msg=n)


def test_a_step_of_all_options_has_the_gradients_of_differences(tool, tmp_path):
    c, inputs, v = step(tool, tmp_path, "full", cfg=dict(SMALL, **FULL), opt={"kind": "sgd", "lr": 1.0})
    assert {"b0.pn1", "b1.pn2", "b0.g1", "b1.g2"} <= set(c["names"])
    nodes = c["graph"]["nodes"]
    assert nodes[c["stepInputs"]["b0.wk"]]["shape"] == [16, 8] and nodes[c["stepInputs"]["x"]]["shape"] == [24]
    rng = np.random.default_rng(0)
    for n in ("tok", "b0.wk", "b1.wv", "b0.pn1", "b0.g2", "b1.ln2.g", "b1.w1", "lnf.b", "head"):
        grad = inputs[n].reshape(-1) - v[c["outputs"][n]]
        way, h = rng.standard_normal(inputs[n].shape), 1e-5
        at = [interp.evaluate(c["graph"], dict(inputs, **{n: inputs[n] + s * h * way}))[c["loss"]][0] for s in (1, -1)]
        slope, want = (at[0] - at[1]) / (2 * h), (grad * way.reshape(-1)).sum()
        # Third derivatives times h^2, and the loss's float64 roundings over h.
        assert abs(slope - want) <= 1e-5 * np.abs(grad * way.reshape(-1)).sum() + 1e-9, (n, slope, want)


@pytest.mark.parametrize("option, why", [({"window": 3}, "'window' takes attention"), ({"kvHeads": 1}, "'kvHeads' takes attention"), ({"gates": True}, "'gates' takes norms"),
                                         ({"residual": 0.5}, "'residual' takes norms"), ({"embedScale": 2}, "'embedScale' takes tokens"), ({"attention": "full"}, "not 'full'"),
                                         ({"norms": "none"}, "not 'none'"), ({"tokens": "words"}, "not 'words'"), ({"attention": "window", "kvHeads": 3}, "3 key heads for 2")])
def test_options_that_are_refused(tool, tmp_path, option, why):
    import tcmi_bridge
    with pytest.raises(tcmi_bridge.ToolError, match=why):
        step(tool, tmp_path, "x", cfg=dict(SMALL, **option))


STEPS = [{"model": "transformer", "B": 4, "opt": "muon", "cfg": FULL | {"kvHeads": 2}}, {"model": "transformer", "B": 3, "V": 301, "opt": "adam", "cfg": dict(FULL, **SMALL)},
         {"model": "transformer", "B": 4, "cfg": ALL, "attention": True}]


def test_a_steps_joint_launches_hold_their_own_parts(tool):
    for r in tool("batch-check", {"models": STEPS}):
        assert r["check"]["ok"], r
        assert r["check"]["saved"] > 20


def test_an_arena_keeps_a_steps_values_until_their_last_use(tool):
    for r in tool("arena-check", {"models": STEPS}):
        assert r["check"]["ok"], r
        assert r["peak"] <= r["bytes"] <= r["peak"] * 1.03 + 4096


def test_schedules_over_streams_wait_for_what_they_read(tool):
    for r in tool("schedule-check", {"models": [dict(s, V=s.get("V", 96)) for s in STEPS[:2]]}):
        assert r["check"]["ok"], r
