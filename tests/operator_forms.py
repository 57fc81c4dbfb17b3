"""Graphs of the operators' forms (js/src/testing/operator_cases.js FORMS) run on the GPU in both lowerings."""
import operator_checks as checks


def forms(tool, names):
    cases = tool("operator-graphs", {"forms": names}, timeout=120)
    assert [c["name"] for c in cases] == names
    return cases


def run(tool, directory, cases, inputs):
    """[(case, inputs, what the GPU gave, its bundle)] of `cases` (operator-graphs' records) on `inputs` by name."""
    import tcmi_bridge
    reqs = [{"name": c["name"], "graph": c["graph"], "keep": c["keep"], "perf": True, "tuning": c["case"].get("tuning"),
             "inputs": {n: checks.plain(x) for n, x in v.items()}} for c, v in zip(cases, inputs)]
    print("gpu step: gpu-graphs " + ", ".join(c["name"] for c in cases), flush=True)
    tool("gpu-graphs", {"graphs": reqs}, out=str(directory), timeout=300)
    b = tcmi_bridge.Bundle(directory)
    got = {c["name"]: c for c in b.cases}
    return [(c, v, got[c["name"]], b) for c, v in zip(cases, inputs)]
