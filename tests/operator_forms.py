"""Graphs of the operators' forms (js/src/testing/operator_cases.js FORMS) run on the GPU in both lowerings."""
import base64
import re

import numpy as np


def forms(tool, names):
    cases = {c["name"]: c for c in tool("operator-graphs", {"forms": names}, timeout=120)}
    return [cases[n] for n in names]


def constants(tool, case):
    """The sizes written into the kernels of `case`: name -> the set of its values over them, as text."""
    r = tool("kernel-unit", {"operators": [case]}, timeout=120)
    out = {}
    for name in r["kernels"]:
        m = re.search(r"struct %s_s \{\n(.*?)\n\};" % name, r["unit"], re.S)
        for k, v in re.findall(r"constexpr \w+ (\w+) = (-?\w+?)u?;", m.group(1) if m else ""):
            out.setdefault(k, set()).add(v)
    return out


def text(x):
    """Values for a request as the text of their bytes."""
    return base64.b64encode(np.ascontiguousarray(x, dtype=np.float32).tobytes()).decode()


def run(tool, directory, cases, inputs):
    """[(case, inputs, what the GPU gave, its bundle)] of `cases` (operator-graphs' records) on `inputs` by name."""
    import tcmi_bridge
    reqs = [{"name": c["name"], "graph": c["graph"], "keep": c["keep"], "perf": True, "tuning": c["case"].get("tuning"),
             "inputs": {n: text(x) for n, x in v.items()}} for c, v in zip(cases, inputs)]
    print("gpu step: gpu-graphs " + ", ".join(c["name"] for c in cases), flush=True)
    tool("gpu-graphs", {"graphs": reqs}, out=str(directory), timeout=300)
    b = tcmi_bridge.Bundle(directory)
    got = {c["name"]: c for c in b.cases}
    return [(c, v, got[c["name"]], b) for c, v in zip(cases, inputs)]
