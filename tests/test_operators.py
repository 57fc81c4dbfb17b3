"""The operators that are one node each (js/src/ir/operators.js) without a GPU: their shape rules and refusals, their
gradients' formulas against differences of their values (float64, oracle/operators.py), and how they lower: an operator's
parts as one launch where the perf lowering keeps several, alone otherwise."""
import pathlib
import re
import shutil
import subprocess
import sys

import numpy as np
import pytest

from oracle import interp
import operator_checks as checks

KERNELS = pathlib.Path(__file__).resolve().parents[1] / "tensor-compiler-webgpu_amd" / "csrc" / "kernels"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def graphs(tool):
    return {f"{g['case']['family']}-{g['name']}": g for g in tool("operator-graphs", {})}


def smooth_inputs(g, seed):
    """Inputs at which every value is finite and its differences mean something."""
    v = {k: x.astype(np.float64) for k, x in checks.inputs_of(g["case"], g["graph"], seed).items()}
    rng = np.random.default_rng(seed)
    for k, x in v.items():
        if k == "at":
            v[k] = rng.integers(0, 40, x.shape).astype(np.float64)
        elif k == "t":
            v[k] = np.where(np.isfinite(x), x, -1)
        elif not np.isfinite(x).all() or np.abs(x).max() > 1e6:
            v[k] = np.where(np.isfinite(x) & (np.abs(x) < 1e6), x, 0.3)
    return v


@pytest.mark.parametrize("name", ["rotary-token", "rotary-heads-first", "rotary-plane", "rotary-adjacent", "rotary-partial", "rotary-odd",
                                  "rotary-odd-adjacent", "rotary-norm-only", "rotary-video", "loss-few", "loss-square", "loss-ragged", "loss-squared", "loss-deep"])
def test_gradients_are_those_of_differences(name, graphs):
    g = graphs[name]
    nodes, at = g["graph"]["nodes"], dict(zip(g["names"], g["keep"]))
    v = smooth_inputs(g, 7)
    values = interp.evaluate(g["graph"], v)
    outs = [k for k in g["names"] if k[0] in "yl"]
    cotangents = {n["attrs"]["name"]: values[i] for i, n in enumerate(nodes) if n["op"] == "input" and n["attrs"]["name"][0] == "d"}

    def total(w):
        got = interp.evaluate(g["graph"], w)
        return sum((got[at[o]] * cotangents[f"d{k}"]).sum() for k, o in enumerate(outs))

    rng = np.random.default_rng(1)
    checked = 0
    for grad in [k for k in g["names"] if k[0] == "d"]:
        x = grad[1:]
        for _ in range(3):
            way = rng.standard_normal(v[x].shape)
            if x == "h":
                way *= np.isfinite(way)
            step = 1e-5
            slope = (total(dict(v, **{x: v[x] + step * way})) - total(dict(v, **{x: v[x] - step * way}))) / (2 * step)
            want = (values[at[grad]] * way.reshape(-1)).sum()
            # Central differences: third derivatives times step^2, and the sums' float64 roundings over it.
            scale = np.abs(values[at[grad]] * way.reshape(-1)).sum() + 1e-3
            assert abs(slope - want) <= 1e-5 * scale, (name, grad, slope, want)
            checked += 1
    assert checked >= 3


def test_parts_that_are_kept_run_as_one_launch(graphs):
    for name, parts in (("loss-few", 4), ("loss-square", 3), ("loss-only-h", 2), ("loss-only-b", 2), ("loss-squared", 3), ("rotary-token", 2)):
        joint = [b for b in graphs[name]["batches"] if b["joint"]]
        assert [b["count"] for b in joint] == [parts], name
    # Alone: no part to run beside.
    assert graphs["loss-values"]["batches"] == []
    # Equal queries and keys, and equal matrices, share dispatches.
    assert [b["count"] for b in graphs["orthogonalize-twins"]["batches"]] == [3]
    # The losses run beside their gradients, before anything that depends on them.
    g = graphs["loss-squared"]
    assert g["perf"][0] == "linear-cross-entropy" and g["perf"].index("linear-cross-entropy-grad") > 1


def test_equal_gradients_share_a_launch(graphs):
    """Queries' and keys' parts in one launch; not those of a rotation of a rotation, of which one reads the other."""
    assert [b["count"] for b in graphs["rotary-twins"]["batches"] if b["joint"]] == [4]
    assert [b["count"] for b in graphs["rotary-twice"]["batches"] if b["joint"]] == [2, 2]
    assert [b["count"] for b in graphs["rotary-step"]["batches"] if b["joint"]] == [2, 2]


def test_every_launch_reads_what_is_written_before_it(tool, graphs):
    r = tool("operator-order", {"cases": [g["case"] for g in graphs.values()]}, timeout=120)
    assert len(r) == len(graphs)
    assert all(x["ok"] for x in r), [x for x in r if not x["ok"]]


def refused(tool, case):
    import tcmi_bridge
    with pytest.raises(tcmi_bridge.ToolError) as e:
        tool("operator-graphs", {"cases": [dict(case, name="refused")]})
    return str(e.value)


@pytest.mark.parametrize("case, why", [
    ({"family": "rotary", "x": [8], "positions": [8]}, "two axes or more"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [4]}, "positions of"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [2, 3, 2]}, "positions of"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3, 2], "options": {"sections": [1, 1, 1]}}, "positions of"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3], "options": {"sections": [5]}}, "at most 4"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3], "options": {"sections": [1.5]}}, "counts of pairs"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3], "options": {"base": 0}}, "base"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3], "options": {"frequencies": [1, 2], "axes": [0, 1], "positionAxes": 1}}, "position axes"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3], "options": {"pairs": "thirds"}}, "pairs are"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [3], "gain": True, "options": {"eps": -1}}, "eps"),
    ({"family": "rotary", "x": [2, 3, 4, 8], "positions": [2], "options": {"axis": 3}}, "no token axis 3"),
    ({"family": "rotary", "x": [3, 1, 4098], "positions": [3], "options": {"axis": 0}}, "at most 4096"),
    ({"family": "loss", "N": 4, "d": 8, "V": 2 ** 24 + 1}, "classes"),
    ({"family": "loss", "N": 65, "d": 8, "V": 2 ** 22 + 1}, "at most 4194304"),
    ({"family": "loss", "N": 65, "d": 2 ** 22 + 1, "V": 8}, "at most 4194304"),
    ({"family": "orthogonalize", "x": [8, 2 ** 22 + 1]}, "at most 4194304"),
    ({"family": "orthogonalize", "x": [65536, 8, 8]}, "at most 65535"),
    ({"family": "orthogonalize", "x": [8]}, "two axes"),
    ({"family": "orthogonalize", "x": [8, 8], "options": {"steps": -1}}, "steps"),
    ({"family": "orthogonalize", "x": [8, 8], "options": {"steps": 1.5}}, "steps"),
    ({"family": "orthogonalize", "x": [8, 8], "options": {"coefficients": [1, 2]}}, "three finite"),
    ({"family": "orthogonalize", "x": [8, 8], "options": {"coefficients": [9, 9, 9]}}, "grow past"),
    ({"family": "orthogonalize", "x": [8, 8], "options": {"eps": -1}}, "eps"),
    ({"family": "orthogonalize", "x": [65536, 1, 1]}, "at most 65535"),
])
def test_calls_that_are_refused(tool, case, why):
    assert why in refused(tool, case)


def test_operands_that_do_not_fit_and_gradients_that_are_none(tool):
    r = tool("operator-refusals", {})
    assert set(r) == {"targets", "inner", "bias", "second", "orthogonalize", "rank", "unknown part"}
    assert "targets of [5] for 4 rows" in r["targets"]
    assert "[rows, d] by [d, classes]" in r["inner"] and "[rows, d] by [d, classes]" in r["rank"]
    assert "a bias of [6] for 5 classes" in r["bias"]
    assert "no adjoint rule for op 'linearCrossEntropyGrad'" in r["second"]
    assert "orthogonalize is not differentiable" in r["orthogonalize"]
    assert "no part 'dt'" in r["unknown part"]


# Every kind of tile and form: all parts of large and small losses of many rows and of few, wide, tall and square matrices, batched ones,
# heads of both pairings.
COMPILED = [
    {"family": "loss", "N": 1001, "d": 515, "V": 50021, "bias": True, "gradient": True}, {"family": "loss", "N": 8192, "d": 256, "V": 96, "bias": True, "gradient": True},
    {"family": "loss", "N": 4096, "d": 512, "V": 32768}, {"family": "loss", "N": 64, "d": 97, "V": 40001, "bias": True, "gradient": True},
    {"family": "loss", "N": 9, "d": 64, "V": 1000, "gradient": True}, {"family": "loss", "N": 128, "d": 64, "V": 96},
    {"family": "loss", "N": 8192, "d": 256, "V": 200, "bias": True, "gradient": True}, {"family": "loss", "N": 9000, "d": 63, "V": 127, "gradient": True},
    {"family": "orthogonalize", "x": [256, 256], "count": 16}, {"family": "orthogonalize", "x": [1300, 777]}, {"family": "orthogonalize", "x": [4096, 4096], "count": 2},
    {"family": "orthogonalize", "x": [2100, 9001]}, {"family": "orthogonalize", "x": [64, 4096], "count": 2}, {"family": "orthogonalize", "x": [999, 31]},
    {"family": "orthogonalize", "x": [3000, 61]}, {"family": "orthogonalize", "x": [7, 51]},
    {"family": "rotary", "x": [2, 64, 4, 128], "positions": [2, 64], "gain": True, "gradient": True, "twin": [2, 64, 4, 128]},
    {"family": "rotary", "x": [64, 4096], "positions": [64], "gain": True, "gradient": True, "options": {"axis": 0, "pairs": "adjacent"}},
]


@pytest.mark.skipif(not pathlib.Path(HIPCC).exists(), reason="hipcc is not installed")
def test_kernels_use_no_scratch(tool, tmp_path):
    """Compiled for gfx950 with the runner's options: no private array or spilled register in memory."""
    r = tool("kernel-unit", {"operators": COMPILED}, timeout=120)
    src = tmp_path / "unit.hip"
    src.write_text(r["unit"])
    opts = ["-O3", "-std=c++17", "-ffp-contract=off", "-fno-fast-math", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    p = subprocess.run([HIPCC, "--offload-arch=gfx950", *opts, f"-I{KERNELS}", "--cuda-device-only", "-c", str(src), "-o", str(tmp_path / "unit.o"),
                        "-Rpass-analysis=kernel-resource-usage"], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stderr[-2000:]
    scratch, name = {}, None
    for line in p.stderr.splitlines():
        m = re.search(r"(Function Name|ScratchSize \[bytes/lane\]): (\S+)", line)
        if m and m.group(1) == "Function Name":
            name = m.group(2)
        elif m:
            scratch[name] = int(m.group(2))
    assert set(scratch) == set(r["kernels"]) and len(scratch) > 40
    assert not any(scratch.values()), {k: v for k, v in scratch.items() if v}


def test_the_smallest_losses_compile_beside_torch(tool, tmp_path):
    """The C ABI's compiler, in a process that has torch's own copy of it loaded: rows of one to three floats, and as few classes, once ended that
    process (rows read under a branch a float)."""
    cases = [{"family": "loss", "N": N, "d": d, "V": V, "bias": True, "gradient": True} for N, d, V in ((63, 1, 3), (5, 2, 1), (70, 3, 2), (9, 1, 130))]
    r = tool("kernel-unit", {"operators": cases}, timeout=120)
    src = tmp_path / "unit.hip"
    src.write_text(r["unit"])
    lib = KERNELS.parents[1] / "lib" / "libtcmi.so"
    code = f"""import ctypes, torch
lib = ctypes.CDLL({str(lib)!r})
lib.tcmi_set_include_dir({str(KERNELS)!r}.encode())
lib.tcmi_set_cache_dir({str(tmp_path)!r}.encode())
raise SystemExit(lib.tcmi_precompile(open({str(src)!r}, "rb").read(), b"", b"gfx950"))"""
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, (p.returncode, p.stderr[-500:])
