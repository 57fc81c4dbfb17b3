"""The operators' forms (js/src/testing/operator_cases.js FORMS) without a GPU: which kernels they take, and that those kernels are whole."""
import pathlib
import re
import shutil
import subprocess

import numpy as np
import pytest

import operator_forms

KERNELS = pathlib.Path(__file__).resolve().parents[1] / "tensor-compiler-webgpu_amd" / "csrc" / "kernels"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def assembly(tool, directory, cases):
    """The gfx950 assembly of every kernel of `cases`, by name, with the runner's options."""
    r = tool("kernel-unit", {"operators": cases}, timeout=120)
    src, out = directory / "unit.hip", directory / "unit.s"
    src.write_text(r["unit"])
    opts = ["-O3", "-std=c++17", "-ffp-contract=off", "-fno-fast-math", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    p = subprocess.run([HIPCC, "--offload-arch=gfx950", *opts, f"-I{KERNELS}", "--cuda-device-only", "-S", str(src), "-o", str(out)],
                       capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stderr[-2000:]
    text = out.read_text()
    return {k: text[text.index(f"\n{k}:"):text.index(f".size\t{k}")] for k in r["kernels"]}


@pytest.mark.skipif(not pathlib.Path(HIPCC).exists(), reason="hipcc is not installed")
def test_every_kernel_writes_its_result_whatever_the_coefficients(tool, tmp_path):
    """Scales of 2^-70 and further apart once left the last product without a store."""
    kernels = assembly(tool, tmp_path, [g["case"] for g in operator_forms.forms(tool, ["linear", "nearly-linear"])])
    assert sum("orthapply" in k for k in kernels) == 3
    for name, text in kernels.items():
        assert re.search(r"global_store|buffer_store", text), name
        if re.search("gram|poly|apply", name):
            assert "v_mfma" in text, name


@pytest.mark.parametrize("c", [0, 1e-20, -1e-20, 1e-300, 1e-9])
def test_how_far_singular_values_grow_does_not_hang_on_a_last_coefficient_near_zero(tool, c):
    """45·(s - s³) reaches 17.3 between its zeros at 0 and 1: past what the pairs' scales hold."""
    import tcmi_bridge
    case = {"name": "grows", "family": "orthogonalize", "x": [96, 100], "options": {"steps": 1, "coefficients": [45, -45, c]}}
    with pytest.raises(tcmi_bridge.ToolError, match="grow past 16"):
        tool("operator-graphs", {"cases": [case]})
    case["options"]["coefficients"] = [40, -40, c]       # 15.4
    tool("operator-graphs", {"cases": [case]})


def test_singular_values_stay_below_what_the_scales_are_made_for(tool):
    """Against the polynomial's largest value over a grid, of coefficients of all magnitudes and signs."""
    rng = np.random.default_rng(3)
    sets = (rng.standard_normal((400, 3)) * 10.0 ** rng.integers(-14, 2, (400, 3))).tolist() + [[3, 0, 0], [0, 1, 0], [0, 0, 1], [0, 0, 0], [1, 0, -1]]
    bounds = tool("singular-bounds", {"sets": sets})
    s = np.linspace(0, 1, 4001)
    for k, (a, b, c) in enumerate(sets):
        top = max(1, np.abs(s * (a + s * s * (b + s * s * c))).max())
        if bounds[k] is None:
            assert top > 16 * (1 - 1e-6), (a, b, c)
        else:
            assert top * (1 - 1e-12) <= bounds[k] <= top * (1 + 1e-5), (a, b, c)


@pytest.mark.parametrize("x", [[320, 3632], [1300, 777]])
def test_matrices_that_depend_on_each_other_take_the_tiles_of_one(tool, x):
    """Equal matrices side by side fill the chip together, and take other tiles; one of the other's result cannot."""
    def kernels(**more):
        return set(tool("kernel-unit", {"operators": [dict({"family": "orthogonalize", "x": x}, **more)]}, timeout=120)["kernels"])
    one = kernels()
    assert kernels(twice=True) == one
    assert not kernels(count=2) & one


# What the named graphs run, that no graph of test_gpu_operators.py does.
TAKEN = {
    "far-rows": {"LKIND": 0, "HKIND": 0, "WKIND": 0, "JOINED": "false"},
    "far-rows-pieces": {"LKIND": 0, "PIECES": 3, "HCHUNKS": None},
    "tall-logits": {"LKIND": 3, "HKIND": 0, "WKIND": 0, "CT": 32, "JOINED": "true", "PIECES": 1, "HCHUNKS": None},
    "tall-logits-pieces": {"LKIND": 3, "PIECES": 3, "HCHUNKS": None},
    "tall-values": {"LKIND": 3, "PIECES": 1},
    "tall-after": {"LKIND": 3},
    "large-split": {"LKIND": 3, "HKIND": 3, "WKIND": 2, "HCHUNKS": None, "WCHUNKS": None, "CT": 128},
    "large-whole": {"LKIND": 3, "HKIND": 3, "WKIND": 2, "HCHUNKS": 1, "WCHUNKS": 1},
    "large-pieces": {"LKIND": 3, "HKIND": 3, "WKIND": 2, "PIECES": 2, "HCHUNKS": None},
    "half": {"KIND": 0, "HALF": "true", "TALL": "false", "GSPLIT": None, "BSPLIT": None},
    "half-tall": {"KIND": 0, "HALF": "true", "TALL": "true", "GSPLIT": None, "BSPLIT": None},
    "square-tall-tiles": {"KIND": 1, "AKIND": 3, "HALF": "true", "TALL": "false"},
    "square-tall-tiles-tall": {"KIND": 1, "AKIND": 3, "HALF": "true", "TALL": "true"},
    "square-wide-tiles": {"KIND": 1, "AKIND": 2, "TALL": "false"},
    "square-wide-tiles-tall": {"KIND": 1, "AKIND": 2, "TALL": "true"},
    "square-tiles": {"KIND": 1, "AKIND": 1, "TALL": "false"},
    "square-tiles-tall": {"KIND": 1, "AKIND": 1, "TALL": "true"},
    "square-split": {"KIND": 1, "GSPLIT": 1, "GCHUNKS": 2, "BSPLIT": 1, "BCHUNKS": 2, "SP": 512},
    "stack-twins": {"KIND": 0, "batch": 3},
    "stack-twins-odd": {"KIND": 0, "batch": 2},
    "eight": {"KIND": 0, "batch": 8},
}


def test_the_named_graphs_take_the_forms_that_they_are_named_for(tool):
    """So that another choice of tiles does not leave a form untested (None: more than 1)."""
    for g in operator_forms.forms(tool, list(TAKEN)):
        sizes = operator_forms.constants(tool, g["case"])
        for k, want in TAKEN[g["name"]].items():
            if k == "batch":
                assert [b["count"] for b in g["batches"]] == [want], g["name"]
            elif want is None:
                assert int(min(sizes[k])) > 1, (g["name"], k, sizes[k])
            else:
                assert sizes[k] == {str(want)}, (g["name"], k, sizes[k])


def refused(tool, case):
    import tcmi_bridge
    with pytest.raises(tcmi_bridge.ToolError) as e:
        tool("operator-graphs", {"cases": [dict(case, name="refused")]})
    return str(e.value)


@pytest.mark.parametrize("count", [257, 0, -1])
def test_position_axes_that_no_kernel_counts_are_refused(tool, count):
    """A kernel's table names its pairs' axes in bytes."""
    case = {"family": "rotary", "x": [4, 1, 600], "positions": [4] + [count] * (count > 1), "options": {"axis": 0, "frequencies": [], "positionAxes": count}}
    if count == 0:
        case["options"].update(frequencies=[1.0], axes=[-1])
    assert "position axes" in refused(tool, case)
    tool("operator-graphs", {"cases": [{"name": "most", "family": "rotary", "x": [4, 1, 600], "positions": [4, 256],
                                        "options": {"axis": 0, "frequencies": [1.0], "axes": [255], "positionAxes": 256}}]})


@pytest.mark.parametrize("V", [5, 200])
def test_more_rows_than_a_kernel_counts_are_refused(tool, V):
    """2^32 + 5 rows were 5 in a kernel's 32 bits."""
    for N in (2 ** 28 + 1, 2 ** 32 + 5):
        assert "rows (at most 268435456)" in refused(tool, {"family": "loss", "N": N, "d": 1, "V": V, "gradient": True})


def test_equal_parts_that_run_side_by_side_pass_the_batch_check(tool):
    """Two nodes of which the same one part is kept: a batch of their own kernels, no joint launch."""
    case = {"name": "dx", "family": "rotary", "x": [3, 40, 2, 64], "positions": [40], "gain": True, "gradient": True, "twin": [3, 40, 2, 64]}
    g = tool("operator-graphs", {"cases": [case]})[0]
    keep = [k for n, k in zip(g["names"], g["keep"]) if n.startswith("dx")]
    r = tool("batch-check", {"graphs": [{"name": "dx", "graph": g["graph"], "keep": keep}]})[0]
    assert r["check"]["ok"] and len(keep) == 2
