"""embedding, residualNorm and windowAttention (js/src/ir/operators.js) without a GPU: their shape rules and refusals, their
gradients' formulas against differences of their values (float64, oracle/operators.py), and how they lower: a node's
parts as one launch where the perf lowering keeps several, alone otherwise."""
import pathlib
import re
import shutil
import subprocess
import sys

import numpy as np
import pytest

from oracle import interp
import context_checks as checks

KERNELS = pathlib.Path(__file__).resolve().parents[1] / "tensor-compiler-webgpu_amd" / "csrc" / "kernels"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def graphs(tool):
    return {f"{g['case']['family']}-{g['name']}": g for g in tool("operator-graphs", {"context": True})}


def evaluate(g, v):
    with np.errstate(all="ignore"):
        return interp.evaluate(g["graph"], v)


@pytest.mark.parametrize("name", ["embedding-token", "embedding-scalar", "embedding-step", "embedding-same", "residual-plain", "residual-sum", "residual-layer",
                                  "residual-sandwich", "residual-all", "residual-full-gate", "residual-gate-alone", "residual-post-alone", "residual-layer-gain", "residual-one",
                                  "residual-only-n", "residual-only-h", "window-one", "window-token", "window-tokens", "window-tokens-beyond", "window-first",
                                  "window-self-sink", "window-sinks-tile", "window-odd-heads", "window-late", "window-more-queries"])
def test_gradients_are_those_of_differences(name, graphs):
    g = graphs[name]
    nodes, at = g["graph"]["nodes"], dict(zip(g["names"], g["keep"]))
    rng = np.random.default_rng(3)
    v = {k: x.astype(np.float64) for k, x in checks.inputs_of(g["case"], g["graph"], 7).items()}
    for k, x in v.items():
        if k not in ("tokens", "lengths"):
            # What nothing sees keeps no number; rows of zeros and of one value have no differences to speak of.
            v[k] = np.where(np.isfinite(x) & (np.abs(x) < 1e6), x, np.nan)
            if g["case"]["family"] == "residual":
                v[k] = rng.standard_normal(x.shape) + (1.0 if k.endswith("ain") else 0.3)
    values = evaluate(g, v)
    outs = [k for k in g["names"] if k in ("e", "h", "n", "o")]
    cotangents = [np.nan_to_num(v[f"d{k}"].reshape(-1)) for k in range(len(outs))]

    def total(w):
        got = evaluate(g, w)
        return sum((got[at[o]] * c).sum() for o, c in zip(outs, cotangents))

    checked = 0
    for grad in [k for k in g["names"] if k[0] == "d"]:
        x = grad[1:]
        assert np.isfinite(values[at[grad]]).all(), grad
        for _ in range(3):
            way, step = rng.standard_normal(v[x].shape), 1e-5
            slope = (total(dict(v, **{x: v[x] + step * way})) - total(dict(v, **{x: v[x] - step * way}))) / (2 * step)
            want = (values[at[grad]] * way.reshape(-1)).sum()
            # Central differences: third derivatives times step^2, and the sums' float64 roundings over it.
            scale = np.abs(values[at[grad]] * way.reshape(-1)).sum() + 1e-3
            assert abs(slope - want) <= 1e-5 * scale, (name, grad, slope, want)
            checked += 1
    assert checked >= 3


def test_a_value_read_beside_its_norm(tool, graphs):
    """h's other readers, and n without h: one gradient for both, with h's whole adjoint; h's own where n has none."""
    r = tool("residual-adjoints", {})
    assert r["both"]["has"] == ["dh", "dn"] and r["both"]["grads"] == 3
    assert r["n"]["has"] == ["dn"] and r["h"]["has"] == ["dh"]
    assert r["asked"]["h"] == "the sum of its readers' shares"


def test_parts_that_are_kept_run_as_one_launch(graphs):
    for name, parts in (("residual-all", [2, 7]), ("residual-sum", [2]), ("residual-only-n", [4]), ("residual-only-dy", [2]), ("window-step", [2, 3]),
                        ("window-only-q", [2]), ("window-token", [2, 3])):
        joint = [b["count"] for b in graphs[name]["batches"] if b["joint"]]
        assert joint == parts, (name, joint)
    for name in ("residual-values", "window-token-all", "embedding-step"):
        assert [b["count"] for b in graphs[name]["batches"]] == ([2] if name == "residual-values" else []), name
    # Without gradients the logarithm of the sums is not formed.
    assert graphs["window-token-all"]["perf"] == ["window-attention"]


def test_every_launch_reads_what_is_written_before_it(tool, graphs):
    r = tool("operator-order", {"cases": [g["case"] for g in graphs.values()]}, timeout=120)
    assert len(r) == len(graphs)
    assert all(x["ok"] for x in r), [x for x in r if not x["ok"]]


@pytest.mark.parametrize("case, why", [
    ({"family": "embedding", "tokens": [4], "V": 2 ** 24 + 1, "d": 1}, "a float32 names 2^24"),
    ({"family": "embedding", "tokens": [2 ** 28 + 1], "V": 3, "d": 1}, "at most 268435456"),
    ({"family": "embedding", "tokens": [2 ** 27], "V": 3, "d": 256}, "2^32 threads"),
    ({"family": "embedding", "tokens": [2 ** 28 - 1], "V": 3, "d": 64}, "2^32 threads"),
    ({"family": "embedding", "tokens": [1], "V": 1, "d": 2 ** 26}, "at most 67107840"),
    ({"family": "embedding", "tokens": [4], "V": 8, "d": 4, "scale": "NaN"}, "scale NaN"),
    ({"family": "residual", "x": [4, 16385], "vectors": ["gain"]}, "at most 16384"),
    ({"family": "residual", "x": [4, 8], "vectors": ["gain", "bias"], "options": {"norm": "rms"}}, "has no bias"),
    ({"family": "residual", "x": [4, 8], "vectors": ["bias"]}, "a bias without its gain"),
    ({"family": "residual", "x": [4, 8], "vectors": ["gain", "postBias"]}, "a bias without its gain"),
    ({"family": "residual", "x": [4, 8], "vectors": ["gain"], "options": {"norm": "group"}}, "norms are"),
    ({"family": "residual", "x": [4, 8], "vectors": ["gain"], "options": {"eps": -1}}, "eps"),
    ({"family": "residual", "x": [4, 8], "vectors": ["gain"], "options": {"residual": "x"}}, "a residual scale"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 3, 8]}, "a whole number of query heads"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 9]}, "equal batches and head sizes"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [2, 4, 2, 8]}, "equal batches and head sizes"),
    ({"family": "window", "q": [4, 2, 8], "k": [4, 2, 8]}, "[batch, tokens, heads, head size]"),
    ({"family": "window", "q": [1, 4, 2, 257], "k": [1, 4, 2, 257]}, "at most 256"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 8], "options": {"window": 0}}, "a window of 0"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 8], "options": {"window": 1.5}}, "a window of 1.5"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 8], "options": {"window": 2 ** 31}}, "a window of"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 8], "options": {"sinks": -1}}, "-1 sinks"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 8], "options": {"queries": "middle"}}, "queries are"),
    ({"family": "window", "q": [1, 4, 2, 8], "k": [1, 4, 2, 8], "options": {"scale": "x"}}, "scale x"),
    ({"family": "window", "q": [1, 2 ** 25, 64, 1], "k": [1, 1, 64, 1]}, "counted in 32 bits"),
    ({"family": "window", "q": [1, 1, 1, 4], "k": [1, 2 ** 30 + 1, 1, 4]}, "counted in 32 bits"),
    ({"family": "window", "q": [1, 1, 1, 4], "k": [1, 2 ** 24 + 1, 1, 4], "lengths": True}, "a float32 names 2^24"),
    ({"family": "window", "q": [4, 2 ** 27, 1, 1], "k": [4, 2 ** 27, 1, 1]}, "workgroups (at most 2^23)"),
])
def test_calls_that_are_refused(tool, case, why):
    import tcmi_bridge
    with pytest.raises(tcmi_bridge.ToolError) as e:
        tool("operator-graphs", {"cases": [dict(case, name="refused")]})
    assert why in str(e.value)


def test_operands_that_do_not_fit_and_gradients_that_are_none(tool):
    r = tool("context-refusals", {})
    assert "a table of [4,4,4]" in r["table"]
    assert "a stream and a branch of one shape" in r["branch"]
    assert "a gain of [7] for rows of 8" in r["gain"] and "a gate of [4,1] for rows of 8" in r["gate"]
    assert "keys of [1,4,2,8] and values of [1,5,2,8]" in r["values"]
    assert "lengths of [2] for 1 sequences" in r["lengths"]
    assert "not differentiable" in r["lse"]
    for k in ("embedding twice", "residual twice", "window twice"):
        assert "no adjoint rule for op" in r[k]
    for k in ("residual part", "window part", "window grad part", "residual grad part"):
        assert "no part" in r[k]


# Every form: rows of each count of lanes, heads of each size that differs, all parts.
COMPILED = [
    {"family": "embedding", "tokens": [8192], "V": 96, "d": 256, "gradient": True}, {"family": "embedding", "tokens": [32768], "V": 65536, "d": 1024, "gradient": True},
    {"family": "embedding", "tokens": [70], "V": 300000, "d": 37, "gradient": True},
    {"family": "residual", "x": [64, 256], "vectors": ["gain", "bias"], "gradient": True},
    {"family": "residual", "x": [8189, 4095], "vectors": ["gain", "postGain", "gate"], "gradient": True},
    {"family": "residual", "x": [64, 4096], "vectors": ["gain", "bias", "postGain", "postBias", "gate"], "gradient": True},
    {"family": "residual", "x": [64, 1023], "vectors": ["gain", "bias", "postGain", "postBias", "gate"], "gate": "full", "gradient": True},
    {"family": "window", "q": [32, 1, 8, 64], "k": [32, 4096, 2, 64], "lengths": True, "options": {"window": 1024, "sinks": 4}},
    {"family": "window", "q": [64, 128, 4, 64], "k": [64, 128, 4, 64], "gradient": True},
    {"family": "window", "q": [3, 1001, 6, 80], "k": [3, 1001, 3, 80], "lengths": True, "options": {"window": 257, "sinks": 3}, "gradient": True},
    {"family": "window", "q": [2, 4096, 16, 128], "k": [2, 4096, 4, 128], "options": {"window": 1024, "sinks": 4}, "gradient": True},
    {"family": "window", "q": [1, 300, 4, 256], "k": [1, 300, 2, 256], "gradient": True},
    {"family": "window", "q": [2, 37, 3, 15], "k": [2, 37, 3, 15], "gradient": True},
    {"family": "window", "q": [4, 2000, 8, 64], "k": [4, 2000, 8, 64], "options": {"window": 100}, "gradient": True},
    {"family": "window", "q": [1, 8192, 8, 64], "k": [1, 8192, 2, 64], "gradient": True}, {"family": "window", "q": [8, 1024, 8, 96], "k": [8, 1024, 2, 96], "lengths": True, "gradient": True},
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
    assert set(scratch) == set(r["kernels"]) and len(scratch) > 25
    assert not any(scratch.values()), {k: v for k, v in scratch.items() if v}


def test_the_smallest_operators_compile_beside_torch(tool, tmp_path):
    """The C ABI's compiler, in a process that has torch's own copy of it loaded."""
    cases = [{"family": "embedding", "tokens": [5], "V": 3, "d": d, "gradient": True} for d in (1, 2, 3)]
    cases += [{"family": "residual", "x": [5, d], "vectors": ["gain", "bias", "postGain", "postBias", "gate"], "gradient": True} for d in (1, 2, 3)]
    cases += [{"family": "window", "q": [2, 5, 2, d], "k": [2, 5, 1, d], "lengths": True, "options": {"window": 2}, "gradient": True} for d in (1, 2, 3)]
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
