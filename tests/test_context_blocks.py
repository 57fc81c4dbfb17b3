"""Which kernels of windowAttention the test graphs take (js/src/testing/operator_cases.js): every form, by one block of lines a wavefront and by
two, forward and in the gradients of queries and of keys."""
import pathlib
import re
import shutil
import subprocess

import pytest

KERNELS = pathlib.Path(__file__).resolve().parents[1] / "tensor-compiler-webgpu_amd" / "csrc" / "kernels"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def kernels(tool, case):
    """The case's kernels: (entry, blocks of lines a wavefront), of one launch's jobs each."""
    unit = tool("kernel-unit", {"operators": [case]}, timeout=120)["unit"]
    blocks = {m.group(1): int(m.group(2)) for m in re.finditer(r"struct (\w+) \{[^}]*? HB = (\d);", unit)}
    calls = re.findall(r"tcmi::(window_(?:rows|wide(?:_dq|_dkv)?|packed(?:_dq|_dkv)?))<(\w+)", unit)
    return {(entry, blocks.get(sizes, 1)) for entry, sizes in calls}


@pytest.mark.parametrize("name, taken", [
    ("blocks", {("window_packed", 2), ("window_packed_dq", 2), ("window_packed_dkv", 2)}),
    ("blocks-odd", {("window_packed", 2), ("window_packed_dq", 2), ("window_packed_dkv", 2)}),
    ("blocks-first", {("window_packed", 2), ("window_packed_dq", 2), ("window_packed_dkv", 2)}),
    ("blocks-large", {("window_packed", 2), ("window_packed_dq", 1), ("window_packed_dkv", 1)}),
    ("blocks-largest", {("window_packed", 2)}),
    ("exact-packed-blocks", {("window_packed", 2), ("window_packed_dq", 2), ("window_packed_dkv", 2)}),
])
def test_two_blocks_a_wavefront(tool, name, taken):
    case = tool("operator-graphs", {"forms": [f"window-{name}"]})[0]["case"]
    assert kernels(tool, case) == taken


def test_every_form_is_run(tool):
    cases = [g["case"] for g in tool("operator-graphs", {"context": True, "family": "window"})]
    found = set().union(*(kernels(tool, c) for c in cases))
    assert found >= {("window_rows", 1), ("window_wide", 1), ("window_wide_dq", 1), ("window_wide_dkv", 1), ("window_packed", 1), ("window_packed_dq", 1),
                     ("window_packed_dkv", 1)}


def test_no_size_is_written_that_no_kernel_reads(tool):
    """The constants of a launch's struct are read by its kernels; blocks of lines are a choice of split operands alone."""
    headers = "".join(p.read_text() for p in KERNELS.glob("tcmi_*.h"))
    cases = [g["case"] for g in tool("operator-graphs", {"context": True})]
    unit = tool("kernel-unit", {"operators": cases}, timeout=120)["unit"]
    structs = {m.group(1): m.group(2) for m in re.finditer(r"struct (\w+_s\d*) \{\n(.*?)\n\};", unit, re.S)}
    names = {n for body in structs.values() for n in re.findall(r"constexpr \w+ (\w+) = ", body)}
    assert not [n for n in names if not re.search(rf"::{n}\b", headers + unit)]
    for entry, sizes in re.findall(r"tcmi::(window_(?:rows|wide(?:_dq|_dkv)?|packed(?:_dq|_dkv)?))<(\w+)", unit):
        assert ("HB" in re.findall(r" (\w+) = ", structs[sizes])) == ("packed" in entry), (entry, sizes)


# Sizes whose kernels keep registers in memory, and how many bytes a lane at most; rows and heads next to them that keep none.
SPILLS = [
    ({"family": "window", "q": [8, 1024, 8, 128], "k": [8, 1024, 8, 128]}, 48), ({"family": "window", "q": [1, 2048, 8, 128], "k": [1, 2048, 2, 128]}, 48),
    ({"family": "window", "q": [4, 512, 8, 128], "k": [4, 4096, 2, 128]}, 48), ({"family": "window", "q": [4, 512, 8, 112], "k": [4, 4096, 2, 112]}, 0),
    ({"family": "window", "q": [2, 16384, 16, 128], "k": [2, 16384, 4, 128], "options": {"window": 1024, "sinks": 4}}, 0),
    ({"family": "window", "q": [4, 1, 8, 128], "k": [4, 50000, 2, 128]}, 0), ({"family": "window", "q": [1, 4096, 8, 192], "k": [1, 4096, 2, 192], "gradient": True}, 0),
    ({"family": "residual", "x": [64, 6000], "vectors": ["gain", "bias", "postGain", "postBias", "gate"], "gradient": True}, 0),
    ({"family": "residual", "x": [64, 8192], "vectors": ["gain", "postGain", "gate"], "gradient": True}, 0),
    ({"family": "residual", "x": [64, 8192], "vectors": ["gain", "bias", "postGain", "postBias", "gate"], "gradient": True}, 20),
    ({"family": "residual", "x": [64, 16384], "vectors": ["gain", "bias", "postGain", "postBias", "gate"], "gradient": True}, 664),
]


@pytest.mark.skipif(not pathlib.Path(HIPCC).exists(), reason="hipcc is not installed")
def test_registers_kept_in_memory(tool, tmp_path):
    """Compiled for gfx950 with the runner's options."""
    lists = [tool("kernel-unit", {"operators": [c]}, timeout=120)["kernels"] for c, _ in SPILLS]
    src = tmp_path / "unit.hip"
    src.write_text(tool("kernel-unit", {"operators": [c for c, _ in SPILLS]}, timeout=120)["unit"])
    opts = ["-O3", "-std=c++17", "-ffp-contract=off", "-fno-fast-math", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    p = subprocess.run([HIPCC, "--offload-arch=gfx950", *opts, f"-I{KERNELS}", "--cuda-device-only", "-c", str(src), "-o", str(tmp_path / "unit.o"),
                        "-Rpass-analysis=kernel-resource-usage"], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stderr[-2000:]
    scratch, name = {}, None
    for m in re.finditer(r"(Function Name|ScratchSize \[bytes/lane\]): (\S+)", p.stderr):
        if m.group(1) == "Function Name":
            name = m.group(2)
        else:
            scratch[name] = int(m.group(2))
    for (case, most), names in zip(SPILLS, lists):
        assert max(scratch[n] for n in names) <= most, (case, {n: scratch[n] for n in names})
