"""The operators' forms (js/src/testing/operator_cases.js FORMS) without a GPU: which kernels they take, and that those kernels are whole."""
import pathlib
import re
import shutil
import subprocess

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
