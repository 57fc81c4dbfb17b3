"""Which kernels of windowAttention the test graphs take (js/src/testing/operator_cases.js): every form, by one block of lines a wavefront and by
two, forward and in the gradients of queries and of keys."""
import re

import pytest


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
    import pathlib
    headers = "".join(p.read_text() for p in (pathlib.Path(__file__).resolve().parents[1] / "tensor-compiler-webgpu_amd" / "csrc" / "kernels").glob("tcmi_*.h"))
    cases = [g["case"] for g in tool("operator-graphs", {"context": True})]
    unit = tool("kernel-unit", {"operators": cases}, timeout=120)["unit"]
    structs = {m.group(1): m.group(2) for m in re.finditer(r"struct (\w+_s\d*) \{\n(.*?)\n\};", unit, re.S)}
    names = {n for body in structs.values() for n in re.findall(r"constexpr \w+ (\w+) = ", body)}
    assert not [n for n in names if not re.search(rf"::{n}\b", headers + unit)]
    for entry, sizes in re.findall(r"tcmi::(window_(?:rows|wide(?:_dq|_dkv)?|packed(?:_dq|_dkv)?))<(\w+)", unit):
        assert ("HB" in re.findall(r" (\w+) = ", structs[sizes])) == ("packed" in entry), (entry, sizes)
