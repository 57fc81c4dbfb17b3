"""windowAttention and its gradients by two blocks of rows or keys a wavefront, as long sequences and large batches take them, against float64 node by
node (test_context_blocks.py: that these graphs do). Sequences of no key and of all, windows and sinks that end inside a tile, queries
outside their sequence, heads that fill no tile."""
import pytest

import context_checks as checks
from test_gpu_context_operators import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["blocks", "blocks-odd", "blocks-first", "blocks-large", "blocks-largest"])
def test_two_blocks_match_float64(name, tmp_path, tool):
    c = tool("operator-graphs", {"forms": [f"window-{name}"]})[0]
    for entry in run(tool, tmp_path, [c], [checks.inputs_of(c["case"], c["graph"], 300)]):
        check(*entry)
