"""Forms, tiles and ranges of the operators that test_gpu_operators.py's sizes do not take, on the GPU in both lowerings,
against float64 within what their roundings allow."""
import pytest

import operator_checks as checks
import operator_forms
from test_gpu_operators import check

pytestmark = pytest.mark.gpu


def check_forms(tool, directory, names):
    cases = operator_forms.forms(tool, names)
    inputs = [checks.inputs_of(c["case"], c["graph"], 300 + k) for k, c in enumerate(cases)]
    for c, v, entry, b in operator_forms.run(tool, directory, cases, inputs):
        check(c, v, entry, b)


def test_coefficients_near_zero(tool, tmp_path):
    """b and c of 0, and next to it: the products' scales are as far apart as they get."""
    check_forms(tool, tmp_path, ["linear", "nearly-linear"])
