"""windowAttention and its gradients on the GPU over float32's range, in every form (few rows, many, operands split once, one block of rows a
wavefront and two): operands far from 1 whose results are not, and what counts as no number."""
import numpy as np
import pytest

from test_gpu_context_operators import run_form

pytestmark = pytest.mark.gpu

FORMS = ["few", "wide", "wide-large", "packed", "packed-odd", "packed-large", "packed-blocks"]

# Exponents of q, k, v and dy, and the results that then stay within float32's normal numbers (those left out leave them).
FAR = {
    "keys": ((-118, 118, -10, -10), ("o", "dq")),
    "keys-back": ((-118, 118, 40, 40), ("o", "dk", "dv")),
    "queries": ((120, -120, -10, -10), ("o", "dk")),
    "queries-back": ((120, -120, 40, 40), ("o", "dq", "dv")),
    "values": ((0, 0, 118, -60), ("o", "dq", "dk", "dv")),
    "cotangents": ((0, 0, -60, 120), ("o", "dq", "dk", "dv")),
}


def exact_inputs(tool, form, seed):
    """Multiples of 1/4 below 4: of five bits, which every split of an operand holds in its first part, as it does their powers of two from
    2^-124 on; their scores (a quarter of q·k, in powers of two) are exact."""
    case = tool("operator-graphs", {"forms": [form]})[0]["case"]
    rng = np.random.default_rng(seed)
    return {n: np.clip(np.round(4 * rng.standard_normal(s)) / 4, -3.75, 3.75).astype(np.float32) for n, s in (("q", case["q"]), ("k", case["k"]), ("v", case["k"]), ("d0", case["q"]))}


@pytest.mark.parametrize("form", FORMS)
def test_far_operands_of_near_results(tool, tmp_path, form):
    """Each operand times its power of two, the scores as they were: every result is its own power of two times what it was, bit for bit."""
    v = exact_inputs(tool, f"window-exact-{form}", 5)
    runs = [{n: np.ldexp(x, e).astype(np.float32) for (n, x), e in zip(v.items(), by)} for by, _ in FAR.values()]
    _, (plain, *got) = run_form(tool, tmp_path, f"window-exact-{form}", [v] + runs)
    for (name, ((q, k, vs, d), kept)), r in zip(FAR.items(), got):
        power = {"o": vs, "dq": k + vs + d, "dk": q + vs + d, "dv": d}
        for n in kept:
            want = np.ldexp(plain[n].astype(np.float64), power[n]).astype(np.float32)
            assert np.isfinite(want).all() and want.any()
            np.testing.assert_array_equal(r[n], want, err_msg=f"{name} {n}")
