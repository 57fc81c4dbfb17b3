"""windowAttention and its gradients on the GPU over float32's range, in every form (few rows, many, operands split once, one block of rows a
wavefront and two): operands far from 1 whose results are not, and what counts as no number; and residualNorm of rows whose squares are below the normal numbers."""
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
    # (dy.o leaves float32, which dv does not hang on.)
    "both": ((0, 0, 100, 100), ("o", "dv")),
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


def touched(c, v, keys, queries, cotangents):
    """Where results are NaN, by name: keys (sequence, key, key head) and rows (sequence, token, head) of q, or of dy alone, that hold no number."""
    from oracle import operators
    node = next(n for n in c["graph"]["nodes"] if n["op"] == "windowAttention")
    (B, T, H, _), (_, S, HK, _) = v["q"].shape, v["k"].shape
    R = H // HK
    sees = np.repeat(operators.window_sees(node, [None] * 3, [v["q"].shape, v["k"].shape, v["k"].shape])[:, None], H, 1)
    key = np.zeros((B, H, S), bool)
    for b, j, hk in keys:
        key[b, hk * R:(hk + 1) * R, j] = True
    row = (sees & key[:, :, None]).any(3)
    for b, t, h in queries:
        row[b, h, t] |= sees[b, h, t].any()
    back = row.copy()
    for b, t, h in cotangents:
        back[b, h, t] |= sees[b, h, t].any()
    at = (sees & back[..., None]).any(2).reshape(B, HK, R, S).any(2)
    return {"o": row.transpose(0, 2, 1), "dq": back.transpose(0, 2, 1), "dk": at.transpose(0, 2, 1), "dv": at.transpose(0, 2, 1)}


NUMBERS = ["few", "few-whole", "few-splits", "few-large", "more", "wide", "wide-large", "packed", "packed-odd", "exact-packed-blocks"]


def check_touched(tool, directory, form, v, bad, keys=(), queries=(), cotangents=()):
    c, (plain, got) = run_form(tool, directory, f"window-{form}", [v, bad])
    for n, at in touched(c, v, keys, queries, cotangents).items():
        x, y = (r[n].reshape(at.shape + (v["q"].shape[3],)) for r in (got, plain))
        assert np.isfinite(y).all() and at.any() == (n != "o" or bool(keys or queries)), n
        assert np.isnan(x[at]).all(), (n, np.argwhere(~np.isnan(x).all(-1) & at)[:5])
        np.testing.assert_array_equal(x[~at], y[~at], err_msg=n)


def normal_inputs(tool, form, seed):
    case = tool("operator-graphs", {"forms": [f"window-{form}"]})[0]["case"]
    rng = np.random.default_rng(seed)
    return {n: rng.standard_normal(s).astype(np.float32) for n, s in (("q", case["q"]), ("k", case["k"]), ("v", case["k"]), ("d0", case["q"]))}


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("form", NUMBERS)
def test_an_infinite_key(tool, tmp_path, form, sign):
    """Its scores are all infinities of one sign: -infinity is no weight of 0."""
    v = normal_inputs(tool, form, 6)
    S = v["k"].shape[1]
    v["q"][..., 1] = np.abs(v["q"][..., 1]) + np.float32(0.1)
    bad = dict(v, k=v["k"].copy())
    bad["k"][0, S - 3, 0, 1] = sign * np.inf
    check_touched(tool, tmp_path, form, v, bad, keys=[(0, S - 3, 0)])


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("form", NUMBERS)
def test_an_infinite_query(tool, tmp_path, form, sign):
    """Where every score of it is -infinity it is not a query that sees nothing."""
    v = normal_inputs(tool, form, 7)
    (_, T, H, _) = v["q"].shape
    v["k"][..., 2] = np.abs(v["k"][..., 2]) + np.float32(0.1)
    bad = dict(v, q=v["q"].copy())
    bad["q"][0, T - 1, 0, 2] = bad["q"][0, 0, H - 1, 2] = sign * np.inf
    check_touched(tool, tmp_path, form, v, bad, queries=[(0, T - 1, 0), (0, 0, H - 1)])


@pytest.mark.parametrize("operand", ["q", "k", "v", "d0"])
@pytest.mark.parametrize("form", NUMBERS)
def test_the_largest_numbers(tool, tmp_path, form, operand):
    """From 2^128 - 2^119 on, which the split into bf16 rounds to infinity: as infinite as infinity, and nothing to what does not see them. The operands
    of up to 16 rows of a key head are not split in the forward pass: there they are numbers, and in the gradients NaN wherever they are split."""
    v = normal_inputs(tool, form, 8)
    (_, T, H, dh), (_, S, _, _) = v["q"].shape, v["k"].shape
    bad = dict(v, **{operand: v[operand].copy()})
    at = {"q": (0, T - 1, 0), "k": (0, S - 3, 0), "v": (0, S - 2, 1), "d0": (0, T // 2, H - 1)}[operand]
    bad[operand][at + (dh // 2,)] = {"q": -1, "d0": -1}.get(operand, 1) * np.finfo(np.float32).max
    planted = {"queries": [at]} if operand == "q" else {"cotangents": [at]} if operand == "d0" else {"keys": [at]}
    if not form.startswith("few") or operand == "d0":
        return check_touched(tool, tmp_path, form, v, bad, **planted)
    c, (plain, got) = run_form(tool, tmp_path, f"window-{form}", [v, bad])
    for n, where in touched(c, v, **dict({"keys": (), "queries": (), "cotangents": ()}, **planted)).items():
        x, y = (r[n].reshape(where.shape + (dh,)) for r in (got, plain))
        np.testing.assert_array_equal(x[~where], y[~where], err_msg=n)
        if n == "dq" and operand != "q" or n != "dq" and n != "o" and operand == "q":
            assert np.isnan(x[where]).all(), n


@pytest.mark.parametrize("operand", ["q", "k", "v", "d0"])
@pytest.mark.parametrize("form", NUMBERS)
def test_numbers_below_the_largest(tool, tmp_path, form, operand):
    """2^128 - 2^120 is a number: in a padded batch's last sequences nothing of the first changes, and o is what a value of that size makes of it."""
    v = normal_inputs(tool, form, 9)
    (_, T, H, dh), (_, S, HK, _) = v["q"].shape, v["k"].shape
    bad = dict(v, **{operand: v[operand].copy()})
    at = {"q": (0, T - 1, 0), "k": (0, S - 1, 0), "v": (0, S - 1, 0), "d0": (0, T - 1, 0)}[operand]
    bad[operand][at + (dh // 2,)] = np.float32(2.0 ** 128 - 2.0 ** 120)
    c, (plain, got) = run_form(tool, tmp_path, f"window-{form}", [v, bad])
    where = touched(c, v, **{k: [at] if k == {"q": "queries", "d0": "cotangents"}.get(operand, "keys") else () for k in ("keys", "queries", "cotangents")})
    for n, w in where.items():
        x, y = (r[n].reshape(w.shape + (dh,)) for r in (got, plain))
        np.testing.assert_array_equal(x[~w], y[~w], err_msg=n)
        if operand == "v" and n == "o":
            # The other values' sum is below half a step of the product.
            seen = x[w][:, dh // 2]
            assert np.isfinite(x).all() and (seen > 2.0 ** 90).all()


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_rows_of_small_numbers(tool, tmp_path, norm):
    """Without an eps, rows of 2^-60 down to 2^-70, whose squares' mean is below the normal numbers from 2^-63 on: it is off by 2^-149 at most there (half a
    step of each square, whose sum is exact, and of the mean), r by half of that relative to it."""
    from oracle import operators
    form = f"residual-small-{norm}"
    D = tool("operator-graphs", {"forms": [form]})[0]["case"]["x"][-1]
    rng = np.random.default_rng(11)
    v = {k: rng.standard_normal((37, D) if k != "gain" else D).astype(np.float32) for k in ("x", "y", "gain", "d0", "d1")}
    down = 2.0 ** -np.linspace(60, 70, 37).round()[:, None]
    v["x"], v["y"] = (v["x"] * down).astype(np.float32), (v["y"] * down).astype(np.float32)
    v["d0"] = np.ldexp(v["d0"], 60).astype(np.float32)
    c, (got,) = run_form(tool, tmp_path, form, [v])
    h = (v["x"] + v["y"]).astype(np.float64)
    attrs = {"norm": norm, "eps": 0.0}
    centred = h - h.mean(1, keepdims=True) if norm == "layer" else h
    square = (centred ** 2).mean(1, keepdims=True)
    assert (square < 2.0 ** -126).any() and (square > 2.0 ** -126).any()
    off = 0.5 * 2.0 ** -149 / square + 2.0 ** -24 * (64 + 8)               # and float32's roundings: 64 terms, eight steps
    r, hat = operators.normalised(attrs, h)
    dn, g = v["d1"].astype(np.float64), v["d1"] * v["gain"].astype(np.float64)
    m, gv = (g.mean(1, keepdims=True) if norm == "layer" else 0.0), (g * hat).mean(1, keepdims=True)
    dx = r * (g - m - hat * gv) + v["d0"]
    mass = r * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(hat) * np.abs(g * hat).mean(1, keepdims=True)) + np.abs(v["d0"])
    np.testing.assert_array_equal(got["h"].reshape(h.shape), h.astype(np.float32))
    for n, want, allowed in (("n", hat * v["gain"], 2 * off * (np.abs(hat) + (r * np.abs(h).max(1, keepdims=True) if norm == "layer" else 0)) * np.abs(v["gain"])),
                             ("dx", dx, 8 * off * mass), ("dgain", (dn * hat).sum(0), 2 * (off * np.abs(dn) * (np.abs(hat) + 4)).sum(0))):
        assert (np.abs(got[n].reshape(want.shape) - want) <= allowed).all(), (n, np.abs(got[n].reshape(want.shape) - want).max(), allowed.min())
