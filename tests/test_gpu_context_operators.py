"""embedding, residualNorm and windowAttention and their gradients on the GPU, in both lowerings, against float64
(oracle/operators.py) within what their roundings allow (context_checks.py): sizes from one element on, tokens that are no row, rows
of one value, windows and sinks that end inside a tile, sequences of no key, queries outside their sequence, shared heads, gradients of some
operands only. Padding past every buffer stays as it was, and the perf lowering, which runs a node's parts as one launch,
gives the plain lowering's bits."""
import numpy as np
import pytest

from oracle import interp
import context_checks as checks

pytestmark = pytest.mark.gpu


def run(tool, directory, cases, inputs):
    import tcmi_bridge
    import operator_forms
    reqs = [{"name": c["name"], "graph": c["graph"], "keep": c["keep"], "perf": True, "inputs": {n: operator_forms.text(x) for n, x in v.items()}}
            for c, v in zip(cases, inputs)]
    print("gpu step: gpu-graphs " + ", ".join(c["name"] for c in cases), flush=True)
    tool("gpu-graphs", {"graphs": reqs}, out=str(directory), timeout=300)
    b = tcmi_bridge.Bundle(directory)
    got = {c["name"]: c for c in b.cases}
    return [(c, got[c["name"]], b) for c in cases]


def check(c, entry, b):
    assert all(entry["canaryFused"]) and entry["canaryPerf"], c["name"]
    graph = entry["fused"]
    with np.errstate(all="ignore"):
        for i, n in enumerate(graph["nodes"]):
            if n["op"] not in checks.ALLOWED:
                continue
            # Node by node: its operands as the GPU had them.
            x = b.arr(entry["gpuFused"][str(i)]).astype(np.float64)
            args = [b.arr(entry["gpuFused"][str(j)]).astype(np.float64) for j in n["inputs"]]
            shapes = [graph["nodes"][j]["shape"] for j in n["inputs"]]
            want = interp.kernel(n, args, graph)
            off, allowed = np.where((x == want) | (np.isnan(x) & np.isnan(want)), 0, np.abs(x - want)), checks.ALLOWED[n["op"]](n, args, shapes)
            bad = ~(off <= allowed)
            assert not bad.any(), (c["name"], n["op"], n["attrs"].get("part"), bad.sum(), np.flatnonzero(bad)[:5], x[bad][:5], want[bad][:5], off[bad][:5], allowed[bad][:5])
            print(f"{c['name']} {n['op']} {n['attrs'].get('part', '')}: {np.max(off / np.maximum(allowed, 1e-300), initial=0):.3f} of what is allowed")
    for k, h in entry["gpuPerf"].items():
        perf, plain = b.arr(h), b.arr(entry["gpuFused"][k])
        same = np.array_equal(perf.view(np.uint32), plain.view(np.uint32))
        assert same, (c["name"], graph["nodes"][int(k)]["op"], np.flatnonzero(perf.view(np.uint32) != plain.view(np.uint32))[:5])


@pytest.mark.parametrize("family", ["embedding", "residual", "window"])
def test_operators_match_float64(family, tmp_path, tool):
    cases = tool("operator-graphs", {"context": True, "family": family})
    inputs = [checks.inputs_of(c["case"], c["graph"], 100 + k) for k, c in enumerate(cases)]
    for c, entry, b in run(tool, tmp_path, cases, inputs):
        check(c, entry, b)


def run_form(tool, directory, form, inputs):
    """The form's graph, and its kept values by name, of the perf lowering: [{name: array}] for each set of inputs."""
    c = tool("operator-graphs", {"forms": [form]})[0]
    cases = [dict(c, name=f"{form}-{k}") for k in range(len(inputs))]
    out = []
    for d, entry, b in run(tool, directory, cases, inputs):
        at = {o: i for i, o in enumerate(entry["origin"])}
        assert all(entry["canaryFused"]) and entry["canaryPerf"]
        out.append({n: b.arr(entry["gpuPerf"][str(at[k])]) for n, k in zip(c["names"], c["keep"])})
    return c, out


def window_inputs(tool, form, seed):
    case = tool("operator-graphs", {"forms": [form]})[0]["case"]
    rng = np.random.default_rng(seed)
    q, k = case["q"], case["k"]
    return q, k, {n: rng.standard_normal(s).astype(np.float32) for n, s in (("q", q), ("k", k), ("v", k), ("d0", q))}


# Of a tile of rows or less, of more, of many that share their split operands; heads of whole tiles and not.
FORMS = ["few", "few-whole", "more", "wide", "wide-large", "packed", "packed-odd"]


@pytest.mark.parametrize("form", FORMS)
def test_numbers_that_are_not_finite_reach_what_sees_them_alone(tool, tmp_path, form):
    """Two keys, a query and a row of dy of sequence 0: what sees them, or is seen by what sees them, is NaN; all else has the same bits."""
    q, k, v = window_inputs(tool, f"window-{form}", 1)
    (B, T, H, dh), (_, S, HK, _) = q, k
    bad = {n: x.copy() for n, x in v.items()}
    bad["k"][0, S - 3, 0, 1] = np.nan
    bad["v"][0, S - 2, 1, dh - 1] = np.inf
    bad["q"][0, T - 1, 0, dh // 2] = -np.inf
    bad["d0"][0, T // 2, H - 1, 0] = np.nan
    c, (plain, got) = run_form(tool, tmp_path, f"window-{form}", [v, bad])
    from oracle import operators
    node = next(n for n in c["graph"]["nodes"] if n["op"] == "windowAttention")
    sees = np.repeat(operators.window_sees(node, [None] * 3, [q, k, k])[:, None], H, 1)         # [B, H, T, S]
    R = H // HK
    bad_key = np.zeros((B, H, S), bool)
    bad_key[0, :R, S - 3] = bad_key[0, R:2 * R, S - 2] = True
    row = (sees & bad_key[:, :, None]).any(3)
    row[0, 0, T - 1] = True
    back = row.copy()
    back[0, H - 1, T // 2] = True
    key = (sees & back[..., None]).any(2).reshape(B, HK, R, S).any(2)
    want = {"o": row.transpose(0, 2, 1), "dq": back.transpose(0, 2, 1), "dk": key.transpose(0, 2, 1), "dv": key.transpose(0, 2, 1)}
    for n, touched in want.items():
        x, y = got[n].reshape(touched.shape + (dh,)), plain[n].reshape(touched.shape + (dh,))
        assert touched.any() and (n in ("dk", "dv") or not touched.all()), n
        assert np.isnan(x[touched]).all(), (n, np.argwhere(~np.isnan(x).all(-1) & touched)[:5])
        assert np.isfinite(y).all()
        np.testing.assert_array_equal(x[~touched], y[~touched], err_msg=n)


@pytest.mark.parametrize("form", FORMS[1:])
def test_numbers_of_any_size_where_a_query_does_not_see_them(tool, tmp_path, form):
    """The last keys and values 1e30 times the others: queries before them have the bits that they have without."""
    q, k, v = window_inputs(tool, f"window-{form}-forward", 2)
    del v["d0"]
    far = dict(v, k=v["k"].copy(), v=v["v"].copy())
    far["k"][:, -2:] *= np.float32(1e30)
    far["v"][:, -2:] *= np.float32(1e30)
    _, (plain, got) = run_form(tool, tmp_path, f"window-{form}-forward", [v, far])
    x, y = (r["o"].reshape(q)[:, :-2] for r in (got, plain))
    np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("form", FORMS)
def test_powers_of_two_pass_through(tool, tmp_path, form):
    """Queries 2^-40 and keys 2^40 times themselves have the scores that they had, and every result is its power of two times what it was,
    bit for bit: the scales of rows and the parts of operands lose nothing. (What is split into parts stays above 2^-102: the smallest, dS
    here, is 2^10 times what it was.)"""
    _, _, v = window_inputs(tool, f"window-{form}", 4)
    by = {"q": -40, "k": 40, "v": 30, "d0": -20}
    _, (plain, got) = run_form(tool, tmp_path, f"window-{form}", [v, {n: np.ldexp(x, by[n]).astype(np.float32) for n, x in v.items()}])
    for n, e in {"o": 30, "dq": 40 + 30 - 20, "dk": -40 + 30 - 20, "dv": -20}.items():
        np.testing.assert_array_equal(got[n], np.ldexp(plain[n], e), err_msg=n)


def test_a_padded_batch_of_the_embedding_and_its_order(tool, tmp_path):
    """Tokens in another order: the same rows, and gradients that differ by no more than their sums' roundings; all padding: zeros."""
    N, V, d = 900, 40, 36
    rng = np.random.default_rng(3)
    t = rng.integers(-1, V - 2, N).astype(np.float32)
    dy = rng.standard_normal((N, d)).astype(np.float32)
    table = rng.standard_normal((V, d)).astype(np.float32)
    order = rng.permutation(N)
    _, (a, b, none) = run_form(tool, tmp_path, "embedding-order", [{"tokens": t, "table": table, "d0": dy}, {"tokens": t[order], "table": table, "d0": dy[order]},
                                                                   {"tokens": np.full(N, -1, np.float32), "table": table, "d0": np.full((N, d), np.nan, np.float32)}])
    np.testing.assert_array_equal(a["e"].reshape(N, d)[order], b["e"].reshape(N, d))
    mass = np.zeros((V, d))
    np.add.at(mass, t[t >= 0].astype(int), 3 * np.abs(dy[t >= 0]))
    assert (np.abs(a["dtable"].reshape(V, d) - b["dtable"].reshape(V, d)) <= 2 * (N + 3) * checks.U * mass).all()
    assert not a["dtable"].reshape(V, d)[V - 2:].any() and not none["e"].any() and not none["dtable"].any()
