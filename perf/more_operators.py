"""Operators that a transformer takes to long contexts and large vocabularies, each as one timed pass.

  embedding  rows of a table by token, times a scale (zeros where the token is no row: padding); forward, or with the
             table's gradient, the sum of each token's rows
  residual   a block's branch y joined to its residual stream x and the next block's norm:
             h = residual.x + gate * norm(y), n = norm(h), norms by the root mean square or with mean and bias,
             the branch's norm and the gate where there are any; forward, or with all gradients
  attention  softmax attention whose queries see the last `window` keys up to their own and the first `sinks` keys,
             several query heads to a key head, sequences of their own lengths; forward (prompts, single tokens over a
             cache), or with the gradients of queries, keys and values

Everything is fp32, the only type the backend has. `own` false: the operators in elementary torch operations. `own`
true: the calls of a user of this framework: a graph of the builder's operators, lowered by the host modules in a node
child, its launches issued in this process through the C ABI, a program in one tcmi_launch_dag call.
"""
import ctypes
import functools
import json
import math
import os
import pathlib
import subprocess
import sys

import numpy as np
import torch

own = False

PKG = pathlib.Path(__file__).resolve().parent.parent / "tensor-compiler-webgpu_amd"
EPS = 1e-5                                # the norms' (LayerNorm's of the transformer)
CHUNK = 1024                              # queries of a sequence that the plain attention takes at a time


# ---- the cases -----------------------------------------------------------------------------

def listed():
    return [
        # The new token of each of 32 sequences over a subword vocabulary: bound by latency.
        embedding("embedding-token", N=32, V=32768, d=1024),
        # The character transformer's own tokens, batch 64 of 128, and its table's gradient: 96 rows that many tokens share.
        embedding("embedding-step", N=8192, V=96, d=256, gradient=True),
        # A training batch over a large vocabulary, as frequent as words are.
        embedding("embedding-large", N=32768, V=65536, d=1024, gradient=True),
        # One token of 32 sequences through the end of a block.
        residual("residual-token", N=32, d=1024, norm="rms", post=True),
        # The character transformer's LayerNorm after a residual sum, batch 64 of 128 tokens.
        residual("residual-step", N=8192, d=256, norm="layer", gradient=True),
        # A wide model's block with norms before and after and a gate for each channel, sizes that divide nothing.
        residual("residual-large", N=8189, d=4095, norm="rms", post=True, gate=True, gradient=True),
        # One token of 32 sequences over a cache, most of it out of the window.
        attention("attention-token", B=32, T=1, S=4096, Hq=8, Hk=2, dh=64, window=1024, sinks=4, lengths=True),
        # One token of a few very long sequences, all of the cache visible.
        attention("attention-far", B=4, T=1, S=131072, Hq=8, Hk=2, dh=64, lengths=True),
        # A layer of the character transformer's training step, batch 64.
        attention("attention-step", B=64, T=128, S=128, Hq=4, Hk=4, dh=64, gradient=True),
        # Padded sequences of sizes that divide nothing.
        attention("attention-ragged", B=3, T=1001, S=1001, Hq=6, Hk=3, dh=80, window=257, sinks=3, lengths=True, gradient=True),
        # Two long prompts through a sliding window with sinks.
        attention("attention-window", B=2, T=16384, S=16384, Hq=16, Hk=4, dh=128, window=1024, sinks=4),
        # A long document's training step, every earlier token visible.
        attention("attention-long", B=1, T=8192, S=8192, Hq=8, Hk=2, dh=64, gradient=True),
    ]


def embedding(name, N, V, d, gradient=False):
    return {"name": name, "family": "embedding", "N": N, "V": V, "d": d, "gradient": gradient}


def residual(name, N, d, norm, post=False, gate=False, gradient=False):
    return {"name": name, "family": "residual", "N": N, "d": d, "norm": norm, "post": post, "gate": gate, "gradient": gradient}


def attention(name, B, T, S, Hq, Hk, dh, window=0, sinks=0, lengths=False, gradient=False):
    return {"name": name, "family": "attention", "B": B, "T": T, "S": S, "Hq": Hq, "Hk": Hk, "dh": dh,
            "window": window, "sinks": sinks, "lengths": lengths, "gradient": gradient}


def draw(rng):
    def spread(lo, hi):
        """A size between lo and hi, even over its logarithm; half of them whole multiples of 16."""
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, n // 16 * 16) if n >= 16 and rng.random() < 0.5 else n

    while True:
        family = rng.choice(["embedding", "residual", "attention", "attention"])
        if family == "embedding":
            c = embedding(None, N=spread(1, 32768), V=spread(2, 65536), d=spread(8, 1024), gradient=rng.random() < 0.7)
        elif family == "residual":
            c = residual(None, N=spread(1, 8192), d=spread(8, 4096), norm=rng.choice(["rms", "layer"]), post=rng.random() < 0.5,
                         gate=rng.random() < 0.5, gradient=rng.random() < 0.6)
        else:
            Hk, dh = rng.choice([1, 2, 3, 4, 8]), rng.choice([16, 32, 48, 64, 80, 96, 128, 256])
            token = rng.random() < 0.35
            T = spread(1, 8) if token else spread(8, 16384)
            S = max(T, spread(16, 131072)) if token else T
            c = attention(None, B=spread(1, 32), T=T, S=S, Hq=Hk * rng.choice([1, 2, 4]), Hk=Hk, dh=dh, window=rng.choice([0, spread(1, 4096)]),
                          sinks=rng.choice([0, 0, 1, 4, 7]), lengths=rng.random() < 0.5, gradient=not token and rng.random() < 0.5)
            # (The plain form walks every sequence in chunks; a cache is held whole.)
            if work(c)["flops"] > 3e11 or 8 * c["B"] * S * Hk * dh > 6e8:
                continue
        del c["name"]
        return c


def pairs_seen(c):
    """Pairs of a query and a key that it sees, of one head of a sequence of full length."""
    at = np.arange(c["S"] - c["T"], c["S"], dtype=np.int64)
    if not c["window"]:
        return int((at + 1).sum())
    first = np.maximum(0, at - c["window"] + 1)
    return int((at + 1 - first + np.minimum(first, c["sinks"])).sum())


def work(case):
    """Inputs read once and outputs written once (of a cache, the keys that the first query or a later one sees; of an
    embedding's table, the rows that its tokens name at most); the flops of the products over pairs that see each other."""
    c = case
    if c["family"] == "embedding":
        N, V, d = c["N"], c["V"], c["d"]
        return {"bytes": 4 * (N + min(N, V) * d + N * d + ((N + V) * d if c["gradient"] else 0)), "flops": 0}
    if c["family"] == "residual":
        rows = 8 if c["gradient"] else 4
        return {"bytes": 4 * (rows * c["N"] * c["d"] + (2 if c["gradient"] else 1) * len(vectors(c)) * c["d"]), "flops": 0}
    seen = c["S"] if not c["window"] else min(c["S"], c["window"] + c["T"] - 1 + c["sinks"])
    q, k = c["B"] * c["T"] * c["Hq"] * c["dh"], c["B"] * seen * c["Hk"] * c["dh"]
    return {"bytes": 4 * ((4 * q + 4 * k) if c["gradient"] else (2 * q + 2 * k)), "flops": (14 if c["gradient"] else 4) * c["dh"] * c["Hq"] * c["B"] * pairs_seen(c)}


# ---- inputs --------------------------------------------------------------------------------

def vectors(c):
    """A residual case's operands of d elements, in the order of the call's options."""
    layer = c["norm"] == "layer"
    return (["gain"] + (["bias"] if layer else []) + ((["postGain"] + (["postBias"] if layer else [])) if c["post"] else [])
            + (["gate"] if c["gate"] else []))


def rho(c):
    """A residual case's scale of the stream: 1 but where norms stand on both sides of the block."""
    return 0.75 if c["post"] else 1.0


def scale(c):
    return math.sqrt(c["d"])


def values(c, seed):
    """A case's inputs by name, in fp32, on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if c["family"] == "embedding":
        N, V, d = c["N"], c["V"], c["d"]
        # Frequencies fall as the rank's inverse; one token in twenty is padding.
        t = (torch.exp(uniform(N).double() * math.log(V + 1)) - 1).floor().clamp(max=V - 1)
        t[uniform(N) < 0.05] = -1
        v = {"tokens": t.float(), "table": normal(V, d, std=0.02)}
        return dict(v, d0=normal(N, d, std=1e-3)) if c["gradient"] else v
    if c["family"] == "residual":
        N, d = c["N"], c["d"]
        # A stream that many blocks were added to, of channels that are larger than others; a branch off centre.
        v = {"x": normal(N, d, std=3.0) * (1 + 4 * (uniform(d) < 0.01)), "y": 0.1 + normal(N, d)}
        for k in vectors(c):
            v[k] = normal(d, std=0.1) + (0.0 if k.endswith("ias") else 0.2 if k == "gate" else 1.0)
        return dict(v, d0=normal(N, d, std=1e-3), d1=normal(N, d, std=1e-3)) if c["gradient"] else v
    B, T, S, dh = c["B"], c["T"], c["S"], c["dh"]
    # Scores of standard deviation 1.5; a cache holds other sequences' keys behind a sequence's own.
    v = {"q": normal(B, T, c["Hq"], dh, std=1.5), "k": normal(B, S, c["Hk"], dh), "v": normal(B, S, c["Hk"], dh)}
    if c["lengths"]:
        v["lengths"] = torch.randint(max(1, S // 2), S + 1, (B,), generator=gen, device="cuda").float()
    return dict(v, d0=normal(B, T, c["Hq"], dh, std=1e-2)) if c["gradient"] else v


def prepare(case, seed):
    v = values(case, seed)
    torch.cuda.synchronize()
    return {"case": case, "v": v, "program": program(case, v) if own else None}


def run(state):
    if own:
        return state["program"].run()
    return PLAIN[state["case"]["family"]](state["case"], state["v"])


# ---- plain forms ---------------------------------------------------------------------------

def embedding_plain(c, v):
    kept = v["tokens"] >= 0
    t = v["tokens"].clamp(min=0).long()
    out = {"e": torch.where(kept[:, None], v["table"][t] * scale(c), 0.0)}
    if c["gradient"]:
        dy = torch.where(kept[:, None], v["d0"] * scale(c), 0.0)
        out["dtable"] = torch.zeros_like(v["table"]).index_add_(0, t, dy)
    return out


def norm_plain(c, x, gain, bias):
    """(1 / deviation, the normalised rows, those with gain and bias)."""
    if c["norm"] == "layer":
        x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    hat = x * r
    return r, hat, hat * gain if bias is None else hat * gain + bias


def norm_back(c, r, hat, g):
    """The gradient of a norm's input from that of its normalised rows."""
    g = g - hat * (g * hat).mean(1, keepdim=True) - (g.mean(1, keepdim=True) if c["norm"] == "layer" else 0.0)
    return r * g


def residual_plain(c, v):
    p = v["y"]
    if c["post"]:
        rp, hp, p = norm_plain(c, p, v["postGain"], v.get("postBias"))
    h = rho(c) * v["x"] + (v["gate"] * p if c["gate"] else p)
    r, hat, n = norm_plain(c, h, v["gain"], v.get("bias"))
    out = {"h": h, "n": n}
    if c["gradient"]:
        dh = v["d0"] + norm_back(c, r, hat, v["d1"] * v["gain"])
        dp = dh * v["gate"] if c["gate"] else dh
        out["dx"] = rho(c) * dh
        out["dy"] = norm_back(c, rp, hp, dp * v["postGain"]) if c["post"] else dp
        sums = {"gain": lambda: v["d1"] * hat, "bias": lambda: v["d1"], "postGain": lambda: dp * hp, "postBias": lambda: dp, "gate": lambda: dh * p}
        for k in vectors(c):
            out["d" + k] = sums[k]().sum(0)
    return out


def attention_plain(c, v):
    """CHUNK queries at a time over the keys that one of them sees, of as many sequences together as keep the scores below 2^28."""
    B, T, S, Hq, Hk, dh = (c[k] for k in ("B", "T", "S", "Hq", "Hk", "dh"))
    R, f = Hq // Hk, 1 / math.sqrt(dh)
    out = {"o": torch.empty_like(v["q"])}
    if c["gradient"]:
        out.update(dq=torch.empty_like(v["q"]), dk=torch.zeros_like(v["k"]), dv=torch.zeros_like(v["v"]))
    keys = torch.arange(S, device="cuda")
    few = max(1, 2 ** 28 // (min(T, CHUNK) * S * Hq))
    for b in (slice(i, min(B, i + few)) for i in range(0, B, few)):
        n = b.stop - b.start
        for t in (slice(i, min(T, i + CHUNK)) for i in range(0, T, CHUNK)):
            m = t.stop - t.start
            # Prompts start at position 0; a token's position is its sequence's last.
            at = torch.arange(t.start + S - T, t.stop + S - T, device="cuda")[None, :, None]
            if c["lengths"] and T != S:
                at = at - S + v["lengths"][b].long()[:, None, None]
            lo, hi = 0, (t.stop if T == S else S)
            if c["window"] and T == S:
                lo = max(0, t.start - c["window"] + 1)
            ends = [slice(0, min(lo, c["sinks"])), slice(lo, hi)]
            j = torch.cat([keys[e] for e in ends])
            sees = j <= at
            if c["window"]:
                sees = sees & ((j > at - c["window"]) | (j < c["sinks"]))
            if c["lengths"]:
                length = v["lengths"][b, None, None]
                sees = sees & (j < length) & (at >= 0) & (at < length)
            # [sequences, key heads, the queries of its heads, dh]
            group = lambda x: x[b, t].reshape(n, m, Hk, R, dh).permute(0, 2, 3, 1, 4).reshape(n, Hk, R * m, dh)
            back = lambda x: x.reshape(n, Hk, R, m, dh).permute(0, 3, 1, 2, 4).reshape(n, m, Hq, dh)
            k, w = (torch.cat([x[b, e] for e in ends], 1).permute(0, 2, 1, 3).contiguous() for x in (v["k"], v["v"]))
            q, sees = group(v["q"] * f), sees.expand(n, m, len(j))[:, None, None]
            s = (q @ k.mT.contiguous()).reshape(n, Hk, R, m, -1)
            e = torch.exp(s - torch.where(sees, s, -math.inf).amax(4, keepdim=True).clamp(min=-3e38))
            e = torch.where(sees, e, 0.0)
            total = e.sum(4, keepdim=True)
            p = torch.where(total > 0, e / total, 0.0).reshape(n, Hk, R * m, -1)
            o = p @ w
            out["o"][b, t] = back(o)
            if c["gradient"]:
                g = group(v["d0"])
                ds = p * (g @ w.mT.contiguous() - (g * o).sum(3, keepdim=True))
                out["dq"][b, t] = back(ds @ k) * f
                out["dk"][b].index_add_(1, j, (ds.mT.contiguous() @ q).permute(0, 2, 1, 3))
                out["dv"][b].index_add_(1, j, (p.mT.contiguous() @ g).permute(0, 2, 1, 3))
    return out


PLAIN = {"embedding": embedding_plain, "residual": residual_plain, "attention": attention_plain}


# ---- the definition in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    c = case
    v = {k: x.double() for k, x in values(c, seed).items()}
    if c["family"] == "embedding":
        # Row by row of the table, by its tokens in order.
        t = v["tokens"]
        padded = torch.cat([v["table"], torch.zeros(1, c["d"], dtype=torch.float64, device="cuda")])
        out = {"e": padded[torch.where(t < 0, float(c["V"]), t).long()] * scale(c)}
        if c["gradient"]:
            order = torch.argsort(t, stable=True)
            order = order[t[order] >= 0]
            total = torch.cat([padded[-1:], torch.cumsum(v["d0"][order], 0)])
            ends = torch.searchsorted(t[order].contiguous(), torch.arange(c["V"], dtype=torch.float64, device="cuda"), right=True)
            out["dtable"] = torch.diff(total[ends], dim=0, prepend=total[:1]) * scale(c)
        return out
    wrt = []
    if c["gradient"]:
        wrt = ["x", "y"] + vectors(c) if c["family"] == "residual" else ["q", "k", "v"]
        for k in wrt:
            v[k].requires_grad_()
    if c["family"] == "residual":
        def norm(x, gain, bias):
            centre = x.mean(1, keepdim=True) if c["norm"] == "layer" else 0.0
            x = (x - centre) / torch.sqrt(torch.mean((x - centre) ** 2, 1, keepdim=True) + EPS) * gain
            return x if bias is None else x + bias

        p = norm(v["y"], v["postGain"], v.get("postBias")) if c["post"] else v["y"]
        h = rho(c) * v["x"] + v.get("gate", 1.0) * p
        out = {"h": h, "n": norm(h, v["gain"], v.get("bias"))}
        if wrt:
            for k, g in zip(wrt, torch.autograd.grad([out["h"], out["n"]], [v[k] for k in wrt], [v["d0"], v["d1"]])):
                out["d" + k] = g
        return {k: x.detach() for k, x in out.items()}
    B, T, S, R = c["B"], c["T"], c["S"], c["Hq"] // c["Hk"]
    if c["Hq"] * B * T * S > 1e10:
        return None
    out = {"o": torch.zeros_like(v["q"])}
    for k in wrt:
        out["d" + k] = torch.zeros_like(v[k])
    for b in range(B):
        length = v["lengths"][b] if c["lengths"] else torch.tensor(float(S), dtype=torch.float64, device="cuda")
        at = torch.arange(T, device="cuda")[:, None] + (0 if T == S else length.long() - T)
        j = torch.arange(S, device="cuda")[None]
        near = (at - j < c["window"]) if c["window"] else torch.ones_like(at - j, dtype=torch.bool)
        hidden = ~((near | (j < c["sinks"])) & (j <= at) & (j < length) & (at < length) & (at >= 0))
        empty = hidden.all(1)
        for head in range(c["Hq"]):
            q, k, w = v["q"][b, :, head], v["k"][b, :, head // R], v["v"][b, :, head // R]
            z = (q @ k.T.contiguous() / math.sqrt(c["dh"])).masked_fill(hidden, -math.inf).masked_fill(empty[:, None], 0.0)
            p = torch.softmax(z, 1).masked_fill(empty[:, None], 0.0)
            o = p @ w
            out["o"][b, :, head] = o.detach()
            if wrt:
                for name, at_head, g in zip("qkv", (head, head // R, head // R), torch.autograd.grad(o, [q, k, w], v["d0"][b, :, head])):
                    out["d" + name][b, :, at_head] += g
    return {k: x.detach() for k, x in out.items()}


# ---- the framework's calls --------------------------------------------------------------------

# Builds, fuses and lowers a case's graph; prints one buffer per owner node, the dispatches in order with their
# operands' nodes, and the kernels' text.
LOWER_JS = r"""
const fs = require('fs'), path = require('path');
const src = (p) => require(path.join(process.argv[1], 'js', 'src', p));
const c = JSON.parse(fs.readFileSync(0, 'utf8'));
const be = src('mi355x/index.js');
const { Graph } = src('ir/graph.js');
const { fuse } = src('fusion/fuse.js');
const { grad } = src('autodiff.js');
const size = (s) => s.reduce((a, b) => a * b, 1);
const g = new Graph();
let outs = [], names = [], wrt = {};
if (c.family === 'embedding') {
  const tokens = g.input('tokens', [c.N]), table = g.input('table', [c.V, c.d]);
  outs = [g.embedding(tokens, table, { scale: c.scale })];
  names = ['e'];
  wrt = { table };
} else if (c.family === 'residual') {
  const x = g.input('x', [c.N, c.d]), y = g.input('y', [c.N, c.d]), o = {};
  for (const k of c.vectors) o[k] = g.input(k, [c.d]);
  const r = g.residualNorm(x, y, Object.assign({ norm: c.norm, residual: c.rho, eps: c.eps }, o));
  outs = [r.h, r.n];
  names = ['h', 'n'];
  wrt = Object.assign({ x, y }, o);
} else {
  const q = g.input('q', [c.B, c.T, c.Hq, c.dh]), k = g.input('k', [c.B, c.S, c.Hk, c.dh]), v = g.input('v', [c.B, c.S, c.Hk, c.dh]);
  const o = { sinks: c.sinks, queries: c.T === c.S ? 'first' : 'last' };
  if (c.window) o.window = c.window;
  if (c.lengths) o.lengths = g.input('lengths', [c.B]);
  outs = [g.windowAttention(q, k, v, o)];
  names = ['o'];
  wrt = { q, k, v };
}
let graph = g, ids = outs;
if (c.gradient) {
  const G = grad(g, outs, Object.values(wrt));
  graph = G.graph;
  ids = outs.concat(G.grads);
  names = names.concat(Object.keys(wrt).map((k) => `d${k}`));
}
const f = fuse(graph, { keep: ids });
const at = ids.map((id) => f.index.get(id));
const lowered = be.lowerMI355X(f.graph, { perf: true, keep: at });
const alias = new Map(lowered.aliases || []);
const none = new Set((lowered.folded || []).concat(lowered.dead || []));
const keep = {}, shapes = {}, inputs = {}, buffers = {}, consts = {};
names.forEach((n, k) => { keep[n] = at[k]; shapes[n] = f.graph.nodes[at[k]].shape; });
for (const n of f.graph.nodes) {
  if (n.op === 'input') inputs[n.attrs.name] = n.id;
  if (alias.has(n.id) || none.has(n.id)) continue;
  buffers[n.id] = size(n.shape);
  if (n.op === 'const') consts[n.id] = n.attrs.value;
}
const batchAt = new Map((lowered.batches || []).map((b) => [b.start, b]));
const dispatches = [], L = lowered.launches;
for (let i = 0; i < L.length;) {
  const b = batchAt.get(i), members = L.slice(i, i + (b ? b.count : 1));
  for (const k of b ? b.kernels : members[0].kernels) {
    dispatches.push({ name: k.name, grid: k.grid, block: k.block, lds: k.lds, stride: b ? b.wsStride : 0,
      params: b ? null : Array.from(members[0].params), members: members.map((l) => ({ inputs: l.inputs, node: l.node })) });
  }
  i += members.length;
}
fs.writeSync(1, JSON.stringify({ keep, shapes, inputs, buffers, consts, dispatches, workspace: lowered.workspace,
  alias: Array.from(alias), sources: Array.from(be.kernelSources(lowered)) }));
"""
MAX_IN, MAX_P = 8, 48          # TcmiArgs: operand pointers and parameter words


@functools.lru_cache(maxsize=None)
def lowered(text):
    p = subprocess.run([os.environ.get("TCMI_NODE", "node"), "-e", LOWER_JS, str(PKG)], input=text.encode(), stdout=subprocess.PIPE, check=True)
    return json.loads(p.stdout)


def program(case, v):
    c = {k: x for k, x in case.items() if k != "name"}
    if c["family"] == "embedding":
        c.update(scale=scale(c))
    if c["family"] == "residual":
        c.update(vectors=vectors(c), rho=rho(c), eps=EPS)
    return Program(lowered(json.dumps(c, sort_keys=True)), v)


class Device:
    """The library, and the functions of every kernel loaded so far (a kernel's name is a hash of its text)."""

    def __init__(self):
        if str(PKG) not in sys.path:
            sys.path.insert(0, str(PKG))
        import tcmi_ctypes
        self.c, self.t = tcmi_ctypes, tcmi_ctypes.load()
        self.t.set_include_dir(str(PKG / "csrc" / "kernels").encode())
        self.t.set_cache_dir(os.environ.get("TCMI_KCACHE", str(PKG / "_build" / "kcache")).encode())
        self.t.init()
        self.loaded = {}

    def functions(self, sources):
        missing = sorted((name, text) for name, text in sources if name not in self.loaded)
        if missing:
            module = self.c.u64()
            text = '#include "tcmi_device.h"\n' + "\n".join(x for _, x in missing)
            self.t.module_compile(text.encode(), b"", ctypes.byref(module))
            for name, _ in missing:
                f = self.c.u64()
                self.t.module_function(module, name.encode(), ctypes.byref(f))
                self.loaded[name] = f.value
        return self.loaded


@functools.lru_cache(maxsize=None)
def device():
    torch.cuda.init()
    return Device()


class Buffer:
    """`n` floats from tcmi_malloc, freed with the last tensor that shows them."""

    def __init__(self, n):
        self.t = device().t
        h = device().c.u64()
        self.t.malloc(max(16, -(-n * 4 // 16) * 16), ctypes.byref(h))
        self.at, self.n = h.value, n

    def tensor(self, shape=None):
        self.__cuda_array_interface__ = {"shape": (self.n,), "typestr": "<f4", "data": (self.at, False), "version": 2}
        x = torch.as_tensor(self, device="cuda")
        return x if shape is None else x.reshape(shape)

    def __del__(self):
        self.t.free(self.at)


class Program:
    """A lowered graph's launches over one buffer per node, their argument blocks packed once, its inputs written."""

    def __init__(self, plan, inputs):
        d = device()
        c, self.t, self.plan = d.c, d.t, plan
        fns = d.functions(plan["sources"])
        self.buffers = {int(k): Buffer(n) for k, n in plan["buffers"].items()}
        for k, value in plan["consts"].items():
            b = self.buffers[int(k)]
            b.tensor().copy_(torch.tensor(value, dtype=torch.float32).reshape(-1).expand(b.n))
        for name, node in plan["inputs"].items():
            self.buffers[node].tensor().copy_(inputs[name].reshape(-1))
        for node, source in plan["alias"]:
            if source in self.buffers:          # a reshape of a value formed inside its readers has no buffer either
                self.buffers[node] = self.buffers[source]
        self.ws = Buffer(max(4, -(-plan["workspace"] // 4)))
        blocks, dims = [], []
        for k in plan["dispatches"]:
            block = b"".join(self.pointers(m, self.ws.at + i * k["stride"]) for i, m in enumerate(k["members"]))
            if k["params"] is not None:
                block += np.array((k["params"] + [0] * MAX_P)[:MAX_P], dtype=np.uint32).tobytes()
            blocks.append(block)
            dims += list(k["grid"]) + list(k["block"]) + [k["lds"]]
        n = len(blocks)
        data = b"".join(blocks)
        offsets = np.cumsum([0] + [len(b) for b in blocks]).tolist()
        self.call = (n, (c.u64 * n)(*(fns[k["name"]] for k in plan["dispatches"])), (c.u32 * (7 * n))(*dims),
                     (ctypes.c_uint8 * len(data)).from_buffer_copy(data), (c.u32 * (n + 1))(*offsets), 1,
                     (ctypes.c_uint8 * n)(), (c.i32 * n)(*([-1] * n)), (c.u32 * (n + 1))(), None)
        self.results = {k: self.buffers[i].tensor(plan["shapes"][k]) for k, i in plan["keep"].items()}
        torch.cuda.synchronize()

    def pointers(self, member, ws):
        ins = [self.buffers[i].at for i in member["inputs"]]
        return np.array(ins + [0] * (MAX_IN - len(ins)) + [self.buffers[member["node"]].at, ws], dtype=np.uint64).tobytes()

    def run(self):
        """Issues the launches on the library's own stream, which torch's streams are not ordered with, and returns the buffers that they write:
        their values are there after torch.cuda.synchronize() (or the library's sync), and inputs change after it too."""
        self.t.launch_dag(*self.call)
        return self.results
