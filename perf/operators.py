"""Operators of a transformer's training step, each as one timed pass.

  rotary         queries and keys normalised for each head (root mean square over the head, one gain vector) and
                 rotated by their tokens' positions, on one axis or on three (time, height, width); forward, or with
                 the gradients of both
  loss           softmax cross entropy of h.W + b against class indices, one loss a row (0 where the target is no
                 class); forward, or with the gradients of h, W and b
  orthogonalize  Newton-Schulz iterations that push a matrix's singular values towards 1, as an optimizer applies
                 them to an update: X <- aX + (bA + cA.A).X with A = X.X^T, from X / (|X| + eps)

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
BASE = 10000.0                            # of the rotation's frequencies
STEPS, COEFFICIENTS, TINY = 5, (3.4445, -4.7750, 2.0315), 1e-7


# ---- the cases -----------------------------------------------------------------------------

def listed():
    return [
        # One new token for each of 32 sequences, far into them, shared key heads: bound by latency.
        rotary("rotary-token", B=32, T=1, Hq=8, Hk=2, dh=64, start=131071),
        # The queries and keys of one layer of the character transformer's training step, batch 64.
        rotary("rotary-step", B=64, T=128, Hq=4, Hk=4, dh=64, gradient=True),
        # Patches of a video clip, three axes, an odd number of tokens.
        rotary("rotary-video", B=1, T=8191, Hq=16, Hk=4, dh=128, axes=3, gradient=True),
        # Two long documents, shared key heads.
        rotary("rotary-long", B=2, T=32768, Hq=32, Hk=8, dh=128),
        # A few sequences scored over the character transformer's vocabulary.
        loss("loss-small", N=128, d=64, V=96, bias=True),
        # The character transformer's own loss and its gradients, batch 64 of 128 tokens.
        loss("loss-step", N=8192, d=256, V=96, bias=True, gradient=True),
        # Evaluation over a subword vocabulary.
        loss("loss-forward", N=4096, d=512, V=32768),
        # Sizes that divide nothing.
        loss("loss-ragged", N=1001, d=515, V=50021, bias=True, gradient=True),
        # A training batch over a large vocabulary.
        loss("loss-large", N=8192, d=1024, V=65536, gradient=True),
        # The sixteen square projections of the character transformer's four layers.
        orthogonalize("orthogonalize-step", count=16, m=256, n=256),
        # A tall matrix of sizes that divide nothing.
        orthogonalize("orthogonalize-ragged", count=1, m=1300, n=777),
        # A wide model's feed-forward weights, and its square ones.
        orthogonalize("orthogonalize-large", count=2, m=4096, n=4096),
    ]


def rotary(name, B, T, Hq, Hk, dh, axes=1, start=0, gradient=False):
    return {"name": name, "family": "rotary", "B": B, "T": T, "Hq": Hq, "Hk": Hk, "dh": dh, "axes": axes, "start": start, "gradient": gradient}


def loss(name, N, d, V, bias=False, gradient=False):
    return {"name": name, "family": "loss", "N": N, "d": d, "V": V, "bias": bias, "gradient": gradient}


def orthogonalize(name, count, m, n):
    return {"name": name, "family": "orthogonalize", "count": count, "m": m, "n": n}


def draw(rng):
    def spread(lo, hi):
        """A size between lo and hi, even over its logarithm; half of them whole multiples of 16."""
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, n // 16 * 16) if n >= 16 and rng.random() < 0.5 else n

    while True:
        family = rng.choice(["rotary", "loss", "loss", "orthogonalize"])
        if family == "rotary":
            Hk = rng.choice([1, 2, 3, 4, 8])
            c = rotary(None, B=spread(1, 64), T=spread(1, 32768), Hq=Hk * rng.choice([1, 2, 4]), Hk=Hk, dh=rng.choice([16, 32, 48, 64, 96, 128, 256]),
                       axes=rng.choice([1, 3]), start=rng.choice([0, 0, rng.randint(1, 1000000)]), gradient=rng.random() < 0.5)
            fits = work(c)["bytes"] <= 2.6e9
        elif family == "loss":
            c = loss(None, N=spread(1, 8192), d=spread(8, 1024), V=spread(2, 65536), bias=rng.random() < 0.5, gradient=rng.random() < 0.6)
            fits = True
        else:
            c = orthogonalize(None, count=rng.choice([1, 1, 2, 4, 16]), m=spread(8, 4096), n=spread(8, 4096))
            fits = work(c)["flops"] <= 30 * 2 * 4096 ** 3
        if fits:
            del c["name"]
            return c


def work(case):
    """Inputs read once and outputs written once; the flops of the products (of the symmetric ones, half)."""
    c = case
    if c["family"] == "rotary":
        rows = c["B"] * c["T"] * (c["Hq"] + c["Hk"]) * c["dh"]
        return {"bytes": 4 * ((4 if c["gradient"] else 2) * rows + (4 if c["gradient"] else 2) * c["dh"] + c["axes"] * c["B"] * c["T"]), "flops": 0}
    if c["family"] == "loss":
        N, d, V = c["N"], c["d"], c["V"]
        once = N * d + d * V + (V if c["bias"] else 0)
        return {"bytes": 4 * (2 * once + 3 * N if c["gradient"] else once + 2 * N), "flops": (6 if c["gradient"] else 2) * N * d * V}
    s, l = min(c["m"], c["n"]), max(c["m"], c["n"])
    return {"bytes": 8 * c["count"] * s * l, "flops": c["count"] * STEPS * (s * s * l + s ** 3 + 2 * s * s * l)}


# ---- inputs --------------------------------------------------------------------------------

def sections(c):
    """The rotated pairs of each axis: height and width three eighths each, time the rest."""
    pairs = c["dh"] // 2
    return [pairs] if c["axes"] == 1 else [pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8]


def values(c, seed):
    """A case's inputs by name, in fp32, on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std

    if c["family"] == "rotary":
        at = torch.arange(c["T"], device="cuda") + c["start"]
        at = at + torch.randint(0, 64, (c["B"], 1), generator=gen, device="cuda")       # a sequence's own offset
        if c["axes"] == 3:
            side = max(1, math.isqrt(c["T"]) // 4)                                      # frames of side x side patches
            at = torch.stack([at // (side * side), at // side % side, at % side], dim=2)
        v = {"q": normal(c["B"], c["T"], c["Hq"], c["dh"]), "k": normal(c["B"], c["T"], c["Hk"], c["dh"], std=3.0),
             "gq": 1 + normal(c["dh"], std=0.1), "gk": 1 + normal(c["dh"], std=0.1), "at": at.float()}
        return dict(v, d0=normal(*v["q"].shape), d1=normal(*v["k"].shape)) if c["gradient"] else v
    if c["family"] == "loss":
        N, d, V = c["N"], c["d"], c["V"]
        # Logits of standard deviation 1.5, in one row of a hundred of 9 (a confident one); one target in twenty is
        # no class (padding).
        h, W = normal(N, d), normal(d, V, std=1.5 / math.sqrt(d))
        h[torch.randperm(N, generator=gen, device="cuda")[: round(N / 100)]] *= 6
        t = torch.randint(0, V, (N,), generator=gen, device="cuda").float()
        t[torch.rand(N, generator=gen, device="cuda") < 0.05] = -1.0
        v = {"h": h, "W": W, "t": t}
        if c["bias"]:
            v["b"] = normal(V, std=0.3)
        # The mean over the rows, each of its own weight.
        return dict(v, d0=(0.5 + torch.rand(N, generator=gen, device="cuda")) / N) if c["gradient"] else v
    # Gradients: noise, and four directions with as much of the norm.
    return {f"x{i}": normal(c["m"], c["n"], std=1e-3) + normal(c["m"], 4, std=5e-4) @ normal(4, c["n"]) for i in range(c["count"])}


def prepare(case, seed):
    v = values(case, seed)
    torch.cuda.synchronize()
    return {"case": case, "v": v, "program": program(case, v) if own else None}


def run(state):
    if own:
        return state["program"].run()
    return PLAIN[state["case"]["family"]](state["case"], state["v"])


# ---- plain forms ---------------------------------------------------------------------------

def turned(c, at):
    """cos and sin of each token's angles [B, T, 1, pairs], the angles in 64 bits (those of far positions need them)."""
    pairs = c["dh"] // 2
    f = BASE ** (torch.arange(pairs, dtype=torch.float64, device=at.device) / -pairs)
    if c["axes"] == 3:
        axis = torch.repeat_interleave(torch.arange(3, device=at.device), torch.tensor(sections(c), device=at.device))
        angle = at.double()[:, :, axis] * f
    else:
        angle = at.double()[:, :, None] * f
    return torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]


def rotary_plain(c, v):
    cos, sin = turned(c, v["at"])
    half = c["dh"] // 2
    out = {}

    def forward(x, gain):
        r = torch.rsqrt((x * x).mean(3, keepdim=True) + EPS)
        n = x * r * gain
        a, b = n[..., :half], n[..., half:]
        return r, torch.cat([a * cos - b * sin, b * cos + a * sin], 3)

    def backward(x, gain, r, dy):
        a, b = dy[..., :half], dy[..., half:]
        dn = torch.cat([a * cos + b * sin, b * cos - a * sin], 3)
        n = x * r
        g = dn * gain
        return r * (g - n * (g * n).mean(3, keepdim=True)), (dn * n).sum((0, 1, 2))

    rq, out["q"] = forward(v["q"], v["gq"])
    rk, out["k"] = forward(v["k"], v["gk"])
    if c["gradient"]:
        out["dq"], out["dgq"] = backward(v["q"], v["gq"], rq, v["d0"])
        out["dk"], out["dgk"] = backward(v["k"], v["gk"], rk, v["d1"])
    return out


def loss_plain(c, v):
    z = v["h"] @ v["W"]
    if c["bias"]:
        z = z + v["b"]
    kept = v["t"] >= 0
    t = v["t"].clamp(min=0).long()[:, None]
    z = z - z.amax(1, keepdim=True)
    zt = z.gather(1, t)
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    out = {"loss": torch.where(kept, (torch.log(s) - zt)[:, 0], 0.0)}
    if c["gradient"]:
        w = torch.where(kept, v["d0"], 0.0)[:, None]
        g = e * (w / s)
        g.scatter_add_(1, t, -w)
        out["dh"], out["dW"] = g @ v["W"].T, v["h"].T @ g
        if c["bias"]:
            out["db"] = g.sum(0)
    return out


def orthogonalize_plain(c, v):
    x = torch.stack([v[f"x{i}"] for i in range(c["count"])])
    a, b, d = COEFFICIENTS
    x = x / ((x * x).sum((1, 2), keepdim=True).sqrt() + TINY)
    x = x.mT.contiguous() if c["m"] > c["n"] else x
    for _ in range(STEPS):
        A = x @ x.mT
        x = a * x + (b * A + d * (A @ A)) @ x
    return {f"y{i}": y for i, y in enumerate(x.mT if c["m"] > c["n"] else x)}


PLAIN = {"rotary": rotary_plain, "loss": loss_plain, "orthogonalize": orthogonalize_plain}


# ---- the definition in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    c = case
    v = {k: x.double() for k, x in values(c, seed).items()}
    if c["family"] == "orthogonalize":
        a, b, d = COEFFICIENTS
        out = {}
        for i in range(c["count"]):
            x = v[f"x{i}"]
            x = x / (torch.linalg.matrix_norm(x) + TINY)
            for _ in range(STEPS):                       # the same polynomial from the side of the columns, if they are fewer
                if c["m"] > c["n"]:
                    A = x.T.contiguous() @ x
                    x = x @ (a * torch.eye(c["n"], dtype=x.dtype, device=x.device) + A @ (b * torch.eye(c["n"], dtype=x.dtype, device=x.device) + d * A))
                else:
                    A = x @ x.T.contiguous()
                    x = (a * torch.eye(c["m"], dtype=x.dtype, device=x.device) + A @ (b * torch.eye(c["m"], dtype=x.dtype, device=x.device) + d * A)) @ x
            out[f"y{i}"] = x
        return out
    wrt = [k for k in (("q", "k", "gq", "gk") if c["family"] == "rotary" else ("h", "W", "b")) if k in v] if c["gradient"] else []
    for k in wrt:
        v[k].requires_grad_()
    if c["family"] == "rotary":
        pairs = c["dh"] // 2
        f = BASE ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
        if c["axes"] == 1:
            angle = v["at"][..., None] * f
        else:
            angle = torch.cat([v["at"][..., i, None] * p for i, p in enumerate(torch.split(f, sections(c)))], 2)
        turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
        out = {}
        for x, g in (("q", "gq"), ("k", "gk")):
            n = v[x] / torch.sqrt(torch.linalg.vector_norm(v[x], dim=3, keepdim=True) ** 2 / c["dh"] + EPS) * v[g]
            y = torch.complex(n[..., :pairs], n[..., pairs:]) * turn
            out[x] = torch.cat([y.real, y.imag], 3)
        ys, names = [out["q"], out["k"]], {"q": "dq", "k": "dk", "gq": "dgq", "gk": "dgk"}
        ds = [v["d0"], v["d1"]] if c["gradient"] else None
    else:
        z = v["h"] @ v["W"]
        if c["bias"]:
            z = z + v["b"]
        kept = v["t"] >= 0
        picked = torch.where(kept, z.gather(1, v["t"].clamp(min=0).long()[:, None])[:, 0], 0.0)
        out = {"loss": torch.where(kept, torch.logsumexp(z, 1), 0.0) - picked}
        ys, names = [out["loss"]], {"h": "dh", "W": "dW", "b": "db"}
        ds = [v["d0"]] if c["gradient"] else None
    if wrt:
        for k, g in zip(wrt, torch.autograd.grad(ys, [v[k] for k in wrt], ds)):
            out[names[k]] = g
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
let outs = [], names = [], wrt = [], grads = [];
if (c.family === 'rotary') {
  const q = g.input('q', [c.B, c.T, c.Hq, c.dh]), k = g.input('k', [c.B, c.T, c.Hk, c.dh]);
  const gq = g.input('gq', [c.dh]), gk = g.input('gk', [c.dh]);
  const at = g.input('at', c.axes === 1 ? [c.B, c.T] : [c.B, c.T, c.axes]);
  const o = { axis: 1, sections: c.sections, base: c.base, eps: c.eps };
  outs = [g.rotary(q, at, Object.assign({ gain: gq }, o)), g.rotary(k, at, Object.assign({ gain: gk }, o))];
  names = ['q', 'k'];
  if (c.gradient) { wrt = [q, k, gq, gk]; grads = ['dq', 'dk', 'dgq', 'dgk']; }
} else if (c.family === 'loss') {
  const h = g.input('h', [c.N, c.d]), W = g.input('W', [c.d, c.V]), t = g.input('t', [c.N]);
  const b = c.bias ? [g.input('b', [c.V])] : [];
  outs = [g.linearCrossEntropy(h, W, t, b[0])];
  names = ['loss'];
  if (c.gradient) { wrt = [h, W].concat(b); grads = ['dh', 'dW', 'db'].slice(0, wrt.length); }
} else {
  for (let i = 0; i < c.count; i++) {
    outs.push(g.orthogonalize(g.input(`x${i}`, [c.m, c.n]), { steps: c.steps, coefficients: c.coefficients, eps: c.eps }));
    names.push(`y${i}`);
  }
}
let graph = g, ids = outs;
if (wrt.length) {
  const G = grad(g, outs, wrt);
  graph = G.graph;
  ids = outs.concat(G.grads);
  names = names.concat(grads);
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
    if c["family"] == "rotary":
        c.update(sections=sections(c), base=BASE, eps=EPS)
    if c["family"] == "orthogonalize":
        c.update(steps=STEPS, coefficients=COEFFICIENTS, eps=TINY)
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
        self.t.launch_dag(*self.call)
        return self.results
