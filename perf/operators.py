"""Activations held in 8 bits, and graph attention that reads them: the cases to measure, and the operators' plain forms.

The operators (`own` decides whether `run` calls them or computes their plain form):

* 8-bit checkpoints: a matrix is cut into groups of neighbouring columns; a group keeps int8 codes and one fp32 scale,
      scale = max|x| / 127 in fp32,   code = x / scale, exactly rounded, ties to even,   value = code * scale     (x^ below)
  and a group whose scale is below the normal numbers keeps zeros
* activations with an 8-bit checkpoint: y = f(x), and dx = dy * f'(x^), from the checkpoint of x alone
* dot-product attention over the incoming edges u -> v of every node, on 8-bit queries, keys and values (a scale per node
  and head), with z = scale * <q^[v], k^[u]>, p = softmax of z over v's incoming edges, out[v] = sum p v^[u]; a node without
  edges gets zeros
* its gradient from the same 8-bit tensors, the probabilities computed anew: o^ the 8-bit form of the incoming gradient,
      dp = <o^[v], v^[u]>,  delta[v] = sum p dp,  ds = p (dp - delta[v]) * scale,
      dq[v] = sum ds k^[u],   dk[u] = sum ds q^[v],   dv[u] = sum p o^[v]
* the attention of a few nodes whose queries just arrived, over keys and values that are kept in 8 bits
"""
from __future__ import annotations

import math

import torch

own = False

# The node and edge counts of this package's benchmark graphs.
FULL = {"nodes": 232_965, "edges": 114_615_892}
DENSE = {"nodes": 232_965, "edges": 20_000_000}
MID = {"nodes": 169_343, "edges": 1_166_243}
SMALL = {"nodes": 19_717, "edges": 88_648}


def listed():
    return [
        # checkpoint of a hidden layer of a small model, made and read back: launches and host time
        {"name": "checkpoint_small", "kind": "checkpoint", "rows": 2000, "cols": 100, "group": 128, "type": "float32"},
        # checkpoint of the input features of the full graph: ragged rows, the last group is short
        {"name": "checkpoint_large", "kind": "checkpoint", "rows": 232_965, "cols": 602, "group": 128, "type": "float32"},
        # activation of a small attention model (8 heads of 8), forward and backward
        {"name": "activation_small", "kind": "activation", "rows": 19_717, "cols": 64, "group": 128, "f": "elu",
         "type": "float32"},
        # activation of the hidden layer of the full-graph model, forward and backward
        {"name": "activation_large", "kind": "activation", "rows": 232_965, "cols": 256, "group": 128, "f": "gelu",
         "type": "float32"},
        # the same in half the bits, odd rows, as under autocast
        {"name": "activation_bf16", "kind": "activation", "rows": 169_343, "cols": 601, "group": 64, "f": "silu",
         "type": "bfloat16"},
        # training pass of an attention layer on a small citation network: latency
        {"name": "attention_small", "kind": "attention", **SMALL, "heads": 8, "d": 8, "train": True, "type": "float32"},
        # training pass on a sparse graph, 8 edges per node
        {"name": "attention_mid", "kind": "attention", **MID, "heads": 4, "d": 32, "train": True, "type": "float32"},
        # odd number of heads of an odd width, half the bits
        {"name": "attention_odd", "kind": "attention", "nodes": 100_003, "edges": 4_000_037, "heads": 3, "d": 41,
         "train": True, "type": "bfloat16"},
        # training pass on a denser graph: 86 edges per node, hubs with tens of thousands
        {"name": "attention_dense", "kind": "attention", **DENSE, "heads": 4, "d": 32, "train": True, "type": "float32"},
        # evaluation pass on the full graph: 492 edges per node, hubs with more than 10^5
        {"name": "attention_eval", "kind": "attention", **FULL, "heads": 4, "d": 16, "train": False, "type": "float32"},
        # one node is asked for
        {"name": "rows_one", "kind": "rows", **DENSE, "rows": 1, "heads": 4, "d": 32, "type": "float32"},
        # a batch of nodes is asked for
        {"name": "rows_batch", "kind": "rows", **DENSE, "rows": 1024, "heads": 4, "d": 32, "type": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["checkpoint", "activation", "attention", "attention", "attention", "rows"])
    c = {"kind": kind, "type": rng.choice(["float32", "float32", "bfloat16", "float16"])}
    if kind in ("checkpoint", "activation"):
        c.update(rows=_log(rng, 200, 232_965), cols=_log(rng, 3, 602), group=rng.choice([8, 32, 64, 100, 128, 128, 256]))
        if kind == "activation":
            c["f"] = rng.choice(["elu", "gelu", "silu"])
        return c
    n = _log(rng, 2000, 232_965)
    heads = rng.choice([1, 1, 2, 3, 4, 4, 6, 8])
    d = _log(rng, 4, 256 // heads)
    if rng.random() < 0.5:
        d = min(max(8, d // 8 * 8), 256 // heads)
    most = 20_000_000 if heads * d <= 128 else 8_000_000
    c.update(nodes=n, edges=_log(rng, 4 * n, min(most, max(8 * n, int(n ** 1.5 * 0.9)))), heads=heads, d=d)
    if kind == "attention":
        c["train"] = rng.random() < 0.75
    else:
        c["rows"] = _log(rng, 1, 2000)
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _edges(case, gen):
    """Edges whose two ends both follow a power law (the most referenced node takes part in about n^-1/2 of them); some
    nodes have none, some edges are there twice."""
    n, e = case["nodes"], case["edges"]

    def ends():
        rank = (torch.rand(e, device="cuda", generator=gen).double().square() * n).long().clamp_(max=n - 1)
        return torch.randperm(n, device="cuda", generator=gen).to(torch.int32)[rank]

    return ends(), ends()


def _inputs(case, seed):
    gen = _generator(seed)
    dtype = getattr(torch, case["type"])

    def randn(*shape, by=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * by).to(dtype)

    kind = case["kind"]
    if kind == "checkpoint":
        return {"x": randn(case["rows"], case["cols"])}
    if kind == "activation":
        return {"x": randn(case["rows"], case["cols"], by=1.5), "grad": randn(case["rows"], case["cols"])}
    n, h, d = case["nodes"], case["heads"], case["d"]
    src, dst = _edges(case, gen)
    s = {"src": src, "dst": dst, "q": randn(n if kind == "attention" else case["rows"], h, d), "k": randn(n, h, d),
         "v": randn(n, h, d)}
    if kind == "attention":
        s["grad"] = randn(n, h, d, by=0.01)
    else:
        s["rows"] = torch.randint(0, n, (case["rows"],), device="cuda", generator=gen)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind in ("attention", "rows"):
        if own:
            import tango_b200 as T
            from tango_b200.graph import Graph
            s["graph"] = T.graph_preprocess(Graph(s.pop("src"), s.pop("dst"), case["nodes"]), hub_block=0)
            if kind == "rows":
                s["k8"], s["v8"] = T.pack8(s.pop("k"), case["d"]), T.pack8(s.pop("v"), case["d"])
        elif kind == "rows":        # what a program that serves keeps: the incoming edges node by node, keys and values in 8 bits
            dst, order = torch.sort(s.pop("dst"))
            s["src"] = s["src"][order]
            s["indptr"] = torch.searchsorted(dst.long(), torch.arange(case["nodes"] + 1, device="cuda"))
            for name in ("k", "v"):
                code, scale = _codes(s.pop(name).flatten(1), case["d"])
                s[name + "8"] = code.view(case["nodes"], case["heads"], case["d"]).to(torch.int8), scale.unsqueeze(-1)
    if own and kind != "rows":
        for name in ("q", "k", "v", "x"):
            if name in s and kind != "checkpoint":
                s[name].requires_grad_(case.get("train", True))
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _codes(x, group):
    """Codes [rows, cols] (whole numbers in fp32) and scales [rows, groups] of a matrix."""
    rows, cols = x.shape
    groups = -(-cols // group)
    x = torch.nn.functional.pad(x.float(), (0, groups * group - cols)).view(rows, groups, group)
    top = x.abs().amax(-1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, torch.zeros_like(scale), scale)
    code = (x.double() / torch.where(scale > 0, scale, torch.full_like(scale, math.inf)).double()).round()  # 64 bits: a border stays one
    code = code.clamp(-127, 127).float()
    return code.reshape(rows, groups * group)[:, :cols], scale.squeeze(-1)


def _values(x, group):
    code, scale = _codes(x, group)
    return code * scale.repeat_interleave(group, 1)[:, :code.size(1)]


def _head_values(t):
    return _values(t.flatten(1), t.size(2)).view(t.shape)


def _f(x, f):
    if f == "elu":
        return torch.where(x > 0, x, torch.expm1(x.clamp(max=0)))
    if f == "gelu":
        return x * 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    return x / (1 + torch.exp(-x))


def _df(x, f):
    if f == "elu":
        return torch.exp(x.clamp(max=0))
    if f == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-x))
    return s * (1 + x * (1 - s))


def _softmax(z, at, n):
    """Softmax of edge scores over the edges that end in the same place `at`."""
    top = torch.full((n,), -math.inf, device=z.device).scatter_reduce_(0, at, z, "amax")
    p = torch.exp(z - top[at])
    total = torch.zeros(n, device=z.device, dtype=torch.float64).index_add_(0, at, p.double())
    return p / total.float()[at]


def _plain_attention(s):
    case = s["case"]
    n, h, d = case["nodes"], case["heads"], case["d"]
    scale = 1 / math.sqrt(d)
    src, dst = s["src"].long(), s["dst"].long()
    q, k, v = (_head_values(s[name]) for name in "qkv")
    grad = _head_values(s["grad"]) if case["train"] else None

    def gathered(t, at):
        return t[:, i].contiguous().index_select(0, at)

    def summed(t, at):
        return torch.zeros(n, t.size(1) if t.dim() > 1 else 1, device=t.device).index_add_(0, at, t.view(t.size(0), -1))

    outs = [torch.empty(n, h, d, device=q.device) for _ in range(4 if case["train"] else 1)]
    for i in range(h):
        z = torch.empty(case["edges"], device=q.device)
        step = 1 << 24
        for a in range(0, case["edges"], step):
            z[a:a + step] = (gathered(q, dst[a:a + step]) * gathered(k, src[a:a + step])).sum(-1) * scale
        p = _softmax(z, dst, n)
        outs[0][:, i] = summed(p[:, None] * gathered(v, src), dst)
        if not case["train"]:
            continue
        for a in range(0, case["edges"], step):
            z[a:a + step] = (gathered(grad, dst[a:a + step]) * gathered(v, src[a:a + step])).sum(-1)
        delta = torch.zeros(n, device=q.device, dtype=torch.float64).index_add_(0, dst, (p * z).double()).float()
        ds = p * (z - delta[dst]) * scale
        outs[1][:, i] = summed(ds[:, None] * gathered(k, src), dst)
        outs[2][:, i] = summed(ds[:, None] * gathered(q, dst), src)
        outs[3][:, i] = summed(p[:, None] * gathered(grad, dst), src)
    dtype = s["q"].dtype
    return [t.to(dtype) for t in outs]


def _plain_rows(s):
    case, rows = s["case"], s["rows"]
    q = _head_values(s["q"])
    first = s["indptr"][rows]
    length = s["indptr"][rows + 1] - first
    at = torch.repeat_interleave(torch.arange(rows.numel(), device=rows.device), length)
    slot = torch.arange(at.numel(), device=rows.device) - (torch.cumsum(length, 0) - length)[at] + first[at]
    u = s["src"][slot].long()
    k, v = (s[name][0][u].float() * s[name][1][u] for name in ("k8", "v8"))
    z = (q[at] * k).sum(-1) / math.sqrt(case["d"])
    p = torch.stack([_softmax(z[:, i], at, rows.numel()) for i in range(case["heads"])], 1)
    return torch.zeros_like(q).index_add_(0, at, p.unsqueeze(-1) * v).to(s["q"].dtype)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "checkpoint":
            return _values(s["x"], case["group"]).to(s["x"].dtype)
        if kind == "activation":
            x = s["x"]
            dx = s["grad"].float() * _df(_values(x, case["group"]), case["f"])
            return _f(x.float(), case["f"]).to(x.dtype), dx.to(x.dtype)
        return _plain_attention(s) if kind == "attention" else _plain_rows(s)
    import tango_b200 as T
    if kind == "checkpoint":
        return T.unpack8(T.pack8(s["x"], case["group"]))
    if kind == "activation":
        x = s["x"]
        x.grad = None
        y = T.activation8(x, case["f"], case["group"])
        y.backward(s["grad"])
        return y.detach(), x.grad
    if kind == "rows":
        return T.edge_attention_rows(s["graph"], s["rows"], s["q"], s["k8"], s["v8"])
    q, k, v = s["q"], s["k"], s["v"]
    if not case["train"]:
        with torch.no_grad():
            return [T.edge_attention(s["graph"], q, k, v)]
    q.grad = k.grad = v.grad = None
    out = T.edge_attention(s["graph"], q, k, v)
    out.backward(s["grad"])
    return [out.detach(), q.grad, k.grad, v.grad]


# ---------------------------------------------------------------------------------------------------- 64 bits
def _rounded(x, group):
    """The 8-bit form of a matrix in 64 bits, group by group; a scale is a 32-bit number."""
    x = x.double()
    out = torch.empty_like(x)
    for a in range(0, x.size(1), group):
        part = x[:, a:a + group]
        scale = (part.abs().max(1, keepdim=True).values / 127).float()
        scale[scale < 2.0 ** -126] = 0
        scale = scale.double()
        out[:, a:a + group] = torch.nan_to_num(torch.round(part / scale), nan=0.0, posinf=0.0, neginf=0.0) * scale
    return out


def _exact_attention(case, s, scale):
    """Head by head as products with the sparse matrices of the probabilities and of the score gradients."""
    n, h, d = case["nodes"], case["heads"], case["d"]
    order = torch.argsort(s["dst"].long() * n + s["src"].long())
    src, dst = s["src"][order].long(), s["dst"][order].long()
    q, k, v = (_rounded(s[name].flatten(1), d).view(-1, h, d) for name in "qkv")
    grad = _rounded(s["grad"].flatten(1), d).view(-1, h, d) if case["train"] else None
    indptr = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    indptr[1:] = torch.bincount(dst, minlength=n).cumsum(0)
    back = torch.argsort(src, stable=True)
    indptr_back = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    indptr_back[1:] = torch.bincount(src, minlength=n).cumsum(0)

    def dots(a, b):         # <a[dst], b[src]> of every edge
        out = torch.empty(src.numel(), device="cuda", dtype=torch.float64)
        for i in range(0, src.numel(), 1 << 24):
            at = slice(i, i + (1 << 24))
            out[at] = torch.linalg.vecdot(a[dst[at]], b[src[at]])
        return out

    def per_node(x):        # sums over the incoming edges
        return torch.sparse_csr_tensor(indptr, src, x, (n, n)) @ torch.ones(n, 1, dtype=torch.float64, device="cuda")

    outs = [[] for _ in range(4 if case["train"] else 1)]
    for i in range(h):
        z = dots(q[:, i].contiguous(), k[:, i].contiguous()) * scale
        top = torch.segment_reduce(z, "max", offsets=indptr, initial=-math.inf)
        p = torch.exp(z - top[dst])
        p /= per_node(p)[dst, 0]
        m = torch.sparse_csr_tensor(indptr, src, p, (n, n))
        outs[0].append(m @ v[:, i].contiguous())
        if case["train"]:
            dp = dots(grad[:, i].contiguous(), v[:, i].contiguous())
            ds = p * (dp - per_node(p * dp)[dst, 0]) * scale
            outs[1].append(torch.sparse_csr_tensor(indptr, src, ds, (n, n)) @ k[:, i].contiguous())
            outs[2].append(torch.sparse_csr_tensor(indptr_back, dst[back], ds[back], (n, n)) @ q[:, i].contiguous())
            outs[3].append(torch.sparse_csr_tensor(indptr_back, dst[back], p[back], (n, n)) @ grad[:, i].contiguous())
    return [torch.stack(t, 1) for t in outs]


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "checkpoint":
        return _rounded(s["x"], case["group"])
    if kind == "activation":
        x, f = s["x"].double(), case["f"]
        if f == "elu":
            y = torch.nn.functional.elu(x)
        elif f == "gelu":
            y = torch.nn.functional.gelu(x)
        else:
            y = torch.nn.functional.silu(x)
        t = _rounded(s["x"], case["group"])
        if f == "elu":
            slope = torch.where(t > 0, torch.ones_like(t), t.exp())
        elif f == "gelu":
            slope = 0.5 * torch.special.erfc(-t / math.sqrt(2)) + t * torch.exp(-t.square() / 2) / math.sqrt(2 * math.pi)
        else:
            slope = torch.sigmoid(t) + t * torch.sigmoid(t) * torch.sigmoid(-t)
        return y, s["grad"].double() * slope
    h, d = case["heads"], case["d"]
    if kind == "attention":
        return _exact_attention(case, s, 1 / math.sqrt(d))
    q, k, v = (_rounded(s[name].flatten(1), d).view(-1, h, d) for name in "qkv")
    out = torch.zeros_like(q)
    order = torch.argsort(s["dst"], stable=True)
    ends = torch.searchsorted(s["dst"][order].contiguous(), torch.stack([s["rows"], s["rows"] + 1]).to(torch.int32)).tolist()
    for r, (a, b) in enumerate(zip(*ends)):
        if a < b:
            u = s["src"][order[a:b]].long()
            p = torch.softmax(torch.einsum("hd,uhd->uh", q[r], k[u]) / math.sqrt(d), 0)
            out[r] = torch.einsum("uh,uhd->hd", p, v[u])
    return out


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    """Every input and output once; checkpoints are written once and read once; of a graph the indices that a pass walks."""
    size = 4 if case["type"] == "float32" else 2
    kind = case["kind"]
    if kind in ("checkpoint", "activation"):
        m, rows = case["rows"] * case["cols"], case["rows"]
        saved = 2 * (m + 4 * rows * -(-case["cols"] // case["group"]))
        return {"bytes": saved + (2 if kind == "checkpoint" else 4) * m * size, "flops": (6 if kind == "checkpoint" else 20) * m}
    n, e, h, d = case["nodes"], case["edges"], case["heads"], case["d"]
    f = h * d
    if kind == "rows":
        r = case["rows"]
        met = max(1, round(r * e / n))                           # edges that end in the nodes asked for, on average
        seen = min(met, n)
        return {"bytes": 2 * r * f * size + 16 * r + 4 * met + 2 * seen * (f + 4 * h), "flops": 4 * met * f}
    index = 4 * (e + n)
    if not case["train"]:
        return {"bytes": index + 4 * n * f * size, "flops": 4 * e * f}
    return {"bytes": 2 * index + 8 * n * f * size, "flops": 14 * e * f}
