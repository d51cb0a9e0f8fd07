"""The operators of the second model that a user puts behind a forest: the leaf of every (row, tree) picks
an embedding row, a row's embeddings are summed, linear layers follow, and a softmax over many classes ends it.

A case is one call:

  "leaf_sum"    h[n] = sum over trees t of table[row of the leaf that row n reached in tree t]
  "leaf_grad"   its gradient with respect to the table
  "linear"      y = activation(x W^T + b) + residual, and, for training, the value before the activation
  "linear_grad" gradients of x, W and b from the gradient of y and the kept value
  "loss"        loss[n] = log sum_v exp(z[n, v]) - z[n, label[n]], z = x W^T + b, and the logarithm itself;
                rows whose label lies outside the classes have loss 0
  "loss_grad"   gradients of x, W and b from the gradient of every row's loss

``run`` computes them from elementary operations in 32 bits where ``own`` is false, and calls this framework's
operators where it is true.  ``exact`` computes them in 64 bits.
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one row scored while its requester waits: the forest of 1000 trees of 8 levels, embeddings of 128
        dict(name="leaf_sum_one_row", op="leaf_sum", rows=1, trees=1000, levels=8, width=128, type="bf16"),
        # the batch whose leaf indices the forest's own cases compute, as the forward pass of training
        dict(name="leaf_sum_20k", op="leaf_sum", rows=20011, trees=1000, levels=8, width=64, type="bf16"),
        # a few trees, refitted on a small batch in full precision; an odd width
        dict(name="leaf_grad_1k", op="leaf_grad", rows=1024, trees=100, levels=6, width=50, type="fp32"),
        # the backward pass of the training batch above
        dict(name="leaf_grad_20k", op="leaf_grad", rows=20011, trees=1000, levels=8, width=64, type="bf16"),
        # one row through one residual layer: nothing but latency and the weights' bytes
        dict(name="linear_one_row", op="linear", rows=1, inputs=1024, outputs=1024, act="relu", bias=True,
             residual=True, keep=False, type="bf16"),
        # the widening layer of a large training batch, value before the activation kept
        dict(name="linear_32k", op="linear", rows=32768, inputs=1024, outputs=4096, act="gelu", bias=True,
             residual=False, keep=True, type="bf16"),
        # ragged sizes: no dimension is a multiple of anything
        dict(name="linear_grad_odd", op="linear_grad", rows=5003, inputs=777, outputs=333, act="silu", bias=True,
             type="fp16"),
        # the backward pass of a layer at training size
        dict(name="linear_grad_16k", op="linear_grad", rows=16384, inputs=1024, outputs=2048, act="gelu", bias=True,
             type="bf16"),
        # the 26 classes of the multiclass configuration
        dict(name="loss_26", op="loss", rows=20011, width=128, classes=26, bias=True, type="fp16"),
        # a catalogue of items as classes, odd count
        dict(name="loss_100k", op="loss", rows=4096, width=512, classes=100003, bias=True, type="bf16"),
        # a small batch over a middling catalogue
        dict(name="loss_grad_5k", op="loss_grad", rows=1000, width=96, classes=5003, bias=True, type="fp16"),
        # the backward pass of a large training batch
        dict(name="loss_grad_32k", op="loss_grad", rows=8192, width=1024, classes=32768, bias=False, type="bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["leaf_sum", "leaf_grad", "linear", "linear_grad", "loss", "loss_grad"])
    half = rng.choice(["bf16", "fp16"])
    while True:
        if op.startswith("leaf"):
            c = dict(op=op, rows=_spread(rng, 1, 32768), trees=_spread(rng, 10, 2600), levels=rng.randint(4, 9),
                     width=_spread(rng, 8, 256), type=rng.choice(["bf16", "fp16", "fp32"]))
            if c["rows"] * c["trees"] * c["width"] <= 20011 * 1000 * 64 and c["trees"] * c["width"] << c["levels"] <= 1 << 25:
                return c
        elif op.startswith("linear"):
            c = dict(op=op, rows=_spread(rng, 1, 32768), inputs=_spread(rng, 16, 4096), outputs=_spread(rng, 1, 4096),
                     act=rng.choice(["identity", "relu", "gelu", "silu"]), bias=rng.random() < 0.8, type=half)
            if op == "linear":
                c.update(residual=rng.random() < 0.5, keep=rng.random() < 0.5)
            if c["rows"] * c["inputs"] * c["outputs"] <= 1 << (37 if op == "linear" else 35):
                return c
        else:
            c = dict(op=op, rows=_spread(rng, 1, 16384), width=_spread(rng, 16, 2048), classes=_spread(rng, 2, 131072),
                     bias=rng.random() < 0.5, type=half)
            if c["rows"] * c["width"] * c["classes"] <= 1 << (37 if op == "loss" else 38) and c["rows"] * c["classes"] <= 1 << 29:
                return c


def _forest(trees, levels):
    """Complete trees of `levels` decision levels, nodes in level order, as flat forest arrays."""
    inner, nodes = (1 << levels) - 1, (2 << levels) - 1
    at = np.arange(nodes)
    left = np.where(at < inner, 2 * at + 1, -1).astype(np.int32)
    right = np.where(at < inner, 2 * at + 2, -1).astype(np.int32)
    return SimpleNamespace(num_trees=trees, tree_off=np.arange(trees + 1, dtype=np.int64) * nodes,
                           left=np.tile(left, trees), right=np.tile(right, trees),
                           feat=np.zeros(trees * nodes, np.int32), thr=np.zeros(trees * nodes, np.float32),
                           class_id=np.zeros(trees, np.int32), num_classes=0, transform=0, initial_value=0.0,
                           num_features=1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, to=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(to)

    s = SimpleNamespace(case=case, own=own)
    op, n = case["op"], case["rows"]
    if op.startswith("leaf"):
        trees, levels, width = case["trees"], case["levels"], case["width"]
        s.inner = (1 << levels) - 1
        s.table_rows = trees << levels
        # every split sends its own share of the rows to the right, as in a grown forest: leaves differ in use
        share = torch.rand(trees, s.inner, generator=g, device="cuda") * 0.8 + 0.1
        node = torch.zeros(n, trees, dtype=torch.int64, device="cuda")
        for _ in range(levels):
            p = torch.gather(share.t(), 0, node)
            node = 2 * node + 1 + (torch.rand(n, trees, generator=g, device="cuda") < p)
        s.ids = node.to(torch.int32)
        if op == "leaf_sum":
            s.table = normal(s.table_rows, width, scale=trees ** -0.5)
        else:
            s.grad = normal(n, width)
        if s.own:
            from treebeard_b200 import leaf_model
            s.leaves = leaf_model.LeafMap(_forest(trees, levels))
    elif op.startswith("linear"):
        s.x = normal(n, case["inputs"])
        s.weight = normal(case["outputs"], case["inputs"], scale=case["inputs"] ** -0.5)
        s.bias = normal(case["outputs"], scale=0.1) if case["bias"] else None
        if op == "linear":
            s.residual = normal(n, case["outputs"]) if case["residual"] else None
        else:
            s.grad = normal(n, case["outputs"])
            s.pre = normal(n, case["outputs"])
    else:
        s.x = normal(n, case["width"])
        s.weight = normal(case["classes"], case["width"], scale=1.5 * case["width"] ** -0.5)
        s.bias = normal(case["classes"], scale=0.5) if case["bias"] else None
        # frequent and rare classes; one row in twenty has no label
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        label = (float(case["classes"]) ** u - 1).to(torch.int64).clamp_(0, case["classes"] - 1)
        s.labels = torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, -1, label)
        if op == "loss_grad":
            # rows of different weight in the mean
            s.grad = (torch.rand(n, generator=g, device="cuda") + 0.5) / n
            lse = torch.empty(n, device="cuda")
            for a in range(0, n, 2048):
                lse[a:a + 2048] = torch.logsumexp(_logits(s.x[a:a + 2048], s.weight, s.bias), dim=1)
            s.lse = lse
    return s


def _logits(x, weight, bias, to=torch.float32):
    z = x.to(to) @ weight.to(to).t()
    return z if bias is None else z + bias.to(to)


def _act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _leaf_rows(s, a, b):
    """Table rows that the batch's rows a..b reached: leaves are numbered tree by tree in node order."""
    t = torch.arange(s.ids.shape[1], device="cuda") * (s.inner + 1)
    return s.ids[a:b].long() - s.inner + t


def _slab(s):
    return max(1, (1 << 27) // (s.ids.shape[1] * s.case["width"]))


def run(state):
    s, case = state, state.case
    op = case["op"]
    if s.own:
        from treebeard_b200 import leaf_model as lm
        if op == "leaf_sum":
            return lm.leaf_sum(s.leaves, s.ids, s.table)
        if op == "leaf_grad":
            return lm.leaf_sum_backward(s.leaves, s.ids, s.grad)
        if op == "linear":
            return lm.linear(s.x, s.weight, s.bias, activation=case["act"], residual=s.residual, keep_pre=case["keep"])
        if op == "linear_grad":
            return lm.linear_backward(s.grad, s.x, s.weight, pre=s.pre, activation=case["act"], bias=s.bias is not None)
        if op == "loss":
            return lm.class_loss(s.x, s.weight, s.labels, s.bias)
        return lm.class_loss_backward(s.grad, s.x, s.weight, s.labels, s.lse, s.bias)
    dtype = _TYPES[case["type"]]
    n = case["rows"]
    if op == "leaf_sum":
        step = _slab(s)
        return torch.cat([s.table[_leaf_rows(s, a, a + step)].float().sum(dim=1) for a in range(0, n, step)]).to(dtype)
    if op == "leaf_grad":
        out = torch.zeros(s.table_rows, case["width"], device="cuda")
        step = _slab(s)
        for a in range(0, n, step):
            rows = _leaf_rows(s, a, a + step)
            part = s.grad[a:a + step].float()
            out.index_add_(0, rows.reshape(-1), part[:, None, :].expand(-1, rows.shape[1], -1).reshape(-1, part.shape[1]))
        return out.to(dtype)
    if op == "linear":
        z = _logits(s.x, s.weight, s.bias)
        y = _act(z, case["act"])
        if s.residual is not None:
            y = y + s.residual.float()
        return (y.to(dtype), z.to(dtype)) if case["keep"] else y.to(dtype)
    if op == "linear_grad":
        dz = s.grad.float() * _slope(s.pre.float(), case["act"])
        return _pull_back(dz, s, dtype)
    z = _logits(s.x, s.weight, s.bias)
    live = (s.labels >= 0) & (s.labels < case["classes"])
    at = torch.where(live, s.labels, 0)[:, None]
    if op == "loss":
        top = z.max(dim=1, keepdim=True).values
        lse = torch.log(torch.exp(z - top).sum(dim=1)) + top[:, 0]
        return torch.where(live, lse - z.gather(1, at)[:, 0], 0.0), lse
    dz = torch.exp(z - s.lse[:, None])
    dz.scatter_add_(1, at, torch.full_like(at, -1, dtype=dz.dtype))
    dz *= torch.where(live, s.grad, 0.0)[:, None]
    return _pull_back(dz, s, dtype)


def _pull_back(dz, s, dtype):
    to = dz.dtype
    grads = [(dz @ s.weight.to(to)).to(dtype), (dz.t() @ s.x.to(to)).to(dtype)]
    return tuple(grads + ([dz.sum(dim=0).to(dtype)] if s.bias is not None else []))


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    op, n = case["op"], case["rows"]
    if op == "leaf_sum":
        out = torch.zeros(n, case["width"], dtype=f64, device="cuda")
        for t in range(case["trees"]):
            leaf = s.ids[:, t].long() - s.inner
            out += s.table[(t << case["levels"]):((t + 1) << case["levels"])].to(f64)[leaf]
        return out
    if op == "leaf_grad":
        out = torch.zeros(s.table_rows, case["width"], dtype=f64, device="cuda")
        grad = s.grad.to(f64)
        for t in range(case["trees"]):
            out.index_add_(0, (t << case["levels"]) + s.ids[:, t].long() - s.inner, grad)
        return out
    b = s.bias.to(f64) if s.bias is not None else 0.0
    x, w = s.x.to(f64), s.weight.to(f64)
    if op == "linear":
        z = torch.einsum("ni,oi->no", x, w) + b
        y = {"identity": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
             "silu": torch.nn.functional.silu}[case["act"]](z)
        y = y + s.residual.to(f64) if s.residual is not None else y
        return (y, z) if case["keep"] else y
    if op == "linear_grad":
        z = s.pre.to(f64).requires_grad_(True)
        y = {"identity": lambda v: v * 1, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
             "silu": torch.nn.functional.silu}[case["act"]](z)
        dz, = torch.autograd.grad(y, z, s.grad.to(f64))
        out = [torch.einsum("no,oi->ni", dz, w), torch.einsum("no,ni->oi", dz, x)]
        return tuple(out + ([dz.sum(dim=0)] if s.bias is not None else []))
    loss, lse = torch.empty(n, dtype=f64, device="cuda"), torch.empty(n, dtype=f64, device="cuda")
    dx, dw = torch.empty_like(x), torch.zeros_like(w)
    db = torch.zeros(case["classes"], dtype=f64, device="cuda")
    for a in range(0, n, 1024):  # rows by rows, so that the logits of the largest cases fit
        part, lab = x[a:a + 1024], s.labels[a:a + 1024]
        has = (lab >= 0) & (lab < case["classes"])
        z = torch.einsum("ni,vi->nv", part, w) + b
        rows = torch.arange(len(part), device="cuda")[has]
        if op == "loss":
            l = torch.logsumexp(z, dim=1)
            lse[a:a + 1024] = l
            loss[a:a + 1024] = 0.0
            loss[a:a + 1024][has] = l[has] - z[rows, lab[has]]
            continue
        # the probabilities are those that the given logarithm stands for
        p = torch.exp(z - s.lse[a:a + 1024].to(f64)[:, None])
        p[rows, lab[has]] -= 1.0
        p *= (s.grad[a:a + 1024].to(f64) * has)[:, None]
        dx[a:a + 1024] = torch.einsum("nv,vi->ni", p, w)
        dw += torch.einsum("nv,ni->vi", p, part)
        db += p.sum(dim=0)
    if op == "loss":
        return loss, lse
    return (dx, dw, db) if s.bias is not None else (dx, dw)


def work(case):
    e, n = _BYTES[case["type"]], case["rows"]
    op = case["op"]
    if op.startswith("leaf"):
        hits, width = n * case["trees"], case["width"]
        rows = case["trees"] << case["levels"]
        moved = min(hits, rows) if op == "leaf_sum" else rows
        return {"bytes": 4 * hits + e * width * (n + moved), "flops": hits * width}
    if op.startswith("linear"):
        i, o = case["inputs"], case["outputs"]
        if op == "linear":
            columns = o * (1 + case["residual"] + case["keep"])
            return {"bytes": e * (n * i + o * i + n * columns + o * case["bias"]), "flops": 2 * n * i * o}
        return {"bytes": e * (2 * n * i + 2 * o * i + 2 * n * o + o * case["bias"]), "flops": 4 * n * i * o}
    d, v = case["width"], case["classes"]
    if op == "loss":
        return {"bytes": e * (n * d + v * d + v * case["bias"]) + 16 * n, "flops": 2 * n * d * v}
    # the logits are not among the inputs: they have to be computed again
    return {"bytes": e * (2 * n * d + 2 * v * d + 2 * v * case["bias"]) + 16 * n, "flops": 6 * n * d * v}
