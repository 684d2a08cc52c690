"""The training-step operators as measured workloads: inputs, plain forms and exact values.

Three operators that stand around the relational layers in a training or serving step:

``layer_norm``      y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension,
                    forward alone (serving) or forward and backward (training)
``grouped_linear``  y[i] = x[i] @ weight[g] + bias[g] for the rows i of group g: consecutive row
                    ranges of ragged sizes, each with its own weight (node types, relations,
                    experts); forward alone or with the gradients of x, weight and bias
``clip``            the global 2-norm over a list of gradient tensors and the gradients scaled to
                    at most ``max_norm``

``own = False`` computes them with elementary torch operations in 32 bits, ``own = True`` with the
package's kernels. ``exact`` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5

# the costliest listed case of each operator; drawn cases stay below
_LN_MAX = 2_000_000 * 256         # elements
_GL_MAX = 3 * 2 * 32768 * 2048 * 4096  # flops
_CLIP_MAX = 1 << 28               # elements


def listed():
    return [
        # serving: the rows of a handful of requests, an odd width; latency is all there is
        dict(name="ln_serve", op="layer_norm", dtype="fp16", rows=7, width=771, pitch=771, train=False),
        # training: the node embeddings of a FB15K-237-sized graph between two relational layers
        dict(name="ln_nodes", op="layer_norm", dtype="fp32", rows=14541, width=128, pitch=128, train=True),
        # training: a batch of wide token embeddings in half-width types
        dict(name="ln_tokens", op="layer_norm", dtype="bf16", rows=16384, width=4096, pitch=4096, train=True),
        # training: every node of a two-million-node graph
        dict(name="ln_graph", op="layer_norm", dtype="fp32", rows=2_000_000, width=256, pitch=256, train=True),
        # serving: one token for each of two experts
        dict(name="gl_token", op="grouped_linear", dtype="bf16", rows=2, groups=8, k=1024, n=1024, skew="few",
             bias=False, train=False),
        # serving: a decode batch over many experts: bound by the weights of those that are hit
        dict(name="gl_decode", op="grouped_linear", dtype="bf16", rows=48, groups=64, k=2048, n=2048, skew="few",
             bias=False, train=False),
        # training: the (node, relation) segments of a FB15K-237-sized graph, a weight per relation
        dict(name="gl_relations", op="grouped_linear", dtype="fp32", rows=207_997, groups=237, k=128, n=128,
             skew="relations", bias=True, train=True),
        # training: a heterogeneous graph with few node types and odd feature widths
        dict(name="gl_types_odd", op="grouped_linear", dtype="fp16", rows=20011, groups=7, k=193, n=301,
             skew="routed", bias=True, train=True),
        # training: experts' products of a large token batch
        dict(name="gl_experts", op="grouped_linear", dtype="bf16", rows=32768, groups=32, k=2048, n=4096,
             skew="routed", bias=False, train=True),
        # the gradients of a small metapath model: every launch counts
        dict(name="clip_small", op="clip", dtype="fp32", tensors=10, elements=50_000),
        # the gradients of a three-layer relational network over 237 relations
        dict(name="clip_net", op="clip", dtype="fp32", tensors=8, elements=7_900_000),
        # the gradients of a model with many layers, matrices in bf16 and vectors in fp32
        dict(name="clip_many", op="clip", dtype="mixed", tensors=400, elements=1 << 28),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "grouped_linear", "grouped_linear", "clip"])
    if op == "layer_norm":
        width = _log_uniform(rng, 16, 8192)
        if rng.random() < 0.6:
            width = (width + 7) // 8 * 8
        rows = _log_uniform(rng, 1, max(1, min(2_000_000, _LN_MAX // (2 * width))))
        pitch = width if rng.random() < 0.7 else width + rng.choice([1, 8, 64])
        return dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=rows, width=width, pitch=pitch,
                    train=rng.random() < 0.7)
    if op == "grouped_linear":
        k, n = _log_uniform(rng, 32, 4096), _log_uniform(rng, 32, 4096)
        if rng.random() < 0.6:
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        groups = min(_log_uniform(rng, 1, 256), max(1, (1 << 28) // (k * n)))
        train = rng.random() < 0.6
        cap = _GL_MAX // 4 // ((3 if train else 1) * 2 * k * n)
        rows = _log_uniform(rng, 1, max(1, min(262_144, cap)))
        return dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=rows, groups=groups, k=k, n=n,
                    skew=rng.choice(["routed", "relations", "few"]), bias=rng.random() < 0.5, train=train)
    tensors = _log_uniform(rng, 1, 500)
    return dict(op="clip", dtype=rng.choice(["fp32", "bf16", "fp16", "mixed"]), tensors=tensors,
                elements=_log_uniform(rng, 1000 + tensors, _CLIP_MAX // 2))


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _apportion(total, weights):
    """total split into whole parts in proportion to the weights."""
    s = sum(weights)
    parts = [int(total * w / s) for w in weights]
    order = sorted(range(len(weights)), key=lambda i: (-weights[i], i))
    left = total - sum(parts)
    for j in range(left):
        parts[order[j % len(order)]] += 1
    return parts


def _group_sizes(case, seed):
    """Rows of each group: the sizes depend on the case, which group has which on the seed too."""
    rng = random.Random(f"{case['rows']}/{case['groups']}/{case['skew']}")
    g, rows = case["groups"], case["rows"]
    if case["skew"] == "relations":  # a few relations hold most of the segments
        sizes = _apportion(rows, [1.0 / (i + 1) ** 0.9 for i in range(g)])
    elif case["skew"] == "routed":   # a learned router: uneven, nobody starved for good
        sizes = _apportion(rows, [math.exp(rng.gauss(0.0, 0.5)) for _ in range(g)])
    else:                            # every row picks its group: many stay empty when rows are few
        sizes = [0] * g
        for _ in range(rows):
            sizes[rng.randrange(g)] += 1
    random.Random(seed).shuffle(sizes)
    return sizes


def _tensor_sizes(case):
    """Element counts of the gradient tensors: matrices and vectors mixed, odd lengths among them."""
    rng = random.Random(f"{case['tensors']}/{case['elements']}")
    n = case["tensors"]
    w = [math.exp(rng.gauss(0.0, 0.7)) * (1.0 if i % 2 == 0 else 1e-3) for i in range(n)]
    return [max(1, s) for s in _apportion(case["elements"], w)]


def _tensor_dtype(case, i):
    if case["dtype"] != "mixed":
        return _DTYPES[case["dtype"]]
    return torch.bfloat16 if i % 2 == 0 else torch.float32


def _buckets(tensors):
    """({dtype: flat zeroed buffer}, [each tensor's view in its type's buffer])."""
    ends, places = {}, []
    for t in tensors:
        places.append(ends.get(t.dtype, 0))
        ends[t.dtype] = places[-1] + (t.numel() + 63) // 64 * 64
    flat = {dt: torch.zeros(n, dtype=dt, device=tensors[0].device) for dt, n in ends.items()}
    return flat, [flat[t.dtype][p:p + t.numel()] for t, p in zip(tensors, places)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return torch.randn(*shape, device=dev, generator=gen, dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    state = {"case": case}
    if case["op"] == "layer_norm":
        dt = _DTYPES[case["dtype"]]
        rows, width = case["rows"], case["width"]
        # columns of a wider buffer (concatenated embeddings) where pitch > width
        state["x"] = randn(rows, case["pitch"], dtype=dt, scale=2.0, shift=0.5)[:, :width]
        state["weight"] = randn(width, dtype=dt, scale=0.2, shift=1.0)
        state["bias"] = randn(width, dtype=dt, scale=0.2)
        if case["train"]:
            state["dy"] = randn(rows, width, dtype=dt)
    elif case["op"] == "grouped_linear":
        dt = _DTYPES[case["dtype"]]
        rows, g, k, n = case["rows"], case["groups"], case["k"], case["n"]
        sizes = _group_sizes(case, seed)
        off = [0]
        for s in sizes:
            off.append(off[-1] + s)
        state["offsets"] = off
        state["group_ptr"] = torch.tensor(off, dtype=torch.int64, device=dev)
        state["x"] = randn(rows, k, dtype=dt)
        state["weight"] = randn(g, k, n, dtype=dt, scale=k ** -0.5)
        state["bias"] = randn(g, n, dtype=dt, scale=0.1) if case["bias"] else None
        if case["train"]:
            state["dy"] = randn(rows, n, dtype=dt)
    else:
        sizes = _tensor_sizes(case)
        state["grads"] = [randn(s, dtype=_tensor_dtype(case, i), scale=0.02) for i, s in enumerate(sizes)]
        # the clipped gradients land in one flat bucket per type, each tensor at a multiple of 64 elements
        state["flat"], state["out"] = _buckets(state["grads"])
        # a third of the expected norm: the step is clipped
        state["max_norm"] = 0.02 * math.sqrt(sum(sizes)) / 3.0
    if own and case["op"] != "clip" and case["train"]:
        for key in ("x", "weight", "bias"):
            if state.get(key) is not None:
                state[key] = state[key].detach().requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "grouped_linear": _own_grouped_linear, "clip": _own_clip}[op](state)
    return {"layer_norm": _plain_layer_norm, "grouped_linear": _plain_grouped_linear, "clip": _plain_clip}[op](state)


def _own_layer_norm(state):
    import mpgnn_amd
    y = mpgnn_amd.layer_norm(state["x"], state["weight"], state["bias"], _EPS)
    if not state["case"]["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["dy"])]


def _own_grouped_linear(state):
    import mpgnn_amd
    y = mpgnn_amd.grouped_linear(state["x"], state["weight"], state["group_ptr"], state["bias"])
    if not state["case"]["train"]:
        return [y]
    leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]


def _own_clip(state):
    import mpgnn_amd
    norm, _ = mpgnn_amd.clip_by_global_norm(state["grads"], state["max_norm"], out=state["out"])
    return [norm, *state["flat"].values()]


def _plain_layer_norm(state):
    dt = state["x"].dtype
    x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
    xc = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(dim=1, keepdim=True) + _EPS)
    xhat = xc * rstd
    y = (xhat * w + b).to(dt)
    if not state["case"]["train"]:
        return [y]
    dy = state["dy"].float()
    dw = (dy * xhat).sum(dim=0)
    db = dy.sum(dim=0)
    h = dy * w
    dx = (h - h.mean(dim=1, keepdim=True) - xhat * (h * xhat).mean(dim=1, keepdim=True)) * rstd
    return [y, dx.to(dt), dw.to(dt), db.to(dt)]


def _plain_grouped_linear(state):
    dt = state["x"].dtype
    x, w = state["x"].float(), state["weight"].float()
    b = None if state["bias"] is None else state["bias"].float()
    off, train = state["offsets"], state["case"]["train"]
    y = torch.empty(x.shape[0], w.shape[2], dtype=torch.float32, device=x.device)
    if train:
        dy = state["dy"].float()
        dx, dw = torch.empty_like(x), torch.zeros_like(w)
        db = None if b is None else torch.zeros_like(b)
    for g in range(w.shape[0]):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        yg = x[lo:hi] @ w[g]
        y[lo:hi] = yg if b is None else yg + b[g]
        if train:
            dx[lo:hi] = dy[lo:hi] @ w[g].t()
            dw[g] = x[lo:hi].t() @ dy[lo:hi]
            if b is not None:
                db[g] = dy[lo:hi].sum(dim=0)
    if not train:
        return [y.to(dt)]
    return [t.to(dt) for t in (y, dx, dw, db) if t is not None]


def _plain_clip(state):
    # squares summed in 64 bits: a long sum
    norm = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt().float()
    scale = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g, o in zip(state["grads"], state["out"]):
        o.copy_(g.float() * scale)
    return [norm, *state["flat"].values()]


# ---------------------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "layer_norm":
        e, b = case["rows"] * case["width"], _BYTES[case["dtype"]]
        if not case["train"]:
            return {"bytes": (2 * e + 2 * case["width"]) * b, "flops": 8 * e}
        # x, dy read; y, dx written; weight and bias read, their gradients written
        return {"bytes": (4 * e + 4 * case["width"]) * b, "flops": 22 * e}
    if case["op"] == "grouped_linear":
        m, k, n, b = case["rows"], case["k"], case["n"], _BYTES[case["dtype"]]
        sizes = _group_sizes(case, 0)
        hit = sum(1 for s in sizes if s)
        nb = n if case["bias"] else 0
        total = m * k + m * n + hit * (k * n + nb)  # x, y, the weights of the groups with rows
        if case["train"]:
            total += m * n + m * k + case["groups"] * (k * n + nb)  # dy, dx, dweight, dbias
        return {"bytes": total * b, "flops": 2 * m * k * n * (3 if case["train"] else 1)}
    total = 0
    for i, s in enumerate(_tensor_sizes(case)):
        total += 2 * s * torch.empty(0, dtype=_tensor_dtype(case, i)).element_size()
    return {"bytes": total + 4, "flops": 3 * case["elements"]}


def exact(case, seed):
    state = prepare(case, seed)
    for key in ("x", "weight", "bias", "dy"):
        if state.get(key) is not None:
            state[key] = state[key].detach().double()
    if case["op"] == "layer_norm":
        x, w, b = state["x"], state["weight"], state["bias"]
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        z = (x - mean) / (var + _EPS).sqrt()
        out = [torch.addcmul(b, z, w)]
        if case["train"]:
            dy = state["dy"]
            g = dy * w
            c1 = g.sum(1, keepdim=True) / case["width"]
            c2 = (g * z).sum(1, keepdim=True) / case["width"]
            out.append((g - c1 - z * c2) / (var + _EPS).sqrt())
            out.append((dy * z).sum(0))
            out.append(dy.sum(0))
        return out
    if case["op"] == "grouped_linear":
        x, w, b = state["x"], state["weight"], state["bias"]
        parts = [state["offsets"][g + 1] - state["offsets"][g] for g in range(case["groups"])]
        xs = x.split(parts)
        ys = [torch.mm(xg, w[g]) if b is None else torch.addmm(b[g], xg, w[g]) for g, xg in enumerate(xs)]
        out = [torch.cat(ys)]
        if case["train"]:
            ds = state["dy"].split(parts)
            out.append(torch.cat([torch.mm(dg, w[g].t()) for g, dg in enumerate(ds)]))
            out.append(torch.stack([torch.mm(xg.t(), dg) for xg, dg in zip(xs, ds)]))
            if b is not None:
                out.append(torch.stack([dg.sum(0) for dg in ds]))
        return out
    total = math.sqrt(math.fsum(float(torch.dot(t.double(), t.double())) for t in state["grads"]))
    factor = min(1.0, state["max_norm"] / (total + 1e-6))
    norm = torch.tensor(total, dtype=torch.float64, device=state["grads"][0].device)
    flat = {}
    for t in state["grads"]:
        flat.setdefault(t.dtype, []).append(torch.nn.functional.pad(t.double() * factor, (0, -t.numel() % 64)))
    return [norm] + [torch.cat(parts) for parts in flat.values()]
