"""The measured cases of the block norm, the 8-bit product and the products that keep their inputs in 8 bits.

Each case is one pass through one operator as a program calls it: the residual join with its norms (forward, or
forward and backward), the product of rows against 8-bit weights, and the layer's node-level products with their
inputs held in 8 bits between the forward and the backward.  ``own`` chooses between the plain form written here and
the library's operators; ``exact`` evaluates the same definitions in 64 bits.
"""
from __future__ import annotations

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TINY = 2.0 ** -100      # rows whose largest magnitude is below this count as zero
EPS = 1e-5


def listed():
    return [
        # --- block norm: joins a block's output to the residual stream and normalises the sum for the next block
        # one molecule of 18 atoms answered on its own: the launch is what counts
        {"name": "norm molecule bf16", "op": "norm", "n": 18, "h": 64, "dtype": "bf16", "kind": "rms", "post": True,
         "gate": "channel", "grad": False},
        # a training step's join on the full Flickr graph, hidden width 64, a gate per node and channel
        {"name": "norm flickr f32 step", "op": "norm", "n": 89250, "h": 64, "dtype": "f32", "kind": "layer", "post": False,
         "gate": "full", "grad": True},
        # the raw feature width of that graph (500) on an odd number of nodes, norms on both sides, a gate per node
        {"name": "norm 500 wide f32 step", "op": "norm", "n": 30011, "h": 500, "dtype": "f32", "kind": "layer", "post": True,
         "gate": "row", "grad": True},
        # the power-law graph with 4 M nodes and hidden width 128: all memory traffic
        {"name": "norm 4M bf16 step", "op": "norm", "n": 4000000, "h": 128, "dtype": "bf16", "kind": "rms", "post": True,
         "gate": "channel", "grad": True},
        # --- rows against 8-bit weights: the forward of a trained model that answers
        # one molecule, 11 atom features to the fused projection of a 64-wide layer
        {"name": "int8 molecule f32", "op": "int8", "n": 18, "k": 11, "m": 128, "dtype": "f32", "rows8": False, "relu": False},
        # Flickr's features to a projection and an update's share (3 x 64 columns) in one product
        {"name": "int8 flickr f32", "op": "int8", "n": 89250, "k": 500, "m": 192, "dtype": "f32", "rows8": False, "relu": False},
        # the fused projection on 4 M nodes
        {"name": "int8 4M bf16", "op": "int8", "n": 4000000, "k": 128, "m": 256, "dtype": "bf16", "rows8": False, "relu": True},
        # wide layers, rows that are held in 8 bits already: the matrix cores are what counts
        {"name": "int8 wide rows8", "op": "int8", "n": 65536, "k": 1024, "m": 2048, "dtype": "bf16", "rows8": True, "relu": False},
        # --- products that keep their inputs in 8 bits for the backward: a whole training step of the product
        # a batch of 1024 molecules, first layer
        {"name": "kept molecules f32 step", "op": "project", "n": 18432, "k": 11, "m": 128, "dtype": "f32"},
        # the update relu([x | aggr] W^T) on the point clouds' 32 x 1024 nodes, hidden width 64
        {"name": "kept update clouds bf16 step", "op": "update", "n": 32768, "k": 64, "m": 64, "dtype": "bf16"},
        # the fused projection of the 4 M-node graph in float32
        {"name": "kept project 4M f32 step", "op": "project", "n": 4000000, "k": 128, "m": 256, "dtype": "f32"},
        # the update on the same graph in bfloat16
        {"name": "kept update 4M bf16 step", "op": "update", "n": 4000000, "k": 128, "m": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "int8", "project", "update"])
    dtype = rng.choice(["f32", "bf16"])
    size = 2 if dtype == "bf16" else 4
    if op == "norm":
        h = _log(rng, 3, 2048)
        if rng.random() < 0.5:
            h = max(8, h // 8 * 8)
        n = min(_log(rng, 1, 4000000), 4000000 * 128 * 2 // (h * size))
        return {"op": op, "n": n, "h": h, "dtype": dtype, "kind": rng.choice(["rms", "layer"]), "post": rng.random() < 0.5,
                "gate": rng.choice(["none", "channel", "row", "full"]), "grad": rng.random() < 0.7}
    k, m = _log(rng, 3, 2048 if op == "int8" else 512), _log(rng, 8, 2048 if op == "int8" else 512)
    if op == "int8":
        if rng.random() < 0.5:
            k, m = max(8, k // 8 * 8), m // 8 * 8
        n = _log(rng, 1, 4000000)
        n = max(1, min(n, 4000000 * 384 // (k + m), 65536 * 1024 * 2048 // (k * m)))
        return {"op": op, "n": n, "k": k, "m": m, "dtype": dtype, "rows8": rng.random() < 0.3, "relu": rng.random() < 0.5}
    if op == "update":
        dtype, size = "bf16", 2         # a float32 relu that is zero to rounding has no one right gradient to compare
    if dtype == "bf16":
        k, m = max(8, k // 8 * 8), m // 8 * 8      # the products' own rule for bfloat16 rows
    n = _log(rng, 1, 4000000)
    n = max(1, min(n, 4000000 * 384 * 2 // ((2 * k + m if op == "update" else k + m) * size), 4000000 * 128 * 128 // (k * m)))
    return {"op": op, "n": n, "k": k, "m": m, "dtype": dtype}


def _quantized(x):
    """Rows in 8 bits: scale = max|x| / 127, value = x * (127 / max|x|) to the nearest whole number, ties to even.
    64 bits for the products, so that values next to a border fall to their own side."""
    top = x.float().abs().amax(dim=1, keepdim=True)
    zero = top < TINY
    inv = torch.where(zero, 0.0, (127.0 / top.double()).float())
    scale = torch.where(zero, 0.0, (top.double() / 127.0).float())
    return torch.round(x.double() * inv.double()).float(), scale


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(scale).to(dtype)

    n = case["n"]
    s = {"case": case}
    if case["op"] == "norm":
        h = case["h"]
        need = case["grad"]
        s["block"] = randn(n, h, scale=0.7).requires_grad_(need)
        s["residual"] = randn(n, h, scale=2.0).requires_grad_(need)
        shape = {"channel": (h,), "row": (n, 1), "full": (n, h)}.get(case["gate"])
        s["gate"] = torch.sigmoid(randn(*shape, dtype=torch.float32)).to(dt).requires_grad_(need) if shape else None
        s["weight"] = (1.0 + randn(h, dtype=torch.float32, scale=0.2)).to(dt).requires_grad_(need)
        s["bias"] = randn(h, scale=0.2).requires_grad_(need) if case["kind"] == "layer" else None
        s["post_weight"] = (1.0 + randn(h, dtype=torch.float32, scale=0.2)).to(dt).requires_grad_(need) if case["post"] else None
        if need:
            s["g_stream"], s["g_normed"] = randn(n, h), randn(n, h)
        return s
    k, m = case["k"], case["m"]
    if case["op"] == "int8":
        x = randn(n, k)
        w = randn(m, k, dtype=torch.float32, scale=k ** -0.5)
        q, scale = _quantized(w)
        pitch = -(-k // 16) * 16
        s["w_values"] = torch.zeros(m, pitch, dtype=torch.int8, device=dev)
        s["w_values"][:, :k] = q.to(torch.int8)
        s["w_scale"] = scale.view(-1)
        s["bias"] = randn(m, scale=0.1)
        if case["rows8"]:
            q, scale = _quantized(x)
            s["x_values"] = torch.zeros(n, pitch, dtype=torch.int8, device=dev)
            s["x_values"][:, :k] = q.to(torch.int8)
            s["x_scale"] = scale.view(-1)
        else:
            s["x"] = x
        return s
    # a layer's inputs are the relu outputs of the layer before it: no negative values, half of them zeros
    x = randn(n, k).relu_().requires_grad_(True)
    s["x"] = x
    cols = k
    if case["op"] == "update":
        s["aggr"] = randn(n, m, scale=2.0).relu_().requires_grad_(True)
        cols = k + m
    s["w"] = randn(m, cols, scale=cols ** -0.5).requires_grad_(True)
    s["gy"] = randn(n, m)
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _norm(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(dim=1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS)
    if weight is not None:
        y = y * weight.float()
    return y if bias is None else y + bias.float()


def _plain_norm(s):
    case = s["case"]
    dt = s["block"].dtype
    branch = s["block"].float()
    if case["post"]:
        branch = _norm(branch, case["kind"], s["post_weight"], None)
    if s["gate"] is not None:
        branch = branch * s["gate"].float()
    stream = s["residual"].float() + branch
    normed = _norm(stream, case["kind"], s["weight"], s["bias"])
    return stream.to(dt), normed.to(dt)


def _plain_int8(s):
    case = s["case"]
    if case["rows8"]:
        q, scale = s["x_values"][:, :case["k"]].float(), s["x_scale"].view(-1, 1)
    else:
        q, scale = _quantized(s["x"])
    y = (q @ s["w_values"][:, :case["k"]].float().t()) * scale * s["w_scale"] + s["bias"].float()
    if case["relu"]:
        y = torch.relu(y)
    return y.to(DTYPES[case["dtype"]])


def _over_rows(g, x):
    """g^T x in pieces of 4096 rows that are added at the end: one float32 sum over millions of rows loses digits."""
    n, m, k = g.size(0), g.size(1), x.size(1)
    whole = n // 4096 * 4096
    pieces = torch.bmm(g[:whole].view(-1, 4096, m).transpose(1, 2), x[:whole].view(-1, 4096, k))
    return pieces.sum(dim=0) + g[whole:].t() @ x[whole:]


def _plain_kept(s):
    x, w, gy = s["x"].detach(), s["w"].detach().float(), s["gy"].float()
    dt = x.dtype
    k = x.size(1)
    q, scale = _quantized(x)
    z = x.float() @ w[:, :k].t()
    if s["case"]["op"] == "project":
        return z.to(dt), (gy @ w).to(dt), _over_rows(gy, q * scale).to(dt)
    aggr = s["aggr"].detach()
    z = z + aggr.float() @ w[:, k:].t()
    qa, scale_a = _quantized(aggr)
    gz = gy * (z > 0)
    gw = torch.cat([_over_rows(gz, q * scale), _over_rows(gz, qa * scale_a)], dim=1)
    return torch.relu(z).to(dt), (gz @ w[:, :k]).to(dt), (gz @ w[:, k:]).to(dt), gw.to(dt)


# ---------------------------------------------------------------------------------------- the library's operators
def _own_norm(s):
    from mpnn_amd import block_norm
    case = s["case"]
    return block_norm(s["block"], s["residual"], norm=case["kind"], eps=EPS, post_norm=case["post"],
                      post_weight=s["post_weight"], gate=s["gate"], weight=s["weight"], bias=s["bias"])


def _own_int8(s):
    from mpnn_amd import Rows8, linear_int8
    case = s["case"]
    k = case["k"]
    w = Rows8(s["w_values"][:, :k], s["w_scale"])
    x = Rows8(s["x_values"][:, :k], s["x_scale"]) if case["rows8"] else s["x"]
    return linear_int8(x, w, bias=s["bias"], relu=case["relu"], dtype=DTYPES[case["dtype"]])


def _own_kept(s):
    from mpnn_amd.dense import project, update
    if s["case"]["op"] == "project":
        y = project(s["x"], s["w"], checkpoint="int8")
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["gy"]))
    y = update(s["x"], s["aggr"], s["w"], checkpoint="int8")
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["aggr"], s["w"]), s["gy"]))


def run(state):
    op = state["case"]["op"]
    if op == "norm":
        stream, normed = (_own_norm if own else _plain_norm)(state)
        out = {"stream": stream.detach(), "normed": normed.detach()}
        if state["case"]["grad"]:
            names = [k for k in ("block", "residual", "gate", "weight", "bias", "post_weight") if state[k] is not None]
            grads = torch.autograd.grad((stream, normed), [state[k] for k in names], (state["g_stream"], state["g_normed"]))
            out.update({"g_" + k: g for k, g in zip(names, grads)})
        return out
    if op == "int8":
        return (_own_int8 if own else _plain_int8)(state)
    names = ("y", "gx", "gw") if op == "project" else ("y", "gx", "gaggr", "gw")
    return dict(zip(names, (_own_kept if own else _plain_kept)(state)))


def work(case):
    n = case["n"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        h = case["h"]
        gate = {"none": 0, "channel": h, "row": n, "full": n * h}[case["gate"]]
        vectors = h * (1 + (case["kind"] == "layer") + bool(case["post"]))
        b = 4 * n * h + gate + vectors                     # block, residual in; stream, normed out
        f = n * h * (8 + 8 * bool(case["post"]))
        if case["grad"]:                                   # the backward reads both inputs again and the two gradients
            b += 6 * n * h + 2 * gate + 2 * vectors
            f += n * h * (16 + 14 * bool(case["post"]))
        return {"bytes": b * size, "flops": f}
    k, m = case["k"], case["m"]
    if case["op"] == "int8":
        rows = n * (k + 4) if case["rows8"] else n * k * size
        return {"bytes": rows + m * (k + 4) + m * size + n * m * size, "flops": 2 * n * m * k}
    cols = k + m if case["op"] == "update" else k
    # forward: the inputs, the output, the kept rows; backward: the upstream gradient, the kept rows, the gradients
    b = size * (2 * n * cols + 2 * n * m + 3 * m * cols) + 2 * n * cols
    if case["op"] == "update":
        b += n * m // 4                                    # one bit of the relu per entry, written and read
    return {"bytes": b, "flops": 6 * n * m * cols}


# ------------------------------------------------------------------------------------------------------ 64 bits
def _rows_to_8(x):
    """The values that rows held in 8 bits stand for: (whole numbers, scales), both as float64."""
    big = x.double().abs().max(dim=1).values
    keep = big >= TINY
    safe = torch.where(keep, big, torch.ones_like(big))
    inverse = torch.where(keep, (127.0 / safe).float().double(), torch.zeros_like(big))
    step = torch.where(keep, (safe / 127.0).float().double(), torch.zeros_like(big))
    return (x.double() * inverse[:, None]).round(), step


def _norm64(v, kind):
    """(normalised rows, 1 / deviation)"""
    if kind == "layer":
        v = v - v.sum(1, keepdim=True) / v.size(1)
    inv = ((v ** 2).sum(1, keepdim=True) / v.size(1) + EPS) ** -0.5
    return v * inv, inv


def _norm64_back(g, hat, inv, kind):
    h = g.size(1)
    out = g - hat * ((g * hat).sum(1, keepdim=True) / h)
    if kind == "layer":
        out = out - g.sum(1, keepdim=True) / h
    return out * inv


def _exact_norm(case, s):
    kind = case["kind"]
    d = {k: (v.detach().double() if torch.is_tensor(v) else v) for k, v in s.items()}
    branch, inner_inv = d["block"], None
    if case["post"]:
        inner_hat, inner_inv = _norm64(branch, kind)
        branch = inner_hat * d["post_weight"]
    gate = 1.0 if d["gate"] is None else d["gate"]
    stream = d["residual"] + gate * branch
    hat, inv = _norm64(stream, kind)
    normed = hat * d["weight"]
    if d["bias"] is not None:
        normed = normed + d["bias"]
    out = {"stream": stream, "normed": normed}
    if not case["grad"]:
        return out
    gn = d["g_normed"]
    out["g_weight"] = (gn * hat).sum(0)
    if d["bias"] is not None:
        out["g_bias"] = gn.sum(0)
    g = d["g_stream"] + _norm64_back(gn * d["weight"], hat, inv, kind)
    out["g_residual"] = g
    if case["gate"] == "full":
        out["g_gate"] = g * branch
    elif case["gate"] == "row":
        out["g_gate"] = (g * branch).sum(1, keepdim=True)
    elif case["gate"] == "channel":
        out["g_gate"] = (g * branch).sum(0)
    g = g * gate
    if case["post"]:
        out["g_post_weight"] = (g * inner_hat).sum(0)
        g = _norm64_back(g * d["post_weight"], inner_hat, inner_inv, kind)
    out["g_block"] = g
    return out


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "norm":
            return _exact_norm(case, s)
        k = case["k"]
        if case["op"] == "int8":
            w = s["w_values"][:, :k].double() * s["w_scale"].double()[:, None]
            if case["rows8"]:
                q, step = s["x_values"][:, :k].double(), s["x_scale"].double()
            else:
                q, step = _rows_to_8(s["x"])
            y = torch.addmm(s["bias"].double(), q * step[:, None], w.t())
            return y.clamp_min_(0.0) if case["relu"] else y
        w, gy = s["w"].double(), s["gy"].double()
        q, step = _rows_to_8(s["x"])
        y = torch.mm(s["x"].double(), w[:, :k].t())
        if case["op"] == "project":
            return {"y": y, "gx": torch.mm(gy, w), "gw": torch.mm(gy.t(), q * step[:, None])}
        y += torch.mm(s["aggr"].double(), w[:, k:].t())
        gy = torch.where(y > 0, gy, torch.zeros_like(gy))
        parts = [torch.mm(gy.t(), q * step[:, None])]
        q, step = _rows_to_8(s["aggr"])
        parts.append(torch.mm(gy.t(), q * step[:, None]))
        return {"y": y.clamp_min_(0.0), "gx": torch.mm(gy, w[:, :k]), "gaggr": torch.mm(gy, w[:, k:]),
                "gw": torch.cat(parts, dim=1)}
