"""Operators of a transformer's feed-forward half with block-sparse weights, as cases that can be timed: the layer norm in front,
the linear layers with bias, activation and residual in the product's epilogue, and the layers of experts whose tokens come in runs
of ragged length.  Each serves (forward) and trains (forward and gradients).  ``own`` false: the plain form, elementary torch
operations in 32 bits on the dense weight.  ``own`` true: the calls a user makes of this framework.

A case is a dict of plain values; ``op`` and ``train`` say which path it takes:
  norm     y = (x - mean) / sqrt(var + eps) * w + b over the features of each token
                                                         void_layer_norm
  linear   y = act(x A^T + b) + r, A block-sparse          void_linear, SparseLinear
  int8     the same with quantised weight and activations  void_linear
  experts  y_t = act(x_t A_e^T + b_e), tokens sorted by expert, A_e block-sparse
                                                         void_expert_linear, SparseExperts
"""
import math

import torch

own = False

TILE = 32
EPS = 1e-5
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACT_CODES = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
GELU_SCALE, GELU_CUBIC = 1.5957691216, 0.044715   # the framework's GELU: x * sigmoid(1.5957691216 (x + 0.044715 x^3))
MOST_DENSE = 3.0e8       # elements of all dense weights of a drawn case


def listed():
    return [
        # decode: the norm in front of a layer for a handful of sequences, one launch's latency
        {"name": "norm_decode", "op": "norm", "train": False, "n": 8, "k": 2048, "dtype": "bf16", "params": "same"},
        # a prompt of two thousand tokens at the width of the two-layer workload
        {"name": "norm_prompt", "op": "norm", "train": False, "n": 2048, "k": 4096, "dtype": "bf16", "params": "same"},
        # training, sizes that are multiples of nothing, fp32 throughout
        {"name": "norm_train_ragged", "op": "norm", "train": True, "n": 3001, "k": 5003, "dtype": "fp32", "params": "same"},
        # training, a batch of sixteen thousand tokens, master weights in fp32
        {"name": "norm_train", "op": "norm", "train": True, "n": 16384, "k": 4096, "dtype": "bf16", "params": "fp32"},
        # decode: the down projection of a feed-forward layer, residual added on the way out
        {"name": "linear_decode", "op": "linear", "train": False, "n": 8, "k": 8192, "m": 2048, "sparsity": 0.8, "dtype": "fp16",
         "act": "none", "residual": True},
        # prompt processing: the down projection for two thousand tokens
        {"name": "linear_prompt", "op": "linear", "train": False, "n": 2048, "k": 16384, "m": 4096, "sparsity": 0.9, "dtype": "bf16",
         "act": "none", "residual": True},
        # the quantised down projection of a served model, bf16 residual stream
        {"name": "int8_prompt", "op": "int8", "train": False, "n": 1024, "k": 8192, "m": 4096, "sparsity": 0.8, "dtype": "bf16",
         "act": "none", "residual": True},
        # a training step of a layer with sizes that are multiples of nothing, GELU
        {"name": "linear_train_ragged", "op": "linear", "train": True, "n": 333, "k": 5003, "m": 3001, "sparsity": 0.85,
         "dtype": "bf16", "act": "gelu", "residual": True},
        # a training step of four thousand tokens through a layer of the published size
        {"name": "linear_train", "op": "linear", "train": True, "n": 4096, "k": 4096, "m": 4096, "sparsity": 0.9, "dtype": "bf16",
         "act": "gelu", "residual": True},
        # decode: sixteen tokens sent to two experts each, most experts with a few of them
        {"name": "experts_decode", "op": "experts", "train": False, "n": 32, "k": 2048, "m": 8192, "experts": 8, "skew": 1.0,
         "spare": 0, "sparsity": 0.8, "dtype": "fp16", "act": "silu"},
        # prompt processing: eight thousand routed tokens, a few popular experts, a buffer longer than what is routed
        {"name": "experts_prompt", "op": "experts", "train": False, "n": 8192, "k": 2048, "m": 8192, "experts": 8, "skew": 0.7,
         "spare": 511, "sparsity": 0.8, "dtype": "bf16", "act": "silu"},
        # a training step of sixteen experts
        {"name": "experts_train", "op": "experts", "train": True, "n": 8192, "k": 2048, "m": 4096, "experts": 16, "skew": 0.5,
         "spare": 0, "sparsity": 0.9, "dtype": "bf16", "act": "gelu"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _side(rng, lo, hi):
    """A width over the whole range: a multiple of 128, a multiple of the tile, or any number."""
    v = _log_int(rng, lo, hi)
    unit = rng.choice((128, 32, 1))
    return max(lo, v // unit * unit)


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(("norm", "norm", "linear", "linear", "linear", "int8", "experts", "experts", "experts"))
        train = op != "int8" and rng.random() < 0.5
        dtype = rng.choice(("fp16", "bf16"))
        sparsity = round(rng.uniform(0.5, 0.98), 3)
        act = rng.choice(("none", "relu", "gelu", "silu"))
        if op == "norm":
            dtype = rng.choice(("fp32", "fp16", "bf16"))
            c = {"op": op, "train": train, "n": _log_int(rng, 1, 16384), "k": _side(rng, 128, 16384), "dtype": dtype,
                 "params": rng.choice(("same", "fp32"))}
        elif op in ("linear", "int8"):
            c = {"op": op, "train": train, "n": _log_int(rng, 16 if train else 1, 4096), "k": _side(rng, 256, 16384),
                 "m": _side(rng, 256, 16384), "sparsity": sparsity, "dtype": dtype, "act": act, "residual": rng.random() < 0.8}
        else:
            n = _log_int(rng, 16 if train else 1, 8192)
            c = {"op": op, "train": train, "n": n, "k": _side(rng, 256, 8192), "m": _side(rng, 256, 8192),
                 "experts": _log_int(rng, 2, 64), "skew": round(rng.uniform(0.0, 1.5), 2),
                 "spare": rng.choice((0, rng.randint(0, n // 2))), "sparsity": sparsity, "dtype": dtype, "act": act}
            if c["experts"] * c["k"] * c["m"] > MOST_DENSE:
                continue
        w = work(c)
        if w["flops"] <= max(x["flops"] for x in most) and w["bytes"] <= max(x["bytes"] for x in most):
            return c


# ------------------------------------------------------------------------------------------ inputs
def _grid(case):
    return (case["m"] + TILE - 1) // TILE, (case["k"] + TILE - 1) // TILE


def _stored(case):
    """Stored tiles of a weight (of each expert's)."""
    nbr, nbc = _grid(case)
    return max(1, round((1.0 - case["sparsity"]) * nbr * nbc))


def _counts(case):
    """Tokens per expert, the most popular first: shares that fall as rank^-skew, rounded to whole tokens."""
    used, experts = case["n"] - case["spare"], case["experts"]
    shares = [(e + 1.0) ** -case["skew"] for e in range(experts)]
    exact = [used * s / sum(shares) for s in shares]
    counts = [int(x) for x in exact]
    by_rest = sorted(range(experts), key=lambda e: counts[e] - exact[e])
    for e in by_rest[:used - sum(counts)]:
        counts[e] += 1
    return counts


def _spread(v):
    """The bits of 16-bit numbers on even positions."""
    for shift, mask in ((8, 0x00FF00FF), (4, 0x0F0F0F0F), (2, 0x33333333), (1, 0x55555555)):
        v = (v | (v << shift)) & mask
    return v


def _tile_list(gen, case):
    """Stored tiles at random places, in Morton order: block rows, block columns and Morton codes."""
    nbr, nbc = _grid(case)
    at = torch.rand(nbr * nbc, generator=gen, device="cuda").argsort()[:_stored(case)]
    rows, cols = at // nbc, at % nbc
    codes, order = (_spread(rows) | (_spread(cols) << 1)).sort()
    return rows[order].int(), cols[order].int(), codes


def _edges_zero(values, rows, cols, case):
    """Tiles hold zeros outside the matrix, like every converted one."""
    m, k = case["m"], case["k"]
    if m % TILE:
        values[rows == m // TILE, m % TILE:, :] = 0
    if k % TILE:
        values[cols == k // TILE, :, k % TILE:] = 0
    return values


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, n, k = case["op"], case["n"], case["k"]
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dtype, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    s = {"case": dict(case)}
    if op == "norm":
        params = torch.float32 if case["params"] == "fp32" else dtype
        # a residual stream: features of different sizes and an offset
        s["x"] = (torch.randn(n, k, generator=gen, device="cuda") * torch.rand(k, generator=gen, device="cuda").add(0.25) + 0.5).to(dtype)
        s["w"], s["b"] = randn(k, dtype=params, scale=0.2, shift=1.0), randn(k, dtype=params, scale=0.2)
        if case["train"]:
            s["g"] = randn(n, k)
        return s
    m, experts = case["m"], case.get("experts", 1)
    lists = [_tile_list(gen, case) for _ in range(experts)]
    s["rows"], s["cols"], s["codes"] = [x[0] for x in lists], [x[1] for x in lists], [x[2] for x in lists]
    stored = _stored(case)
    if op == "int8":
        values = torch.randint(-128, 128, (stored, TILE, TILE), generator=gen, device="cuda", dtype=torch.int8)
        s["values"] = [_edges_zero(values, s["rows"][0], s["cols"][0], case)]
        s["scales"] = torch.rand(stored, generator=gen, device="cuda").add(0.5) * 0.0135 * ((1.0 - case["sparsity"]) * k) ** -0.5
        s["x"] = torch.randint(-128, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
        s["x_scale"] = torch.rand(n, generator=gen, device="cuda").add(0.5) * 0.0135
    else:
        scale = ((1.0 - case["sparsity"]) * k) ** -0.5
        s["values"] = [_edges_zero(randn(stored, TILE, TILE, scale=scale), s["rows"][e], s["cols"][e], case) for e in range(experts)]
        s["x"] = randn(n, k)
    bias_type = dtype if case["train"] else torch.float32
    if op == "experts":
        s["bias"] = randn(experts, m, dtype=bias_type, scale=0.2)
        counts = _counts(case)
        order = torch.randperm(experts, generator=torch.Generator().manual_seed(int(seed))).tolist()
        s["counts"] = [counts[e] for e in order]
        s["offsets"] = torch.tensor([0] + s["counts"], dtype=torch.int64).cumsum(0).int().cuda()
    else:
        s["bias"] = randn(m, dtype=bias_type, scale=0.2)
        if case["residual"]:
            s["r"] = randn(n, m)
    if case["train"]:
        s["g"] = randn(n, m)
    return s


def _handles(s):
    """What a user's program keeps of this framework: the weight, or the layer around it."""
    import void_b200 as void
    case = s["case"]
    for name in ("x", "w", "b", "r"):
        if case["train"] and name in s:
            s[name].requires_grad_(True)
    if case["op"] == "norm":
        return
    k, m, stored = case["k"], case["m"], _stored(case)
    nbr, nbc = _grid(case)
    if case["op"] == "int8":
        s["a"] = void.Int8VOIDTensor(s["values"][0], s["scales"], torch.zeros(stored, dtype=torch.int8, device="cuda"), s["rows"][0],
                                     s["cols"][0], (m, k), (TILE, TILE), stored, void.IntQuantConfig())
        return
    a = [void.VOIDTensor(values=v, block_rows=r, block_cols=c, morton_codes=z, shape=(m, k), tile_size=(TILE, TILE),
                         nnz_original=v.numel(), n_blocks=stored, density=stored / (nbr * nbc), dtype=v.dtype)
         for v, r, c, z in zip(s["values"], s["rows"], s["cols"], s["codes"])]
    s["a"] = void.stack_experts(a) if case["op"] == "experts" else a[0]
    if case["train"]:
        if case["op"] == "experts":
            s["layer"] = void.SparseExperts(s["a"], bias=True, activation=case["act"])
        else:
            s["layer"] = void.SparseLinear(k, m, s["a"], bias=True, activation=case["act"])
        with torch.no_grad():
            s["layer"].bias.copy_(s["bias"])


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handles(s)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import void_b200 as void
    case = s["case"]
    op, x = case["op"], s["x"]
    if op == "norm":
        y = void.void_layer_norm(x, s["w"], s["b"], EPS)
        if not case["train"]:
            return y
        dx, dw, db = torch.autograd.grad(y, (x, s["w"], s["b"]), s["g"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    act = ACT_CODES[case["act"]]
    if not case["train"]:
        if op == "experts":
            return void.void_expert_linear(s["a"], x, s["offsets"], s["bias"], act)
        if op == "int8":
            return void.void_linear(s["a"], x, s["bias"], act, x_scale=s["x_scale"], out_dtype=DTYPES[case["dtype"]], residual=s.get("r"))
        return void.void_linear(s["a"], x, s["bias"], act, residual=s.get("r"))
    layer = s["layer"]
    if op == "experts":
        y = layer(x, s["offsets"])
        grads = torch.autograd.grad(y, (x, layer.values, layer.bias), s["g"])
    else:
        y = layer(x, residual=s.get("r"))
        leaves = (x, layer.sparse_weight.values, layer.bias) + ((s["r"],) if case["residual"] else ())
        grads = torch.autograd.grad(y, leaves, s["g"])
    return {"y": y.detach(), "grads": list(grads)}


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return z * torch.sigmoid(GELU_SCALE * (z + GELU_CUBIC * z * z * z))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "none":
        return torch.ones_like(z)
    if act == "gelu":
        u, du = GELU_SCALE * (z + GELU_CUBIC * z * z * z), GELU_SCALE * (1.0 + 3.0 * GELU_CUBIC * z * z)
    else:
        u, du = z, 1.0
    p = torch.sigmoid(u)
    return p + z * p * (1.0 - p) * du


def _dense(values, rows, cols, case):
    nbr, nbc = _grid(case)
    w = torch.zeros(nbr, nbc, TILE, TILE, device="cuda")
    w[rows.long(), cols.long()] = values.float()
    return w.permute(0, 2, 1, 3).reshape(nbr * TILE, nbc * TILE)[:case["m"], :case["k"]]


def _tiles_of(dense, rows, cols, case):
    nbr, nbc = _grid(case)
    padded = torch.zeros(nbr * TILE, nbc * TILE, device="cuda")
    padded[:case["m"], :case["k"]] = dense
    return padded.view(nbr, TILE, nbc, TILE)[rows.long(), :, cols.long()]


def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    xhat = c * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y
    g = s["g"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (g * xhat).sum(0).to(s["w"].dtype),
            "db": g.sum(0).to(s["b"].dtype)}


def _plain_layer(s, x, w, bias, g):
    """(z, dz, dx, dw, db) of one weight's tokens; without g only z."""
    z = x @ w.t() + bias
    if g is None:
        return z, None, None, None, None
    dz = g * _act_slope(z, s["case"]["act"])
    return z, dz, dz @ w, dz.t() @ x, dz.sum(0)


def _run_plain(s):
    case = s["case"]
    op, act, train = case["op"], case.get("act"), case["train"]
    if op == "norm":
        return _plain_norm(s)
    dtype = DTYPES[case["dtype"]]
    x = s["x"].float()
    w = [_dense(v, r, c, case) for v, r, c in zip(s["values"], s["rows"], s["cols"])]
    if op == "int8":
        row = s["rows"][0].long()
        nbr = _grid(case)[0]
        scales = s["scales"].double()   # (sums whose order does not show in 32 bits)
        total = torch.zeros(nbr, dtype=torch.float64, device="cuda").index_add_(0, row, scales)
        held = torch.zeros(nbr, dtype=torch.float64, device="cuda").index_add_(0, row, torch.ones_like(scales))
        mean = (total / held.clamp_min(1.0)).float().repeat_interleave(TILE)[:case["m"]]
        y = _act((x @ w[0].t()) * mean * s["x_scale"][:, None] + s["bias"], act)
        return (y + s["r"].float() if case["residual"] else y).to(dtype)
    if op == "linear":
        z, _, dx, dw, db = _plain_layer(s, x, w[0], s["bias"].float(), s["g"].float() if train else None)
        y = _act(z, act)
        y = (y + s["r"].float() if case["residual"] else y).to(dtype)
        if not train:
            return y
        grads = [dx.to(dtype), _tiles_of(dw, s["rows"][0], s["cols"][0], case).to(dtype), db.to(s["bias"].dtype)]
        return {"y": y, "grads": grads + ([s["g"]] if case["residual"] else [])}
    runs = s["counts"] + [case["n"] - sum(s["counts"])]
    xs = x.split(runs)
    gs = s["g"].float().split(runs) if train else [None] * len(runs)
    parts = [_plain_layer(s, xs[e], w[e], s["bias"][e].float(), gs[e]) for e in range(case["experts"])]
    rest = runs[-1]
    y = torch.cat([_act(p[0], act) for p in parts] + [torch.zeros(rest, case["m"], device="cuda")]).to(dtype)
    if not train:
        return y
    dx = torch.cat([p[2] for p in parts] + [torch.zeros(rest, case["k"], device="cuda")]).to(dtype)
    dv = torch.cat([_tiles_of(p[3], r, c, case) for p, r, c in zip(parts, s["rows"], s["cols"])]).to(dtype)
    return {"y": y, "grads": [dx, dv, torch.stack([p[4] for p in parts]).to(s["bias"].dtype)]}


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    op, n = case["op"], case["n"]
    if op == "norm":
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        k = case["k"]
        mean = x.sum(1) / k
        var = (x * x).sum(1) / k - mean * mean
        inv = 1.0 / (var + EPS).sqrt()
        unit = torch.einsum("nk,n->nk", x, inv) - (mean * inv)[:, None]
        y = unit * w + b
        if not case["train"]:
            return y
        g = s["g"].double()
        a = torch.einsum("nk,k->n", g, w) / k
        c = torch.einsum("nk,k,nk->n", g, w, unit) / k
        dx = (g * w - a[:, None] - unit * c[:, None]) * inv[:, None]
        return {"y": y, "dx": dx, "dw": torch.einsum("nk,nk->k", g, unit), "db": torch.einsum("nk->k", g)}
    if 6.0 * n * case["m"] * case["k"] * (3 if case["train"] else 1) > 2e14:
        return None
    nbr, nbc = _grid(case)
    m, k = case["m"], case["k"]
    ends = [0]
    for e in range(case.get("experts", 1)):
        ends.append(ends[-1] + (s["counts"][e] if op == "experts" else n))
    y = torch.zeros(n, m, dtype=torch.float64, device="cuda")
    dx = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    dv, db = [], []
    inside = torch.arange(TILE, device="cuda")
    for e in range(len(ends) - 1):
        lo, hi = ends[e], ends[e + 1]
        at_row = (s["rows"][e].long()[:, None] * TILE + inside)[:, :, None]
        at_col = (s["cols"][e].long()[:, None] * TILE + inside)[:, None, :]
        values = s["values"][e].double()
        if op == "int8":   # every tile of a tile row counts with the mean of that row's tile scales
            row = s["rows"][e].long()
            mean = torch.zeros(nbr, dtype=torch.float64, device="cuda").scatter_reduce(0, row, s["scales"].double(), "mean", include_self=False)
            values = values * mean[row][:, None, None]
        a = torch.zeros(nbr * TILE, nbc * TILE, dtype=torch.float64, device="cuda").index_put_((at_row, at_col), values)[:m, :k]
        x = s["x"][lo:hi].double()
        if op == "int8":
            x = x * s["x_scale"].double()[:, None]
        z = torch.einsum("nk,mk->nm", x, a) + (s["bias"][e] if op == "experts" else s["bias"]).double()
        gate = {"gelu": 1.0 / (1.0 + torch.exp(-GELU_SCALE * (z + GELU_CUBIC * z ** 3))), "silu": 1.0 / (1.0 + torch.exp(-z)),
                "relu": (z > 0).double(), "none": torch.ones_like(z)}[case["act"]]
        y[lo:hi] = z * gate
        if op != "experts" and case["residual"]:
            y += s["r"].double()
        if not case["train"]:
            continue
        inner = {"gelu": GELU_SCALE * (1.0 + 3.0 * GELU_CUBIC * z ** 2), "silu": torch.ones_like(z)}.get(case["act"], torch.zeros_like(z))
        dz = s["g"][lo:hi].double() * (gate + z * gate * (1.0 - gate) * inner)
        dx[lo:hi] = torch.einsum("nm,mk->nk", dz, a)
        whole = torch.zeros(nbr * TILE, nbc * TILE, dtype=torch.float64, device="cuda")
        whole[:m, :k] = torch.einsum("nm,nk->mk", dz, x)
        dv.append(whole[at_row, at_col])
        db.append(torch.einsum("nm->m", dz))
    if not case["train"]:
        return y
    if op == "experts":
        return {"y": y, "grads": [dx, torch.cat(dv), torch.stack(db)]}
    return {"y": y, "grads": [dx, dv[0], db[0]] + ([s["g"].double()] if case["residual"] else [])}


# ------------------------------------------------------------------------------------------ what a pass is worth
def work(case):
    """Bytes and operations of one pass.  norm: the tokens in and out (training: the gradients too), a dozen operations per
    element.  The layers: the stored tiles of every weight that has tokens with their block columns, the tokens, biases and the
    residual in, the result out, two operations per multiply-add over the stored tiles of a token's weight; training reads the
    incoming gradient and writes those of tiles, tokens and biases, at three times the operations."""
    op, n, k = case["op"], case["n"], case["k"]
    es = 4 if case["dtype"] == "fp32" else 2
    if op == "norm":
        ps = 4 if case["params"] == "fp32" else es
        if case["train"]:
            return {"bytes": n * k * es * 4 + 4 * k * ps, "flops": 20.0 * n * k}
        return {"bytes": n * k * es * 2 + 2 * k * ps, "flops": 8.0 * n * k}
    m, stored = case["m"], _stored(case)
    if op == "experts":
        counts = _counts(case)
        used, active = sum(counts), sum(c > 0 for c in counts)
    else:
        used, active = n, 1
    tile = TILE * TILE * (1 if op == "int8" else es)
    ops = 2.0 * stored * TILE * TILE * used
    bias = active * m * (es if case["train"] else 4)
    x = used * k * (1 if op == "int8" else es)
    r = used * m * es if case.get("residual") else 0
    total = active * stored * (tile + 4) + bias + x + r + n * m * es + (n * 4 + stored * 4 if op == "int8" else 0)
    if case["train"]:
        total += case.get("experts", 1) * (stored * tile + m * es) + used * m * es + n * k * es
        ops *= 3.0
    return {"bytes": total, "flops": ops}
