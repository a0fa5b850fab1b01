"""What stands around the products of a layer of experts, and its products on dense 8-bit weights, as cases that can be timed: the
router that chooses a token's experts, the tokens brought into runs by expert and back, and linear layers whose e4m3 weights carry a
scale for each block of 128 x 128, as one matrix and as the matrices of experts.  ``own`` false: the plain form, elementary torch
operations in 32 bits.  ``own`` true: the calls a user makes of this framework.

A case is a dict of plain values; ``op`` and ``train`` say which path it takes:
  route     the k largest of a token's scores and their softmax                    void_route
  dispatch  tokens copied into the run of each of their experts                    void_dispatch
  combine   y_t = r_t + sum_j w_tj e(t, j), e the row that came of token t's j-th expert
                                                                                   void_combine
  linear    y = act(Q(x) A^T + b) + r, Q(x) x in e4m3 with a scale for each token's 128 features (the smallest power of two that
            keeps them within 448), A e4m3 with a scale for each block of 128 x 128
                                                                                   void_linear
  experts   the same for tokens sorted by expert, A_e and b_e of each run's expert void_expert_linear
"""
import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
INDEX = {"int32": torch.int32, "int64": torch.int64}
ACT_CODES = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
GELU_SCALE, GELU_CUBIC = 1.5957691216, 0.044715   # the framework's GELU: x * sigmoid(1.5957691216 (x + 0.044715 x^3))
MOST_WEIGHTS = 3.0e8     # elements of all experts' weights of a drawn case


def listed():
    return [
        # decode: sixteen tokens choose four of 64 experts, one launch's latency
        {"name": "route_decode", "op": "route", "train": False, "n": 16, "experts": 64, "top": 4, "dtype": "bf16", "normalize": True},
        # a training step of sixteen thousand tokens, eight of 128 experts, the softmax over all of them
        {"name": "route_train", "op": "route", "train": True, "n": 16384, "experts": 128, "top": 8, "dtype": "fp32", "normalize": False},
        # decode: sixteen tokens sent to two of eight experts each
        {"name": "dispatch_decode", "op": "dispatch", "train": False, "n": 16, "d": 2048, "experts": 8, "top": 2, "skew": 1.0,
         "dropped": 0.0, "dtype": "bf16", "index": "int32"},
        # prompt processing: eight thousand tokens to four of 64 experts each
        {"name": "dispatch_prompt", "op": "dispatch", "train": False, "n": 8192, "d": 4096, "experts": 64, "top": 4, "skew": 0.7,
         "dropped": 0.0, "dtype": "bf16", "index": "int32"},
        # training with sizes that are multiples of nothing; a tenth of the choices was dropped
        {"name": "dispatch_train_ragged", "op": "dispatch", "train": True, "n": 3001, "d": 5003, "experts": 17, "top": 3, "skew": 0.5,
         "dropped": 0.1, "dtype": "fp32", "index": "int64"},
        # decode: the experts' rows of sixteen tokens added to the residual stream
        {"name": "combine_decode", "op": "combine", "train": False, "n": 16, "d": 2048, "experts": 8, "top": 2, "skew": 1.0,
         "dropped": 0.0, "dtype": "bf16", "residual": True},
        # a training step of eight thousand tokens: gradients of the experts' rows and of the weights
        {"name": "combine_train", "op": "combine", "train": True, "n": 8192, "d": 4096, "experts": 64, "top": 4, "skew": 0.7,
         "dropped": 0.0, "dtype": "bf16", "residual": False},
        # decode: eight sequences through a layer of the headline's width
        {"name": "linear_decode", "op": "linear", "train": False, "n": 8, "k": 8192, "m": 8192, "dtype": "bf16", "act": "none",
         "residual": True},
        # sizes that are multiples of nothing
        {"name": "linear_ragged", "op": "linear", "train": False, "n": 333, "k": 5003, "m": 3001, "dtype": "fp16", "act": "gelu",
         "residual": False},
        # prompt processing: eight thousand tokens through the same layer
        {"name": "linear_prompt", "op": "linear", "train": False, "n": 8192, "k": 8192, "m": 8192, "dtype": "bf16", "act": "none",
         "residual": True},
        # decode: sixteen tokens sent to two experts each
        {"name": "experts_decode", "op": "experts", "train": False, "n": 32, "k": 2048, "m": 8192, "experts": 8, "skew": 1.0,
         "spare": 0, "dtype": "bf16", "act": "silu"},
        # prompt processing: sixteen thousand routed tokens, a few popular experts, a buffer longer than what is routed
        {"name": "experts_prompt", "op": "experts", "train": False, "n": 16384, "k": 2048, "m": 8192, "experts": 16, "skew": 0.7,
         "spare": 511, "dtype": "bf16", "act": "silu"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _side(rng, lo, hi):
    """A width over the whole range: a multiple of the block, of 16, or any number."""
    v = _log_int(rng, lo, hi)
    unit = rng.choice((128, 16, 1))
    return max(lo, v // unit * unit)


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(("route", "dispatch", "dispatch", "combine", "combine", "linear", "linear", "experts", "experts"))
        dtype = rng.choice(("fp32", "fp16", "bf16"))
        act = rng.choice(("none", "relu", "gelu", "silu"))
        experts = _log_int(rng, 2, 256)
        top = rng.randint(1, min(8, experts))
        skew = round(rng.uniform(0.0, 1.5), 2)
        if op == "route":
            c = {"op": op, "train": rng.random() < 0.5, "n": _log_int(rng, 1, 16384), "experts": experts, "top": top, "dtype": dtype,
                 "normalize": rng.random() < 0.5}
        elif op in ("dispatch", "combine"):
            c = {"op": op, "train": rng.random() < 0.5, "n": _log_int(rng, 1, 16384), "d": _side(rng, 128, 16384), "experts": experts,
                 "top": top, "skew": skew, "dropped": rng.choice((0.0, round(rng.uniform(0.0, 0.5), 2))), "dtype": dtype}
            if op == "dispatch":
                c["index"] = rng.choice(("int32", "int64"))
            else:
                c["residual"] = rng.random() < 0.5
        elif op == "linear":
            c = {"op": op, "train": False, "n": _log_int(rng, 1, 8192), "k": _side(rng, 256, 16384), "m": _side(rng, 256, 16384),
                 "dtype": dtype, "act": act, "residual": rng.random() < 0.5}
        else:
            n = _log_int(rng, 1, 16384)
            c = {"op": op, "train": False, "n": n, "k": _side(rng, 256, 8192), "m": _side(rng, 256, 8192),
                 "experts": _log_int(rng, 2, 64), "skew": skew, "spare": rng.choice((0, rng.randint(0, n // 2))), "dtype": dtype, "act": act}
            if c["experts"] * c["k"] * c["m"] > MOST_WEIGHTS:
                continue
        w = work(c)
        if w["flops"] <= max(x["flops"] for x in most) and w["bytes"] <= max(x["bytes"] for x in most):
            return c


# ------------------------------------------------------------------------------------------ inputs
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


def _choices(gen, case):
    """Every token's experts, no expert twice, popular ones as rank^-skew; some choices dropped (-1)."""
    n, experts, top = case["n"], case["experts"], case["top"]
    share = -case["skew"] * (torch.randperm(experts, generator=gen, device="cuda") + 1.0).log()
    noise = -(-torch.rand(n, experts, generator=gen, device="cuda").clamp_min(1e-30).log()).log()
    chosen = (share + noise).topk(top, dim=1).indices
    return torch.where(torch.rand(n, top, generator=gen, device="cuda") < case["dropped"], -1, chosen)


def _places(chosen, experts):
    """Row of every choice when all are sorted by expert in the order of the tokens, -1 for a dropped one, and the runs' ends."""
    flat = chosen.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = key.sort(stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device="cuda")
    place = torch.where(flat < 0, -1, place).view(chosen.shape)
    counts = (key[:, None] == torch.arange(experts, device="cuda")).sum(0)
    return place.int(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()


def _weights(gen, case, experts):
    """e4m3 weights as they come of quantised normal ones, and a scale per block."""
    k, m = case["k"], case["m"]
    shape = (m, k) if experts is None else (experts, m, k)
    blocks = shape[:-2] + ((m + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK)
    values = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    for part in (values,) if experts is None else values:
        part.copy_((torch.randn(m, k, generator=gen, device="cuda") * 110.0).clamp_(-FP8_MAX, FP8_MAX))
    return values, (torch.rand(blocks, generator=gen, device="cuda") + 0.5) * (k ** -0.5 / 110.0)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, n = case["op"], case["n"]
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = {"case": dict(case)}
    if op == "route":
        s["scores"] = randn(n, case["experts"], scale=2.0)
        if case["train"]:
            s["g"] = randn(n, case["top"], dtype=torch.float32)
        return s
    if op in ("dispatch", "combine"):
        d, rows = case["d"], n * case["top"]
        chosen = _choices(gen, case)
        if op == "dispatch":
            s["x"], s["chosen"] = randn(n, d), chosen.to(INDEX[case["index"]])
            if case["train"]:
                s["g"] = randn(rows, d)
            return s
        s["chosen"] = chosen.int()
        s["y"] = randn(rows, d)
        s["w"] = torch.rand(n, case["top"], generator=gen, device="cuda")
        if case["residual"]:
            s["r"] = randn(n, d)
        if case["train"]:
            s["g"] = randn(n, d)
        return s
    k, m, experts = case["k"], case["m"], case.get("experts")
    s["values"], s["scales"] = _weights(gen, case, experts)
    # activations: features of different sizes
    s["x"] = (torch.randn(n, k, generator=gen, device="cuda") * torch.rand(k, generator=gen, device="cuda").add_(0.25)).to(dtype)
    if op == "linear":
        s["bias"] = randn(m, dtype=torch.float32, scale=0.2)
        if case["residual"]:
            s["r"] = randn(n, m)
        return s
    s["bias"] = randn(experts, m, dtype=torch.float32, scale=0.2)
    counts = _counts(case)
    order = torch.randperm(experts, generator=torch.Generator().manual_seed(int(seed))).tolist()
    s["counts"] = [counts[e] for e in order]
    s["offsets"] = torch.tensor([0] + s["counts"], dtype=torch.int64).cumsum(0).int().cuda()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if own:
        import void_b200 as void
        if case["train"]:
            for name in ("scores", "x", "y", "w", "r"):
                if name in s:
                    s[name].requires_grad_(True)
        if op == "combine":
            s["routes"] = void.sort_by_expert(s["chosen"], case["experts"])
        elif op in ("linear", "experts"):
            s["a"] = void.FP8BlockTensor(s["values"], s["scales"])
    elif op == "combine":
        s["place"] = _places(s["chosen"], case["experts"])[0]
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import void_b200 as void
    case = s["case"]
    op, train = case["op"], case["train"]
    if op == "route":
        chosen, w = void.void_route(s["scores"], case["top"], normalize=case["normalize"])
        if not train:
            return {"chosen": chosen, "w": w}
        return {"chosen": chosen, "w": w.detach(), "ds": torch.autograd.grad(w, s["scores"], s["g"])[0]}
    if op == "dispatch":
        xs, routes = void.void_dispatch(s["x"], s["chosen"], case["experts"])
        out = {"xs": xs.detach(), "offsets": routes.offsets, "place": routes.position}
        if train:
            out["dx"] = torch.autograd.grad(xs, s["x"], s["g"])[0]
        return out
    if op == "combine":
        y = void.void_combine(s["y"], s["routes"], s["w"], residual=s.get("r"))
        if not train:
            return y
        leaves = (s["y"], s["w"]) + ((s["r"],) if case["residual"] else ())
        return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, s["g"]))}
    if op == "linear":
        return void.void_linear(s["a"], s["x"], s["bias"], ACT_CODES[case["act"]], residual=s.get("r"))
    return void.void_expert_linear(s["a"], s["x"], s["offsets"], s["bias"], ACT_CODES[case["act"]])


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return z * torch.sigmoid(GELU_SCALE * (z + GELU_CUBIC * z * z * z))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _plain_route(s):
    case = s["case"]
    scores = s["scores"].float()
    best, chosen = scores.sort(dim=1, descending=True, stable=True)     # (ties: the lowest index first)
    best, chosen = best[:, :case["top"]], chosen[:, :case["top"]]
    e = (best - best[:, :1]).exp()
    if case["normalize"]:
        w = e / e.sum(1, keepdim=True)
    else:
        p = (scores - best[:, :1]).exp()
        p = p / p.sum(1, keepdim=True)
        w = p.gather(1, chosen)
    out = {"chosen": chosen.int(), "w": w}
    if case["train"]:
        g = s["g"]
        mean = (g * w).sum(1, keepdim=True)
        if case["normalize"]:
            ds = torch.zeros_like(scores).scatter(1, chosen, w * (g - mean))
        else:
            ds = p * (torch.zeros_like(scores).scatter(1, chosen, g) - mean)
        out["ds"] = ds.to(s["scores"].dtype)
    return out


def _plain_dispatch(s):
    case = s["case"]
    x, top = s["x"], case["top"]
    place, offsets = _places(s["chosen"], case["experts"])
    flat = place.reshape(-1).long()
    token = torch.arange(flat.numel(), device="cuda") // top
    rows = torch.where(flat < 0, flat.numel(), flat)
    xs = torch.zeros(flat.numel() + 1, case["d"], dtype=x.dtype, device="cuda")
    xs[rows] = torch.where((flat < 0)[:, None], 0.0, x[token]).to(x.dtype)
    out = {"xs": xs[:-1], "offsets": offsets, "place": place}
    if case["train"]:
        g = torch.cat([s["g"].float(), torch.zeros(1, case["d"], device="cuda")])
        out["dx"] = g[rows].view(case["n"], top, -1).sum(1).to(x.dtype)
    return out


def _plain_combine(s):
    case = s["case"]
    y, n, top, d = s["y"], case["n"], case["top"], case["d"]
    place = s["place"].long()
    kept = place >= 0
    rows = torch.cat([y, torch.zeros(1, d, dtype=y.dtype, device="cuda")])[torch.where(kept, place, n * top)].float()
    w = torch.where(kept, s["w"], 0.0)
    z = (rows * w[:, :, None]).sum(1)
    if case["residual"]:
        z = z + s["r"].float()
    z = z.to(y.dtype)
    if not case["train"]:
        return z
    g = s["g"].float()
    dw = (rows * g[:, None, :]).sum(2)
    dy = torch.zeros(n * top + 1, d, device="cuda")
    dy[torch.where(kept, place, n * top).reshape(-1)] = (w[:, :, None] * g[:, None, :]).view(n * top, d)
    return {"y": z, "grads": [dy[:-1].to(y.dtype), dw] + ([s["g"]] if case["residual"] else [])}


def _plain_quantised(x):
    """x in e4m3 with a scale for each row's 128 columns, as the values it stands for."""
    n, k = x.shape
    blocks = (k + BLOCK - 1) // BLOCK
    padded = torch.zeros(n, blocks * BLOCK, device="cuda")
    padded[:, :k] = x.float()
    padded = padded.view(n, blocks, BLOCK)
    part, power = torch.frexp(padded.abs().amax(2, keepdim=True))      # 448 is 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(part), (power - 9 + (part > 0.875).int()).clamp_min(-100))
    q = (padded / scale).to(torch.float8_e4m3fn).float()
    return (q * scale).view(n, blocks * BLOCK)[:, :k]


def _plain_weight(values, scales):
    m, k = values.shape
    return values.float() * scales.repeat_interleave(BLOCK, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        return _plain_route(s)
    if op == "dispatch":
        return _plain_dispatch(s)
    if op == "combine":
        return _plain_combine(s)
    dtype, act = DTYPES[case["dtype"]], case["act"]
    x = _plain_quantised(s["x"])
    if op == "linear":
        y = _act(x @ _plain_weight(s["values"], s["scales"]).t() + s["bias"], act)
        return (y + s["r"].float() if case["residual"] else y).to(dtype)
    y = torch.zeros(case["n"], case["m"], dtype=dtype, device="cuda")
    at = 0
    for e, count in enumerate(s["counts"]):
        if count:
            y[at:at + count] = _act(x[at:at + count] @ _plain_weight(s["values"][e], s["scales"][e]).t() + s["bias"][e], act).to(dtype)
        at += count
    return y


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def _rows_of(chosen, experts):
    """Rows (flat choice numbers) by expert, in the order of the tokens, and the runs' ends, expert by expert."""
    flat = chosen.reshape(-1)
    runs = [(flat == e).nonzero().flatten() for e in range(experts)]
    ends = [0]
    for r in runs:
        ends.append(ends[-1] + r.numel())
    return torch.cat(runs), torch.tensor(ends, dtype=torch.int32, device="cuda")


def _e4m3(v):
    """The nearest e4m3 number (ties to the even one) of numbers of at most 448: three bits behind the leading one, steps of 2^-9 at
    the least."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def exact(case, seed):
    s = _inputs(case, seed)
    op, n = case["op"], case["n"]
    if op == "route":
        scores, top = s["scores"].double(), case["top"]
        left, picks = scores.clone(), []
        for _ in range(top):
            best = left.max(1, keepdim=True).values
            at = (left == best).to(torch.int8).argmax(1, keepdim=True)
            picks.append(at)
            left = left.scatter(1, at, -math.inf)
        chosen = torch.cat(picks, 1)
        picked = torch.zeros_like(scores, dtype=torch.bool).scatter(1, chosen, True)
        among = picked if case["normalize"] else torch.ones_like(picked)
        p = torch.softmax(torch.where(among, scores, -math.inf), dim=1)
        out = {"chosen": chosen.int(), "w": p.gather(1, chosen)}
        if case["train"]:
            g = torch.zeros_like(scores).scatter(1, chosen, s["g"].double())
            out["ds"] = p * g - p * torch.einsum("ne,ne->n", p, g)[:, None]
        return out
    if op in ("dispatch", "combine"):
        top, d = case["top"], case["d"]
        order, ends = _rows_of(s["chosen"], case["experts"])
        place = torch.full((n * top,), -1, dtype=torch.int32, device="cuda")
        place[order] = torch.arange(order.numel(), dtype=torch.int32, device="cuda")
        token = order // top
        if op == "dispatch":
            xs = torch.zeros(n * top, d, dtype=torch.float64, device="cuda")
            xs[:order.numel()] = s["x"][token].double()
            out = {"xs": xs, "offsets": ends, "place": place.view(n, top)}
            if case["train"]:
                out["dx"] = torch.zeros(n, d, dtype=torch.float64, device="cuda").index_add_(0, token, s["g"][:order.numel()].double())
            return out
        w = s["w"].double().reshape(-1)[order]
        rows = s["y"][:order.numel()].double()
        z = s["r"].double() if case["residual"] else torch.zeros(n, d, dtype=torch.float64, device="cuda")
        z = z.index_add(0, token, w[:, None] * rows)
        if not case["train"]:
            return z
        g = s["g"].double()
        dy = torch.zeros(n * top, d, dtype=torch.float64, device="cuda")
        dy[:order.numel()] = w[:, None] * g[token]
        dw = torch.zeros(n * top, dtype=torch.float64, device="cuda")
        dw[order] = torch.einsum("rd,rd->r", rows, g[token])
        return {"y": z, "grads": [dy, dw.view(n, top)] + ([g] if case["residual"] else [])}
    k, m = case["k"], case["m"]
    x = s["x"].double()
    for first in range(0, k, BLOCK):
        part = x[:, first:first + BLOCK]
        unit = torch.exp2(torch.ceil(torch.log2(part.abs().max(1, keepdim=True).values / FP8_MAX)).clamp_min(-100.0))
        x[:, first:first + BLOCK] = _e4m3(part / unit) * unit
    gates = {"gelu": lambda z: 1.0 / (1.0 + torch.exp(-GELU_SCALE * (z + GELU_CUBIC * z ** 3))),
             "silu": lambda z: 1.0 / (1.0 + torch.exp(-z)), "relu": lambda z: (z > 0).double(), "none": torch.ones_like}
    y = torch.zeros(n, m, dtype=torch.float64, device="cuda")
    at = 0
    for e, count in enumerate([n] if op == "linear" else s["counts"]):
        values, scales, bias = (s["values"], s["scales"], s["bias"]) if op == "linear" else (s["values"][e], s["scales"][e], s["bias"][e])
        for first in range(0, m, BLOCK):
            a = values[first:first + BLOCK].double()
            a *= scales[first // BLOCK].double().repeat_interleave(BLOCK)[:k]
            z = torch.einsum("nk,mk->nm", x[at:at + count], a) + bias[first:first + BLOCK].double()
            y[at:at + count, first:first + BLOCK] = z * gates[case["act"]](z)
        at += count
    return y + s["r"].double() if case.get("residual") else y


# ------------------------------------------------------------------------------------------ what a pass is worth
def work(case):
    """Bytes and operations of one pass.  route: the scores in, the choices and their weights out (training: the weights' gradient in,
    the scores' out).  dispatch, combine: the tokens on one side, the rows of all choices on the other (training: the gradients of
    both).  linear, experts: the weights of every matrix that has tokens with their scales, the tokens, biases and the residual in, the
    result out, two operations per multiply-add."""
    op, n = case["op"], case["n"]
    es = 4 if case["dtype"] == "fp32" else 2
    if op == "route":
        experts, top = case["experts"], case["top"]
        passes = 2 if case["train"] else 1
        return {"bytes": n * experts * es * passes + n * top * (8 + 4 * (passes - 1)), "flops": 6.0 * n * experts * passes}
    if op in ("dispatch", "combine"):
        d, top = case["d"], case["top"]
        rows = round(n * top * (1.0 - case["dropped"]))
        if op == "dispatch":
            index = 4 if case["index"] == "int32" else 8
            total = n * d * es + n * top * d * es + n * top * (index + 4) + 4 * (case["experts"] + 1)
            return {"bytes": total + ((rows + n) * d * es if case["train"] else 0), "flops": float(rows * d if case["train"] else n * top)}
        total = rows * d * es + n * d * es * (2 if case["residual"] else 1) + n * top * 8
        if case["train"]:
            total += n * d * es + n * top * d * es + n * top * 4
        return {"bytes": total, "flops": 2.0 * rows * d * (3 if case["train"] else 1)}
    k, m = case["k"], case["m"]
    blocks = ((m + BLOCK - 1) // BLOCK) * ((k + BLOCK - 1) // BLOCK)
    if op == "linear":
        used, active = n, 1
    else:
        counts = _counts(case)
        used, active = sum(counts), sum(c > 0 for c in counts)
    total = active * (m * k + 4 * blocks + 4 * m) + used * k * es + n * m * es + (n * m * es if case.get("residual") else 0)
    return {"bytes": total, "flops": 2.0 * used * k * m}
