"""Cases for the operators that a conditional flow's context net is trained with: ``nessai_amd.ops.embedding``,
``group_norm_act``, ``grad_norm`` and ``clip_grad_norm_``.

``own`` False: the operators in elementary torch operations, in 32 bits, rounded once.  ``own`` True: the calls that a
user of the framework makes.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "int64": 8}


def listed():
    return [
        # gradients of the default RealNVP of a low-dimensional problem, slices of the flow's flat gradient: latency alone
        dict(name="clip_small_flow", op="clip", tensors=48, total=9_600, spread=3.0, layout="flat", dtype="float32",
             norm="2"),
        # the 32-dimensional spline flow (6 couplings, 64 hidden units, 8 bins): 72 tensors, 250 thousand values
        dict(name="clip_spline_flow", op="clip", tensors=72, total=249_888, spread=5.0, layout="flat", dtype="float32",
             norm="2"),
        # a flow with a context net kept in 16 bits, every gradient a tensor of its own at an odd place
        dict(name="clip_many_bf16", op="clip", tensors=301, total=40_000_001, spread=8.0, layout="pieces",
             dtype="bfloat16", norm="2"),
        # the norm alone, as a loop reports it: a large table and hundreds of smaller tensors, 1.2 GB
        dict(name="norm_large", op="norm", tensors=400, total=300_000_000, spread=9.0, layout="pieces", dtype="float32",
             norm="2"),
        # hidden features of a minibatch of 1000 live points, 64 wide
        dict(name="group_norm_minibatch", op="group_norm", samples=1000, length=1, channels=64, groups=8,
             dtype="float32", affine="same", activation="silu", train=True),
        # the same for rows of a large training set in one piece, 128 wide
        dict(name="group_norm_rows", op="group_norm", samples=200_003, length=1, channels=128, groups=32,
             dtype="float32", affine="same", activation="tanh", train=True),
        # time series (16 of 4096 positions, 256 features) on the way to a context, evaluation only
        dict(name="group_norm_series", op="group_norm", samples=16, length=4096, channels=256, groups=32,
             dtype="bfloat16", affine="float32", activation="silu", train=False),
        # one long time series in training, an odd length and a width that no vector divides
        dict(name="group_norm_odd", op="group_norm", samples=3, length=20_001, channels=90, groups=9, dtype="float16",
             affine="same", activation="relu", train=True),
        # labels of a minibatch (which of six models): a table of six rows
        dict(name="embedding_labels", op="embedding", tokens=1000, vocab=6, width=16, dtype="float32", index="int64",
             skew="uniform", pad=False, train=True),
        # labels of a million draws: long sums into few rows
        dict(name="embedding_draws", op="embedding", tokens=1_000_000, vocab=40, width=64, dtype="float32",
             index="int64", skew="uniform", pad=False, train=True),
        # event identifiers looked up for evaluation, a table larger than the caches
        dict(name="embedding_lookup", op="embedding", tokens=200_003, vocab=400_000, width=512, dtype="bfloat16",
             index="int32", skew="uniform", pad=False, train=False),
        # identifiers of uneven frequency with padding in training, a width that is no power of two
        dict(name="embedding_uneven", op="embedding", tokens=131_072, vocab=32_768, width=320, dtype="bfloat16",
             index="int64", skew="uneven", pad=True, train=True),
    ]


def _between(rng, low, high):
    """A whole number, spread over the logarithm of the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["clip", "norm", "group_norm", "group_norm", "embedding", "embedding"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    if op in ("clip", "norm"):
        total = _between(rng, 500, 100_000_000)
        return dict(op=op, tensors=min(total, _between(rng, 1, 600)), total=total, spread=rng.choice([0.0, 3.0, 8.0]),
                    layout=rng.choice(["flat", "pieces"]), dtype=dtype, norm=rng.choice(["2", "2", "2", "inf", "1"]))
    if op == "group_norm":
        groups = rng.choice([1, 2, 3, 4, 6, 8, 9, 16, 32])
        channels = groups * _between(rng, 1, max(1, 1024 // groups))
        length = 1 if rng.random() < 0.4 else _between(rng, 2, 40_000)
        if length * channels // groups < 8:
            channels = 8 * groups  # (of two or three values the gradient is a difference of nearly equal numbers)
        samples = _between(rng, 1, max(1, min(300_000, 25_000_000 // (length * channels))))
        train = rng.random() < 0.7
        # (a training case has relu in 16 bits only: where z is within a rounding of zero its gradient jumps)
        activations = ["none", "tanh", "silu"] + ([] if train and dtype == "float32" else ["relu"])
        return dict(op=op, samples=samples, length=length, channels=channels, groups=groups, dtype=dtype,
                    affine=rng.choice(["none", "same", "float32"]), activation=rng.choice(activations), train=train)
    width = _between(rng, 1, 1024)
    tokens = _between(rng, 1, max(1, min(1_000_000, 60_000_000 // width)))
    vocab = _between(rng, 2, max(2, min(400_000, 100_000_000 // width)))
    return dict(op=op, tokens=tokens, vocab=vocab, width=width, dtype=dtype, index=rng.choice(["int64", "int32"]),
                skew=rng.choice(["uniform", "uneven"]), pad=rng.random() < 0.4, train=rng.random() < 0.7)


# -- inputs ---------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _sizes(case):
    """Sizes of the tensors: the same for every seed, spread over ``exp(spread)``, all together about ``total``."""
    weights = [math.exp(case["spread"] * ((i * 0.6180339887498949) % 1.0)) for i in range(case["tensors"])]
    scale = case["total"] / sum(weights)
    return [max(1, int(w * scale)) for w in weights]


def _places(case):
    """(start, size) of each tensor in the buffer, and the buffer's length: side by side, or apart by odd gaps."""
    places, at = [], 0
    for i, size in enumerate(_sizes(case)):
        if case["layout"] == "pieces":
            at += 1 + (7 * i) % 13
        places.append((at, size))
        at += size
    return places, at


def _gradients(case, seed):
    """Gradients as a backward pass leaves them: each tensor with a scale of its own."""
    places, length = _places(case)
    gen = _generator(seed)
    flat = _normal((length,), gen)
    scales = torch.exp(2.0 * _normal((len(places),), gen)) * 1e-2
    starts = torch.tensor([start for start, _ in places], device=DEVICE)
    which = torch.searchsorted(starts, torch.arange(length, device=DEVICE), right=True).sub_(1).clamp_(min=0)
    return flat.mul_(scales[which]).to(DTYPES[case["dtype"]])


MAX_NORM = {"2": 0.05, "inf": 1e-3, "1": 5.0}  # small enough that every case is clipped


def _group_norm_inputs(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    n, length, channels = case["samples"], case["length"], case["channels"]
    centre, width = 2.0 * _normal((channels,), gen), torch.exp(0.5 * _normal((channels,), gen))
    x = (_normal((n, length, channels), gen) * width + centre).to(dtype)
    x = x.reshape(n, channels) if length == 1 else x
    weight = bias = None
    if case["affine"] != "none":
        kind = torch.float32 if case["affine"] == "float32" else dtype
        weight = (1.0 + 0.3 * _normal((channels,), gen)).to(kind)
        bias = (0.3 * _normal((channels,), gen)).to(kind)
    dy = _normal(tuple(x.shape), gen).to(dtype) if case["train"] else None
    return x, weight, bias, dy


def _embedding_inputs(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    u = torch.rand((case["tokens"],), generator=gen, device=DEVICE, dtype=torch.float64)
    if case["skew"] == "uneven":  # frequencies that fall as one over the rank
        ids = torch.exp(u * math.log(case["vocab"] + 1.0)) - 1.0
    else:
        ids = u * case["vocab"]
    ids = ids.to(torch.int64).clamp_(0, case["vocab"] - 1).to(getattr(torch, case["index"]))
    weight = (_normal((case["vocab"], case["width"]), gen) / math.sqrt(case["width"])).to(dtype)
    dy = _normal((case["tokens"], case["width"]), gen).to(dtype) if case["train"] else None
    return ids, weight, dy


def prepare(case, seed):
    state = dict(case)
    if case["op"] in ("clip", "norm"):
        fresh = _gradients(case, seed)
        flat = fresh.clone()
        values = torch.zeros_like(flat)
        params = []
        for start, size in _places(case)[0]:
            p = torch.nn.Parameter(values[start : start + size])
            p.grad = flat[start : start + size]
            params.append(p)
        state.update(fresh=fresh, flat=flat, params=params, p=float(case["norm"]), max_norm=MAX_NORM[case["norm"]])
    elif case["op"] == "group_norm":
        x, weight, bias, dy = _group_norm_inputs(case, seed)
        if case["train"]:
            x.requires_grad_(True)
            if weight is not None:
                weight.requires_grad_(True)
                bias.requires_grad_(True)
        state.update(x=x, weight=weight, bias=bias, dy=dy)
    else:
        ids, weight, dy = _embedding_inputs(case, seed)
        if case["train"]:
            weight.requires_grad_(True)
        state.update(ids=ids, weight=weight, dy=dy, scale=math.sqrt(case["width"]), padding=0 if case["pad"] else None)
    return state


# -- one pass -------------------------------------------------------------------------------------------------------


def run(state):
    if state["op"] in ("clip", "norm"):
        return _run_clip(state)
    if state["op"] == "group_norm":
        return _run_group_norm(state)
    return _run_embedding(state)


def _plain_norm(grads, p):
    if p == math.inf:
        return torch.stack([g.float().abs().max() for g in grads]).max()
    if p == 1.0:
        return torch.stack([g.float().abs().sum() for g in grads]).sum()
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _run_clip(state):
    if state["op"] == "norm":
        if own:
            from nessai_amd import ops

            return {"norm": ops.grad_norm([p.grad for p in state["params"]], state["p"])}
        return {"norm": _plain_norm([p.grad for p in state["params"]], state["p"])}
    # the gradients of this step arrive in the buffer that is clipped in place (a pass over clipped gradients would
    # have nothing to clip); the copy is part of the pass on both sides
    state["flat"].copy_(state["fresh"])
    if own:
        from nessai_amd import ops

        norm = ops.clip_grad_norm_(state["params"], state["max_norm"], norm_type=state["p"])
    else:
        grads = [p.grad for p in state["params"]]
        norm = _plain_norm(grads, state["p"])
        factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        [g.copy_(g.float() * factor) for g in grads]
    return {"norm": norm, "grads": state["flat"]}


def _act(z, name):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "tanh":
        t = torch.tanh(z)
        return 1.0 - t * t
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


EPS = 1e-5


def _run_group_norm(state):
    x, weight, bias, dy = state["x"], state["weight"], state["bias"], state["dy"]
    name = state["activation"]
    if own:
        from nessai_amd import ops

        y = ops.group_norm_act(x, state["groups"], weight, bias, eps=EPS, activation=None if name == "none" else name)
        if not state["train"]:
            return {"y": y}
        wanted = [x] if weight is None else [x, weight, bias]
        grads = torch.autograd.grad(y, wanted, dy)
        return {"y": y, **dict(zip(("dx", "dweight", "dbias"), grads))}
    with torch.no_grad():
        shape = (state["samples"], state["length"], state["groups"], state["channels"] // state["groups"])
        xf = x.float().reshape(shape)
        w = torch.ones((), device=x.device) if weight is None else weight.float().reshape(shape[2:])
        b = torch.zeros((), device=x.device) if bias is None else bias.float().reshape(shape[2:])
        centred = xf - xf.mean((1, 3), keepdim=True)
        rstd = 1.0 / torch.sqrt(centred.square().mean((1, 3), keepdim=True) + EPS)
        xh = centred * rstd
        z = xh * w + b
        out = {"y": _act(z, name).reshape(x.shape).to(x.dtype)}
        if state["train"]:
            dz = dy.float().reshape(shape) * _act_slope(z, name)
            dxh = dz * w
            mean_1, mean_2 = dxh.mean((1, 3), keepdim=True), (dxh * xh).mean((1, 3), keepdim=True)
            out["dx"] = (rstd * (dxh - mean_1 - xh * mean_2)).reshape(x.shape).to(x.dtype)
            if weight is not None:
                out["dweight"] = (dz * xh).sum((0, 1)).reshape(-1).to(weight.dtype)
                out["dbias"] = dz.sum((0, 1)).reshape(-1).to(bias.dtype)
        return out


def _run_embedding(state):
    ids, weight, dy, scale = state["ids"], state["weight"], state["dy"], state["scale"]
    if own:
        from nessai_amd import ops

        out = ops.embedding(ids, weight, scale=scale, padding_idx=state["padding"])
        if not state["train"]:
            return {"out": out}
        (dweight,) = torch.autograd.grad(out, [weight], dy)
        return {"out": out, "dweight": dweight}
    with torch.no_grad():
        out = {"out": (weight[ids].float() * scale).to(weight.dtype)}
        if state["train"]:
            # the rows in the order of their identifiers, and differences of one running sum (64 bits: it is long)
            order = torch.argsort(ids, stable=True)
            sums = torch.cumsum(dy[order].double().t().contiguous(), 1)
            sums = torch.cat([torch.zeros_like(sums[:, :1]), sums], 1)
            rows = torch.arange(weight.shape[0], dtype=ids.dtype, device=ids.device)
            ends = torch.searchsorted(ids[order], rows, right=True)
            starts = torch.cat([torch.zeros_like(ends[:1]), ends[:-1]])
            total = (sums[:, ends] - sums[:, starts]).t() * scale
            if state["padding"] is not None:
                total[state["padding"]] = 0.0
            out["dweight"] = total.to(weight.dtype).contiguous()
        return out


# -- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] in ("clip", "norm"):
        values = sum(_sizes(case))
        if case["op"] == "norm":
            return {"bytes": values * size, "flops": 2 * values}
        return {"bytes": 4 * values * size, "flops": 3 * values}  # the gradients' arrival, then one read and one write
    if case["op"] == "group_norm":
        values = case["samples"] * case["length"] * case["channels"]
        if case["train"]:  # x and dy in, y and dx out
            return {"bytes": 4 * values * size, "flops": 40 * values}
        return {"bytes": 2 * values * size, "flops": 15 * values}
    n, width, vocab = case["tokens"], case["width"], case["vocab"]
    # (rows of the table that are read: at most as many as there are tokens)
    total = n * BYTES[case["index"]] + min(n, vocab) * width * size + n * width * size
    if case["train"]:
        total += n * BYTES[case["index"]] + n * width * size + vocab * width * size
    return {"bytes": total, "flops": n * width * (2 if case["train"] else 1)}


# -- the definitions in 64 bits -------------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] in ("clip", "norm"):
        return _exact_clip(case, seed)
    if case["op"] == "group_norm":
        return _exact_group_norm(case, seed)
    return _exact_embedding(case, seed)


def _exact_clip(case, seed):
    flat = _gradients(case, seed).double()
    inside = torch.zeros(flat.numel() + 1, dtype=torch.int32, device=DEVICE)
    places, _ = _places(case)
    starts = torch.tensor([s for s, _ in places], device=DEVICE)
    ends = torch.tensor([s + n for s, n in places], device=DEVICE)
    one = torch.ones(len(places), dtype=torch.int32, device=DEVICE)
    inside.index_add_(0, starts, one).index_add_(0, ends, -one)
    inside = torch.cumsum(inside, 0)[:-1] > 0
    p = float(case["norm"])
    norm = torch.linalg.vector_norm(flat[inside], p)
    if case["op"] == "norm":
        return {"norm": norm}
    factor = min(1.0, MAX_NORM[case["norm"]] / (float(norm) + 1e-6))
    return {"norm": norm, "grads": torch.where(inside, flat * factor, flat)}


def _exact_group_norm(case, seed):
    x, weight, bias, dy = _group_norm_inputs(case, seed)
    shape = (case["samples"], case["length"], case["groups"], -1)
    leaves = [t.double().requires_grad_(case["train"]) for t in (x, weight, bias) if t is not None]
    rows = leaves[0].reshape(shape)
    var, mean = torch.var_mean(rows, (1, 3), correction=0, keepdim=True)
    z = ((rows - mean) / torch.sqrt(var + EPS)).reshape(x.shape)
    if weight is not None:
        z = z * leaves[1] + leaves[2]
    y = {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh, "silu": lambda v: v * torch.sigmoid(v)}[
        case["activation"]](z)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, leaves, dy.double())
    return {"y": y.detach(), **dict(zip(("dx", "dweight", "dbias"), grads))}


def _exact_embedding(case, seed):
    ids, weight, dy = _embedding_inputs(case, seed)
    ids, scale = ids.long(), math.sqrt(case["width"])
    out = {"out": weight.double().index_select(0, ids) * scale}
    if case["train"]:
        total = torch.zeros(weight.shape, dtype=torch.float64, device=DEVICE).index_add_(0, ids, dy.double())
        if case["pad"]:
            total[0] = 0.0
        out["dweight"] = total * scale
    return out
