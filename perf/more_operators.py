"""The pieces of a mixture-of-experts layer over frozen MXFP4 weights, with their gradients, as
timed cases: tokens sorted by expert and back, the router's gradient, products with bias,
activation and residual (dense, or every row by its own expert's matrix), and the experts'
gated projection.

T tokens choose top_k of E experts each: slot t * top_k + i is token t's i-th choice, and `perm`
lists the slots by expert, in slot order within one; `offsets` says where each expert's begin.
An MXFP4 row holds, per 32 values, one E8M0 byte s and 32 E2M1 codes (two to a byte, the low
nibble first); value = e2m1(code) * 2^(s - 127).

    rows[p] = x[perm[p] div top_k]; place[perm[p]] = p     (and the sum of a token's rows back)
    y[t] = residual[t] + sum_i w[t, i] rows[place[t top_k + i]]
    dlogit of a chosen expert: w_i (dw_i - sum_j w_j dw_j); of any other: 0
    y = residual + act(x W^T + b); gelu is its tanh form
    h = act(x Wg^T + bg, x Wu^T + bu): silu(g) u, or, clamped, with g' = min(g, 7) and
        u' = u between -7 and 7: g' sigmoid(1.702 g') (u' + 1)

A training pass keeps the pre-activations as bf16 values, and its gradients are those at the
values kept.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------- the cases

def listed():
    return [
        # a decode token's row copied to its experts' places: latency
        dict(name="sort_2880_t1", path="sort", t=1, k=4, e=32, c=2880, x="bf16", train=False),
        # a training batch of 4096 tokens, each to eight of 128 experts, and its gradient
        dict(name="sort_train_2048_t4096", path="sort", t=4096, k=8, e=128, c=2048, x="bf16",
             train=True),
        # five decoding sequences' experts summed onto the fp32 residual stream
        dict(name="combine_2880_t5", path="combine", t=5, k=4, e=32, c=2880, x="bf16", y="f32",
             residual=True, train=False),
        # the training batch back to its tokens, then the gradients of rows and weights
        dict(name="combine_train_2048_t4096", path="combine", t=4096, k=8, e=128, c=2048,
             x="bf16", y="bf16", residual=True, train=True),
        # a short prompt's router gradient: latency
        dict(name="route_gradient_t37_e32", path="route", t=37, k=4, e=32),
        # the training batch's
        dict(name="route_gradient_t4096_e128", path="route", t=4096, k=8, e=128),
        # one decode token through a feed-forward layer's first matrix, with bias and GELU
        dict(name="linear_4096x14336_m1", path="linear", m=1, k=4096, n=14336, act="gelu",
             bias=True, residual=False, y="bf16", train=False),
        # the ragged last chunk of a prompt through its second one, onto the fp32 residual
        dict(name="linear_14336x4096_m77", path="linear", m=77, k=14336, n=4096, act="none",
             bias=True, residual=True, y="f32", train=False),
        # a training step of an adapter's base layer with bias and GELU, forward and back
        dict(name="linear_train_4096x14336_m1024", path="linear", m=1024, k=4096, n=14336,
             act="gelu", bias=True, residual=False, y="bf16", train=True),
        # a prefill chunk of 512 tokens through 32 experts' down matrices with biases
        dict(name="experts_linear_2880_t512", path="experts", t=512, top=4, e=32, k=2880,
             n=2880, act="none", y="bf16", train=False),
        # one decode token through four of 32 experts' gated projections with biases
        dict(name="experts_gated_2880_t1", path="gated", t=1, top=4, e=32, k=2880, n=2880,
             act="clamped", bias=True, train=False),
        # a training batch through 128 small experts, forward and back
        dict(name="experts_train_2048x768_t4096", path="gated", t=4096, top=8, e=128, k=2048,
             n=768, act="silu", bias=False, train=True),
    ]


def draw(rng):
    def spread(low, high):  # log-uniform whole number
        return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))

    path = rng.choice(["sort", "combine", "route", "linear", "linear", "experts", "gated",
                       "gated"])
    train = rng.random() < 0.5
    e = spread(4, 256)
    top = rng.randint(1, min(8, e))
    if path == "route":
        return dict(path=path, t=spread(1, 8192), k=top, e=e)
    if path in ("sort", "combine"):
        c = spread(64, 8192)  # odd widths among them
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        case = dict(path=path, t=spread(1, 2 ** 25 // (c * top)), k=top, e=e, c=c, x=x,
                    train=train)
        if path == "combine":
            case.update(y=rng.choice([x, "f32"]), residual=rng.random() < 0.5)
        return case
    k = 32 * spread(8, 448)
    if path == "linear":
        n = 32 * spread(8, 448) if train else spread(256, 16384)
        return dict(path=path, m=spread(1, min(2048, 4 * 10 ** 10 // (k * n))), k=k, n=n,
                    act=rng.choice(["none", "silu", "gelu"]), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.5, y="bf16" if train else rng.choice(["bf16", "f32"]),
                    train=train)
    k = 32 * spread(8, 128)
    n = 32 * spread(8, min(448, 2 * 10 ** 8 // (32 * e * k)))
    t = spread(1, min(4096, 4 * 10 ** 10 // (k * n * top)))
    if path == "experts":
        return dict(path=path, t=t, top=top, e=e, k=k, n=n,
                    act=rng.choice(["none", "silu", "gelu"]), y=rng.choice(["bf16", "f32"]),
                    train=False)
    return dict(path=path, t=t, top=top, e=e, k=k, n=n, act=rng.choice(["silu", "clamped"]),
                bias=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------------- their inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def activations(rows, cols):  # channels of uneven strength, as layer norms leave them
        return normal(rows, cols) * torch.exp(0.5 * normal(cols))

    def stack(count, rows, cols):  # matrices of a trained one's spread, quantised
        blocks = torch.empty(count, rows, cols // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(count, rows, cols // 32, dtype=torch.uint8, device="cuda")
        for i in range(count):
            blocks[i], scales[i] = quantized(normal(rows, cols) * (0.7 / math.sqrt(cols)))
        return blocks, scales

    state = {"case": c}
    if c["path"] == "linear":
        state["x"] = activations(c["m"], c["k"]).bfloat16()
        state["w"] = stack(1, c["n"], c["k"])
        if c["bias"]:
            state["bias"] = 0.3 * normal(1, c["n"])
        if c["residual"]:
            state["residual"] = activations(c["m"], c["n"]).to(TYPES[c["y"]])
        if c["train"]:
            state["dy"] = (0.01 * activations(c["m"], c["n"])).bfloat16()
    else:
        # a router's choices: some experts are more popular than others
        top = c["k"] if c["path"] in ("sort", "combine", "route") else c["top"]
        logits = normal(c["t"], c["e"]) + 0.7 * normal(c["e"])
        chosen, idx = torch.topk(logits, top, dim=1)
        weights = torch.softmax(chosen, dim=1).contiguous()
        flat, perm = torch.sort(idx.reshape(-1), stable=True)
        counts = torch.bincount(flat, minlength=c["e"])
        offsets = torch.zeros(c["e"] + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = torch.cumsum(counts, 0)
        perm = perm.int()
        if c["path"] == "sort":
            state["x"] = activations(c["t"], c["c"]).to(TYPES[c["x"]])
            state["perm"] = perm
            if c["train"]:
                state["drows"] = (0.01 * activations(c["t"] * top, c["c"])).to(TYPES[c["x"]])
        elif c["path"] == "combine":
            state["rows"] = activations(c["t"] * top, c["c"]).to(TYPES[c["x"]])
            state["weights"] = weights
            place = torch.empty_like(perm)
            place[perm.long()] = torch.arange(c["t"] * top, dtype=torch.int32, device="cuda")
            state["place"] = place
            if c["residual"]:
                state["residual"] = activations(c["t"], c["c"]).to(TYPES[c["y"]])
            if c["train"]:
                state["dy"] = (0.01 * activations(c["t"], c["c"])).to(TYPES[c["y"]])
        elif c["path"] == "route":
            state["idx"], state["weights"] = idx.int().contiguous(), weights
            state["dweights"] = 0.1 * normal(c["t"], top)
        else:
            state["x"] = activations(c["t"], c["k"]).bfloat16()[perm.long() // top].contiguous()
            state["offsets"] = offsets
            state["counts"] = counts.tolist()  # (the plain form goes from expert to expert)
            if c["path"] == "experts":
                state["w"] = stack(c["e"], c["n"], c["k"])
                state["bias"] = 0.3 * normal(c["e"], c["n"])
            else:
                state["gate"], state["up"] = (stack(c["e"], c["n"], c["k"]) for _ in range(2))
                if c["bias"]:
                    state["gate_bias"], state["up_bias"] = (0.3 * normal(c["e"], c["n"])
                                                            for _ in range(2))
                if c["train"]:
                    state["dh"] = (0.01 * activations(c["t"] * top, c["n"])).bfloat16()
    if own:  # a program packs its weights once, when it loads them
        from kadan_amd import ops
        for name in ("w", "gate", "up"):
            if name in state:
                blocks, scales = state[name]
                if c["path"] == "linear":
                    blocks, scales = blocks[0], scales[0]
                state[name + "_packed"] = ops.mxfp4_pack(blocks, scales)
                if c["train"]:
                    state[name + "_transposed"] = ops.mxfp4_pack(blocks, scales, transposed=True)
    return state


# ------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return own_pass(state)
    c = state["case"]
    if c["path"] == "sort":
        perm = state["perm"].long()
        rows = state["x"][perm // c["k"]]
        place = torch.empty_like(state["perm"])
        place[perm] = torch.arange(perm.numel(), dtype=torch.int32, device=perm.device)
        if not c["train"]:
            return rows, place
        back = state["drows"].float()[place.long()].reshape(c["t"], c["k"], c["c"])
        return rows, place, back.sum(1).to(TYPES[c["x"]])
    if c["path"] == "combine":
        rows = state["rows"].float()[state["place"].long()].reshape(c["t"], c["k"], c["c"])
        y = (state["weights"].unsqueeze(2) * rows).sum(1)
        if c["residual"]:
            y = y + state["residual"].float()
        y = y.to(TYPES[c["y"]])
        if not c["train"]:
            return y
        dy = state["dy"].float().unsqueeze(1)
        dweights = (dy * rows).sum(2)
        drows = torch.empty_like(state["rows"])
        drows[state["place"].long()] = (state["weights"].unsqueeze(2) * dy).flatten(0, 1).to(
            TYPES[c["x"]])
        return y, drows, dweights
    if c["path"] == "route":
        w, dw = state["weights"], state["dweights"]
        of = w * (dw - (w * dw).sum(1, keepdim=True))
        out = torch.zeros(c["t"], c["e"], device=w.device)
        return out.scatter_(1, state["idx"].long(), of)
    if c["path"] == "gated":
        return plain_gated(state)
    counts = state["counts"] if c["path"] == "experts" else [c["m"]]
    pre = products(state["x"].float(), state["w"], counts)
    if "bias" in state:
        pre = pre + repeated(state["bias"], counts)
    y = activated(pre, c["act"])
    if "residual" in state:
        y = y + state["residual"].float()
    y = y.to(TYPES[c["y"]])
    if not c["train"]:
        return y
    dy = state["dy"].float()
    dpre = dy if c["act"] == "none" else dy * slope(pre.bfloat16().float(), c["act"])
    return y, (dpre @ values(*state["w"])[0]).bfloat16(), dpre.bfloat16()


def own_pass(state):
    from kadan_amd import ops
    c = state["case"]
    if c["path"] == "sort":
        rows, place = ops.moe_sort(state["x"], state["perm"], c["k"])
        if not c["train"]:
            return rows, place
        return rows, place, ops.moe_sort_backward(state["drows"], place, c["k"])
    if c["path"] == "combine":
        y = ops.moe_combine(state["rows"], state["weights"], state["place"],
                            residual=state.get("residual"), dtype=TYPES[c["y"]])
        if not c["train"]:
            return y
        return (y, *ops.moe_combine_backward(state["dy"], state["rows"], state["weights"],
                                             state["place"]))
    if c["path"] == "route":
        return ops.moe_route_backward(state["idx"], state["weights"], state["dweights"], c["e"])
    if c["path"] == "gated":
        more = dict(activation=c["act"])
        h = ops.mxfp4_experts_gated(state["x"], state["offsets"], state["gate_packed"],
                                    state["up_packed"], c["n"], gate_bias=state.get("gate_bias"),
                                    up_bias=state.get("up_bias"),
                                    save="bf16" if c["train"] else None, **more)
        if not c["train"]:
            return h
        h, saved = h
        return (h, *ops.mxfp4_experts_gated_backward(
            state["dh"], state["offsets"], saved, state["gate_transposed"],
            state["up_transposed"], c["k"], **more))
    act = None if c["act"] == "none" else c["act"]
    bias = state.get("bias")
    if c["path"] == "experts":
        return ops.mxfp4_linear(state["x"], state["w_packed"], c["n"], bias=bias, activation=act,
                                dtype=TYPES[c["y"]], offsets=state["offsets"])
    bias = None if bias is None else bias[0]
    y = ops.mxfp4_linear(state["x"], state["w_packed"], c["n"], bias=bias, activation=act,
                         residual=state.get("residual"), dtype=TYPES[c["y"]],
                         save=c["train"] and act is not None)
    if not c["train"]:
        return y
    y, saved = y if act else (y, None)
    return (y, *ops.mxfp4_linear_backward(state["dy"], state["w_transposed"], c["k"], saved=saved,
                                          activation=act))


# ------------------------------------------------------------------------- the plain forms

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values(blocks, scales):
    """MXFP4 matrices (uint8 [count, rows, cols/2] and [count, rows, cols/32]) as fp32."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=blocks.device)
    codes = torch.stack([blocks & 15, blocks >> 4], -1).reshape(*scales.shape, 32)
    return torch.ldexp(table[codes.int()], scales.int().unsqueeze(-1) - 127).flatten(2)


def quantized(x):
    """fp32 [rows, cols] as MXFP4 rows: uint8 [rows, cols/2] and [rows, cols/32]."""
    v = x.reshape(x.shape[0], -1, 32)
    exponent = (torch.frexp(v.abs().amax(-1)).exponent - 3).clamp(min=-127)  # floor(log2) - 2
    v = torch.ldexp(v, -exponent.unsqueeze(-1))
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)  # round() takes ties to the even code
    code = (2 * a.clamp(max=2) + (a.clamp(2, 4) - 2) + (a.clamp(4, 6) - 4) / 2).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).flatten(1)
    return code[:, 0::2] | (code[:, 1::2] << 4), (exponent + 127).to(torch.uint8)


def products(x, matrices, counts, transposed=False):
    """Every row times its expert's matrix (transposed: from the matrix's rows to its columns)."""
    used = [i for i, count in enumerate(counts) if count]
    w = values(matrices[0][used], matrices[1][used])
    parts = [part for part in torch.split(x, counts) if part.shape[0]]
    return torch.cat([part @ (w[i] if transposed else w[i].T) for i, part in enumerate(parts)])


def repeated(bias, counts):
    return torch.cat([bias[i].expand(count, -1) for i, count in enumerate(counts)])


def sigmoid(z):
    return 1 / (1 + torch.exp(-z))


def inner(v, act):
    """z of v sigmoid(z), and its derivative."""
    if act == "silu":
        return v, torch.ones_like(v)
    c = 2 * math.sqrt(2 / math.pi)
    return c * (v + 0.044715 * v * v * v), c * (1 + 3 * 0.044715 * v * v)


def activated(v, act):
    return v if act == "none" else v * sigmoid(inner(v, act)[0])


def slope(v, act):
    z, dz = inner(v, act)
    s = sigmoid(z)
    return s + v * s * (1 - s) * dz


def gate(g, u, act):
    if act == "silu":
        return g * sigmoid(g) * u
    g, u = g.clamp(max=7), u.clamp(-7, 7)
    return g * sigmoid(1.702 * g) * (u + 1)


def gate_slopes(dh, g, u, act):
    if act == "silu":
        s = sigmoid(g)
        return dh * u * (s * (1 + g * (1 - s))), dh * (g * s)
    in_g, in_u = g <= 7, u.abs() <= 7
    g, u = g.clamp(max=7), u.clamp(-7, 7)
    s = sigmoid(1.702 * g)
    return (torch.where(in_g, dh * (u + 1) * (s * (1 + 1.702 * g * (1 - s))), 0.0),
            torch.where(in_u, dh * (g * s), 0.0))


def plain_gated(state):
    c, counts = state["case"], state["counts"]
    x = state["x"].float()
    g, u = products(x, state["gate"], counts), products(x, state["up"], counts)
    if c["bias"]:
        g, u = g + repeated(state["gate_bias"], counts), u + repeated(state["up_bias"], counts)
    h = gate(g, u, c["act"]).bfloat16()
    if not c["train"]:
        return h
    dg, du = gate_slopes(state["dh"].float(), g.bfloat16().float(), u.bfloat16().float(),
                         c["act"])
    dx = (products(dg, state["gate"], counts, transposed=True) +
          products(du, state["up"], counts, transposed=True))
    return h, dx.bfloat16(), torch.cat([dg, du], 1).bfloat16()


# ------------------------------------------------------------------------- what it needs

def work(case):
    c = case
    if c["path"] == "route":
        return {"bytes": 12 * c["t"] * c["k"] + 4 * c["t"] * c["e"], "flops": 4 * c["t"] * c["k"]}
    if c["path"] in ("sort", "combine"):
        tokens, slots = c["t"] * c["c"], c["t"] * c["k"] * c["c"]
        index = 8 * c["t"] * c["k"]
        if c["path"] == "sort":
            once = (tokens + slots) * SIZE[c["x"]] + index
            return {"bytes": once * (2 if c["train"] else 1),
                    "flops": slots if c["train"] else 0}
        size = slots * SIZE[c["x"]] + index + tokens * SIZE[c["y"]] * (2 if c["residual"] else 1)
        if c["train"]:
            size += 2 * slots * SIZE[c["x"]] + tokens * SIZE[c["y"]] + 3 * index // 2
        return {"bytes": size, "flops": 2 * slots * (3 if c["train"] else 1)}
    k, n = c["k"], c["n"]
    if c["path"] == "linear":
        m, matrices = c["m"], 1
    else:  # the experts that T tokens are likely to reach
        m = c["t"] * c["top"]
        matrices = c["e"] * (1 - (1 - c["top"] / c["e"]) ** c["t"])
    weights = matrices * n * k * 17 / 32
    if c["path"] == "gated":
        size = 2 * weights + 2 * m * (k + n)
        if c["train"]:  # pre-activations kept and read, dh read, dg, du and dx written
            size += 2 * m * (2 * n + 2 * n + n + 2 * n + k)
        return {"bytes": int(size), "flops": (8 if c["train"] else 4) * m * n * k}
    size = weights + 2 * m * k + SIZE[c["y"]] * m * n
    if c.get("residual"):
        size += SIZE[c["y"]] * m * n
    if c["train"]:
        kept = 0 if c["act"] == "none" else 2 * n
        size += 2 * m * (kept + n + n + k)
    return {"bytes": int(size), "flops": (4 if c["train"] else 2) * m * n * k}


# ------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["path"] == "sort":
        place = torch.argsort(s["perm"])
        rows = s["x"].repeat_interleave(c["k"], 0)[s["perm"].long()].double()
        if not c["train"]:
            return rows, place.int()
        dx = torch.zeros(c["t"], c["c"], dtype=torch.float64, device="cuda")
        dx.index_add_(0, s["perm"].long() // c["k"], s["drows"].double())
        return rows, place.int(), dx
    if c["path"] == "combine":
        y = torch.zeros(c["t"], c["c"], dtype=torch.float64, device="cuda")
        for i in range(c["k"]):
            y += s["weights"][:, i:i + 1].double() * s["rows"][s["place"][i::c["k"]].long()].double()
        if c["residual"]:
            y += s["residual"].double()
        if not c["train"]:
            return y
        slot = torch.argsort(s["place"])
        dy = s["dy"].double()[slot // c["k"]]
        dweights = torch.empty(c["t"] * c["k"], dtype=torch.float64, device="cuda")
        dweights[slot] = (dy * s["rows"].double()).sum(1)
        return y, dy * s["weights"].reshape(-1, 1).double()[slot], dweights.reshape(c["t"], c["k"])
    if c["path"] == "route":
        w, dw = s["weights"].double(), s["dweights"].double()
        # the Jacobian of the softmax over the chosen logits, row by row
        jacobian = torch.diag_embed(w) - w.unsqueeze(2) * w.unsqueeze(1)
        out = torch.zeros(c["t"], c["e"], dtype=torch.float64, device="cuda")
        return out.scatter(1, s["idx"].long(), (jacobian @ dw.unsqueeze(2)).squeeze(2))
    counts = s["counts"] if c["path"] != "linear" else [c["m"]]
    x = s["x"].double()

    def by_expert(rows, name, transposed=False):
        out, at = [], 0
        for i, count in enumerate(counts):
            if count:
                w = decoded(s[name][0][i], s[name][1][i])
                out.append(rows[at:at + count] @ (w if transposed else w.T))
            at += count
        return torch.cat(out)

    def biased(rows, name):
        of = torch.repeat_interleave(torch.arange(len(counts), device="cuda"),
                                     torch.tensor(counts, device="cuda"))
        return rows + s[name].double()[of] if name in s else rows

    if c["path"] != "gated":
        pre = biased(by_expert(x, "w"), "bias")
        y = activation(pre, c["act"])
        if "residual" in s:
            y = y + s["residual"].double()
        if not c["train"]:
            return y
        dpre = s["dy"].double()
        if c["act"] != "none":
            dpre = dpre * derivative(lambda v: activation(v, c["act"]), pre.bfloat16().double())
        return y, by_expert(dpre, "w", transposed=True), dpre
    g, u = biased(by_expert(x, "gate"), "gate_bias"), biased(by_expert(x, "up"), "up_bias")
    h = gated(g, u, c["act"])
    if not c["train"]:
        return h
    g, u = g.bfloat16().double(), u.bfloat16().double()
    dh = s["dh"].double()
    dg = dh * derivative(lambda v: gated(v, u, c["act"]), g)
    du = dh * derivative(lambda v: gated(g, v, c["act"]), u)
    dx = by_expert(dg, "gate", transposed=True) + by_expert(du, "up", transposed=True)
    return h, dx, torch.cat([dg, du], 1)


def decoded(blocks, scales):
    """float64 [rows, cols] from the bits: sign, two exponent bits, one mantissa bit."""
    out = torch.empty(blocks.shape[0], blocks.shape[1] * 2, dtype=torch.float64,
                      device=blocks.device)
    for half in (0, 1):
        code = (blocks.long() >> (4 * half)) & 15
        e, mantissa, sign = (code >> 1) & 3, code & 1, code >> 3
        magnitude = torch.where(e > 0, (2 + mantissa) * 2.0 ** (e.double() - 2), 0.5 * mantissa)
        out[:, half::2] = torch.where(sign > 0, -magnitude, magnitude)
    return out * (2.0 ** (scales.double() - 127)).repeat_interleave(32, dim=1)


def activation(v, act):
    if act == "none":
        return v
    if act == "silu":
        return torch.nn.functional.silu(v)
    return torch.nn.functional.gelu(v, approximate="tanh")


def gated(g, u, act):
    if act == "silu":
        return torch.nn.functional.silu(g) * u
    g, u = torch.clamp(g, max=7.0), torch.clamp(u, min=-7.0, max=7.0)
    return (u + 1) * g * torch.sigmoid(1.702 * g)


def derivative(f, at):
    """f', element by element, as autograd has it."""
    with torch.enable_grad():
        at = at.detach().requires_grad_(True)
        slope_at, = torch.autograd.grad(f(at).sum(), at)
    return slope_at
