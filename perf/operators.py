"""The MXFP4 operators of a dense layer, as timed cases: quantising rows and reading them
back, products with a packed MXFP4 matrix (bf16 or MXFP4 activations), the gated
feed-forward projection silu(x Wg^T) * (x Wu^T) and its backward pass.

An MXFP4 row holds, per 32 values, one E8M0 byte s and 32 E2M1 codes (two to a byte, the
low nibble first); value = e2m1(code) * 2^(s - 127).  Quantising takes, per 32 values,
s - 127 = floor(log2(largest magnitude)) - 2 (s at least 0) and rounds value / 2^(s - 127)
to the nearest E2M1 value, ties to the even code, magnitudes above 6 to 6.

A case names its path, the sizes m (rows of activations), k (values of a row of x) and n
(rows of the matrix) and, where there is a choice, the types.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------- the cases

def case(name, path, m, k, n, **more):
    return dict(name=name, path=path, m=m, k=k, n=n, **more)


def listed():
    return [
        # the activations of a few decoding sequences quantised and read back: latency
        case("quantize_bf16_4x2880", "quantize", 4, 2880, 0, x="bf16"),
        # an FFN matrix of a float checkpoint quantised and read back to see its error
        case("quantize_f32_14336x4096", "quantize", 14336, 4096, 0, x="f32"),
        # one decode token through an FFN gate or up matrix
        case("product_4096x14336_m1", "product", 1, 4096, 14336, y="bf16"),
        # the ragged last chunk of a prompt through an FFN down matrix, onto an fp32 residual
        case("product_14336x4096_m77", "product", 77, 14336, 4096, y="f32"),
        # a prefill chunk of 512 tokens
        case("product_4096x14336_m512", "product", 512, 4096, 14336, y="bf16"),
        # eight sequences decoding together, their activations in MXFP4
        case("quantized_4096x14336_m8", "quantized", 8, 4096, 14336, y="bf16"),
        # a long prefill with MXFP4 activations: the FP4 matrix rate
        case("quantized_4096x14336_m2048", "quantized", 2048, 4096, 14336, y="bf16"),
        # one decode token through the gated projection
        case("gated_4096x14336_m1", "gated", 1, 4096, 14336),
        # a ragged chunk through a smaller model's
        case("gated_2880x2880_m333", "gated", 333, 2880, 2880),
        # a training step of an adapter's base layer: the projection with its
        # pre-activations kept in 8 bits, then the backward pass from them
        case("train_4096x14336_m2048", "train", 2048, 4096, 14336),
        # the backward pass of a small batch from pre-activations kept in bf16
        case("backward_2048x768_m64", "backward", 64, 2048, 768),
        # and of a long one
        case("backward_4096x14336_m1024", "backward", 1024, 4096, 14336),
    ]


def draw(rng):
    def spread(low, high):  # log-uniform whole number
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    path = rng.choice(["quantize", "product", "product", "quantized", "gated", "train",
                       "backward"])
    k = 32 * spread(16, 448)
    if path == "quantize":
        return dict(path=path, m=spread(1, 2 ** 25 // k), k=k, n=0,
                    x=rng.choice(["bf16", "f16", "f32"]))
    if path in ("product", "quantized"):
        n = spread(256, 16384)
        return dict(path=path, m=spread(1, min(2048, 10 ** 11 // (k * n))), k=k, n=n,
                    y=rng.choice(["bf16", "f32"]))
    n = 32 * spread(16, 448)
    return dict(path=path, m=spread(1, min(2048, 10 ** 11 // (k * n))), k=k, n=n)


# ------------------------------------------------------------------------- their inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def activations(rows, cols):  # channels of uneven strength, as layer norms leave them
        return normal(rows, cols) * torch.exp(0.5 * normal(cols))

    def matrix(rows, cols):  # a trained matrix's spread, quantised
        return quantized(normal(rows, cols) * (0.7 / math.sqrt(cols)))

    state = {"case": c}
    if c["path"] == "quantize":
        state["x"] = activations(c["m"], c["k"]).to(TYPES[c["x"]])
        return state
    if c["path"] in ("product", "quantized"):
        x = activations(c["m"], c["k"]).bfloat16()
        state["x"] = quantized(x.float()) if c["path"] == "quantized" else x
        state["w"] = matrix(c["n"], c["k"])
    else:
        state["gate"], state["up"] = matrix(c["n"], c["k"]), matrix(c["n"], c["k"])
        if c["path"] in ("gated", "train"):
            state["x"] = activations(c["m"], c["k"]).bfloat16()
        if c["path"] in ("backward", "train"):
            state["dh"] = (activations(c["m"], c["n"]) * 0.01).bfloat16()
        if c["path"] == "backward":
            state["saved"] = normal(c["m"], 2 * c["n"]).bfloat16()
    if own:  # a program packs its weights once, when it loads them
        from kadan_amd import ops
        for name in ("w", "gate", "up"):
            if name in state and c["path"] != "backward":
                state[name + "_packed"] = ops.mxfp4_pack(*state[name])
            if name in state and c["path"] in ("backward", "train"):
                state[name + "_transposed"] = ops.mxfp4_pack(*state[name], transposed=True)
    return state


# ------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return own_pass(state)
    c = state["case"]
    if c["path"] == "quantize":
        return values(*quantized(state["x"].float()))
    if c["path"] == "product":
        return (state["x"].float() @ values(*state["w"]).T).to(TYPES[c["y"]])
    if c["path"] == "quantized":
        return (values(*state["x"]) @ values(*state["w"]).T).to(TYPES[c["y"]])
    gate, up = values(*state["gate"]), values(*state["up"])
    if c["path"] == "backward":
        g, u = state["saved"].float().chunk(2, dim=1)
        return plain_backward(state["dh"].float(), g, u, gate, up)
    x = state["x"].float()
    g, u = x @ gate.T, x @ up.T
    h = (g / (1 + torch.exp(-g)) * u).bfloat16()
    if c["path"] == "gated":
        return h
    dx, dgu = plain_backward(state["dh"].float(), eight_bits(g), eight_bits(u), gate, up)
    return h, dx, dgu


def own_pass(state):
    from kadan_amd import ops
    c = state["case"]
    if c["path"] == "quantize":
        return ops.mxfp4_dequantize(*ops.mxfp4_quantize(state["x"]), c["m"], c["k"])
    if c["path"] == "product":
        return ops.mxfp4_product(state["x"], state["w_packed"], c["n"], dtype=TYPES[c["y"]])
    if c["path"] == "quantized":
        return ops.mxfp4_product_quantized(*state["x"], state["w_packed"], c["n"],
                                           dtype=TYPES[c["y"]])
    if c["path"] == "gated":
        return ops.mxfp4_gated(state["x"], state["gate_packed"], state["up_packed"], c["n"])
    if c["path"] == "backward":
        return ops.mxfp4_gated_backward(state["dh"], state["saved"], state["gate_transposed"],
                                        state["up_transposed"], c["k"])
    h, saved = ops.mxfp4_gated(state["x"], state["gate_packed"], state["up_packed"], c["n"],
                               save="q8")
    dx, dgu = ops.mxfp4_gated_backward(state["dh"], saved, state["gate_transposed"],
                                       state["up_transposed"], c["k"])
    return h, dx, dgu


# ------------------------------------------------------------------------- the plain forms

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values(blocks, scales):
    """MXFP4 rows (uint8 [rows, cols/2] and [rows, cols/32]) as fp32 [rows, cols]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=blocks.device)
    codes = torch.stack([blocks & 15, blocks >> 4], -1).reshape(blocks.shape[0], -1, 32)
    return torch.ldexp(table[codes.int()], scales.int().unsqueeze(-1) - 127).flatten(1)


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


def eight_bits(v):
    """fp32 rows through 8 bits: per 32 values the scale is their largest magnitude / 127."""
    b = v.reshape(v.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    q = torch.round(b * torch.where(amax > 0, 127 / amax, 0.0))
    return (q * (amax / 127)).reshape(v.shape)


def plain_backward(dh, g, u, gate, up):
    s = 1 / (1 + torch.exp(-g))
    dg, du = dh * u * (s * (1 + g * (1 - s))), dh * (g * s)
    return (dg @ gate + du @ up).bfloat16(), torch.cat([dg, du], 1).bfloat16()


# ------------------------------------------------------------------------- what it needs

def work(case):
    m, k, n, path = case["m"], case["k"], case["n"], case["path"]
    if path == "quantize":  # read, codes and scales written and read, fp32 written
        return {"bytes": m * k * (SIZE[case["x"]] + 4) + m * k * 17 // 16, "flops": 4 * m * k}
    if path == "product":
        return {"bytes": n * k * 17 // 32 + 2 * m * k + SIZE[case["y"]] * m * n,
                "flops": 2 * m * n * k}
    if path == "quantized":
        return {"bytes": (n + m) * k * 17 // 32 + SIZE[case["y"]] * m * n,
                "flops": 2 * m * n * k}
    weights = 2 * n * k * 17 // 32
    forward = 2 * m * (k + n)               # x read, h written
    backward = 2 * m * (n + 2 * n + k)      # dh read, dg, du and dx written
    if path == "gated":
        return {"bytes": weights + forward, "flops": 4 * m * n * k}
    if path == "backward":
        return {"bytes": weights + backward + 4 * m * n, "flops": 4 * m * n * k}
    kept = 2 * m * n * 9 // 8               # 8 bits a value and a scale per 32
    return {"bytes": weights + forward + backward + 2 * kept, "flops": 8 * m * n * k}


# ------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    path = case["path"]
    if path == "quantize":
        return nearest(s["x"].double())
    if path == "product":
        return s["x"].double() @ decoded(s["w"]).T
    if path == "quantized":
        return decoded(s["x"]) @ decoded(s["w"]).T
    gate, up = decoded(s["gate"]), decoded(s["up"])
    if path == "backward":
        n = case["n"]
        return derivatives(s["dh"].double(), s["saved"][:, :n].double(),
                           s["saved"][:, n:].double(), gate, up)
    g, u = s["x"].double() @ gate.T, s["x"].double() @ up.T
    h = g * torch.sigmoid(g) * u
    if path == "gated":
        return h
    return (h,) + derivatives(s["dh"].double(), in_eight_bits(g), in_eight_bits(u), gate, up)


def decoded(matrix):
    """float64 [rows, cols] from the bits: sign, two exponent bits, one mantissa bit."""
    blocks, scales = matrix
    rows = blocks.shape[0]
    out = torch.empty(rows, blocks.shape[1] * 2, dtype=torch.float64, device=blocks.device)
    for half in (0, 1):
        code = (blocks.long() >> (4 * half)) & 15
        e, mantissa, sign = (code >> 1) & 3, code & 1, code >> 3
        magnitude = torch.where(e > 0, (2 + mantissa) * 2.0 ** (e.double() - 2), 0.5 * mantissa)
        out[:, half::2] = torch.where(sign > 0, -magnitude, magnitude)
    return out * (2.0 ** (scales.double() - 127)).repeat_interleave(32, dim=1)


def nearest(x):
    """The values that quantising x stands for, each found among E2M1's by its distance."""
    level = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    middle = (level[1:] + level[:-1]) / 2
    out = torch.empty_like(x)
    for at in range(0, x.shape[0], 2048):
        b = x[at:at + 2048].reshape(-1, 32)
        top = b.abs().amax(1, keepdim=True)
        scale = 2.0 ** (torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 2).clamp(min=-127)
        a = (b.abs() / scale).contiguous()
        code = torch.bucketize(a, middle)               # a tie stays at the lower level
        tie = (a == middle[code.clamp(max=6)]) & (code < 7)
        code = torch.where(tie & (code % 2 == 1), code + 1, code)  # of two, the even code
        out[at:at + 2048] = (torch.sign(b) * level[code] * scale).reshape(-1, x.shape[1])
    return out


def in_eight_bits(v):
    b = v.reshape(-1, 32)
    d = b.abs().amax(1, keepdim=True) / 127
    return (torch.round(b / d.clamp(min=1e-300)) * d).reshape(v.shape)


def derivatives(dh, g, u, gate, up):
    s = torch.sigmoid(g)
    dgu = torch.cat([dh * u * s * (1 + g - g * s), dh * s * g], dim=1)
    return dgu @ torch.cat([gate, up]), dgu
