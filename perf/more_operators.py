"""4-bit training and serving of the MLP's products, and the experts' layer for a few tokens, as cases that can be
timed and compared.

Four operators, each in a plain torch form (``own`` false) and through the package's entry points (``own`` true):

* ``quant``    microscaled 4-bit codes (32 values of a row, e2m1 each, share one power of two) of a matrix, of its
               transpose or of both, and the values they stand for (``mxfp4_quantize``, ``mxfp4_dequantize``)
* ``matmul``   the product of two matrices held in such codes (``mxfp4_matmul``)
* ``linear``   a linear layer whose product runs on such codes, in training with the gradients of input and weight
               (``mxfp4_linear``)
* ``experts``  a whole mixture-of-experts layer for a few tokens: router, gate and up, SwiGLU, down, weighted sum, from
               bf16 or 4-bit weights (``decode_routed_experts``)
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2, "mxfp4": 17 / 32}  # bytes of an element
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the codes 0 .. 7 stand for; 8 .. 15 are their negatives
LARGEST = {"quant": 65536 * 1024, "matmul": 16384 * 8192 * 4096, "linear": 16384 * 4096 * 2048,
           "experts": 64 * 6 * 2048 * 1032}


def listed():
    return [
        # the benchmark's batch and width, written along rows for a forward product
        {"name": "quant_batch", "kind": "quant", "R": 65536, "C": 1024, "along": "rows", "dtype": "bf16"},
        # a short micro-batch of an odd width, along rows and columns at once, as training needs it
        {"name": "quant_both_ragged", "kind": "quant", "R": 5003, "C": 1001, "along": "both", "dtype": "fp16"},
        # generation, eight sequences at once: a wide projection
        {"name": "matmul_few", "kind": "matmul", "M": 8, "N": 8192, "K": 2048, "dtype": "bf16"},
        # an uneven chunk of a prompt, results in 32 bits
        {"name": "matmul_ragged", "kind": "matmul", "M": 1003, "N": 2050, "K": 1000, "dtype": "fp32"},
        # a large batch through a wide layer
        {"name": "matmul_large", "kind": "matmul", "M": 16384, "N": 8192, "K": 4096, "dtype": "bf16"},
        # generation, four sequences at once, weights kept in 4 bits
        {"name": "linear_decode", "kind": "linear", "T": 4, "K": 4096, "N": 4096, "train": False, "dtype": "bf16"},
        # a training step of one projection from its fp32 master
        {"name": "linear_train", "kind": "linear", "T": 16384, "K": 2048, "N": 4096, "train": True, "dtype": "bf16"},
        # a padded micro-batch of uneven length, sizes that are no multiple of a block
        {"name": "linear_ragged", "kind": "linear", "T": 2003, "K": 1000, "N": 1030, "train": True, "dtype": "bf16"},
        # generation of one sequence, many small experts
        {"name": "experts_one", "kind": "experts", "T": 1, "E": 128, "k": 8, "D": 2048, "I": 768, "weights": "bf16",
         "score": "softmax", "bias": False, "mask": False, "renorm": True, "scale": 1.0},
        # the benchmark's experts, sixteen sequences at once
        {"name": "experts_8x2", "kind": "experts", "T": 16, "E": 8, "k": 2, "D": 1024, "I": 1536, "weights": "bf16",
         "score": "softmax", "bias": False, "mask": False, "renorm": True, "scale": 1.0},
        # weights in 4 bits, sigmoid scores with a bias for balance
        {"name": "experts_4bit", "kind": "experts", "T": 4, "E": 128, "k": 8, "D": 2048, "I": 768, "weights": "mxfp4",
         "score": "sigmoid", "bias": True, "mask": False, "renorm": True, "scale": 2.5},
        # the most tokens, some of them padding, an uneven inner width
        {"name": "experts_many", "kind": "experts", "T": 64, "E": 64, "k": 6, "D": 2048, "I": 1032, "weights": "bf16",
         "score": "softmax", "bias": False, "mask": True, "renorm": False, "scale": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["quant", "matmul", "matmul", "linear", "linear", "experts", "experts"])
    if kind == "quant":
        R = _log(rng, 1, 65536)
        C = _log(rng, 1, min(8192, LARGEST[kind] // R))
        return {"kind": kind, "R": R, "C": C, "along": rng.choice(["rows", "columns", "both"]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "matmul":
        M, K = _log(rng, 1, 16384), _log(rng, 32, 8192)
        return {"kind": kind, "M": M, "K": K, "N": _log(rng, 16, min(8192, LARGEST[kind] // (M * K))),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "linear":
        train = rng.random() < 0.6
        T = _log(rng, 64, 16384) if train else _log(rng, 1, 256)
        K = rng.choice([1, 2, 8, 8]) * _log(rng, 16, 512)
        return {"kind": kind, "T": T, "K": K, "N": _log(rng, 32, min(4096, LARGEST[kind] // (T * K))), "train": train,
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    E = rng.choice([8, 16, 60, 64, 128])
    k = rng.randint(1, 8)
    D, I = 8 * rng.randint(32, 256), 8 * rng.randint(32, 192)
    return {"kind": kind, "T": _log(rng, 1, min(64, LARGEST[kind] // (k * D * I))), "E": E, "k": k, "D": D, "I": I,
            "weights": rng.choice(["bf16", "mxfp4"]), "score": rng.choice(["softmax", "sigmoid"]),
            "bias": rng.random() < 0.4, "mask": rng.random() < 0.3, "renorm": rng.random() < 0.6,
            "scale": rng.choice([1.0, 2.5])}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Activations N(0, 1) with channels that are larger and smaller, weights N(0, 1 / fan-in), upstream gradients
    N(0, 1e-3)."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=dev, generator=gen).mul_(std)

    def activation(rows, width):
        return normal(rows, width) * torch.exp(normal(width, std=0.5))

    kind, v = case["kind"], {}
    if kind == "quant":
        v["x"] = activation(case["R"], case["C"]).to(DTYPES[case["dtype"]])
    elif kind == "matmul":  # both operands as an earlier step or a checkpoint left them, in codes
        v["a"] = _plain_quantize(activation(case["M"], case["K"]))
        v["b"] = _plain_quantize(normal(case["N"], case["K"], std=case["K"] ** -0.5))
    elif kind == "linear":
        v["x"] = activation(case["T"], case["K"]).to(DTYPES[case["dtype"]])
        v["w"] = normal(case["N"], case["K"], std=case["K"] ** -0.5)  # the fp32 master
        if not case["train"]:
            v["w"] = _plain_quantize(v["w"])
        v["dy"] = normal(case["T"], case["N"], std=1e-3).to(DTYPES[case["dtype"]])
    else:
        T, E, D, I = case["T"], case["E"], case["D"], case["I"]
        v["x"] = normal(T, D).to(torch.bfloat16)
        v["router"] = normal(E, D, std=D ** -0.5).to(torch.bfloat16)
        v["w_gu"] = normal(E, 2 * I, D, std=D ** -0.5).to(torch.bfloat16)
        v["w_down"] = normal(E, D, I, std=I ** -0.5).to(torch.bfloat16)
        if case["weights"] == "mxfp4":
            v["w_gu"], v["w_down"] = _plain_quantize(v["w_gu"]), _plain_quantize(v["w_down"])
        v["bias"] = normal(E, std=0.05) if case["bias"] else None
        v["mask"] = torch.rand(T, device=dev, generator=gen) >= 0.125 if case["mask"] else None
    return v


def prepare(case, seed):
    v = _inputs(case, seed)
    v["case"] = case
    v["grid"] = _grid()
    if case["kind"] == "linear" and case["train"]:
        v["x"].requires_grad_(True)
        v["w"].requires_grad_(True)
    return v


def _grid():
    return torch.tensor(GRID + tuple(-g for g in GRID), device="cuda")


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        with torch.no_grad():
            return PLAIN[kind](s, case)
    import spark_gpt_amd as sg

    if kind == "quant":
        q = sg.mxfp4_quantize(s["x"], along=case["along"])
        return [sg.mxfp4_dequantize(one) for one in (q if case["along"] == "both" else (q,))]
    if kind == "matmul":
        a, b = sg.MXFP4(*s["a"], (case["M"], case["K"])), sg.MXFP4(*s["b"], (case["N"], case["K"]))
        return sg.mxfp4_matmul(a, b, dtype=DTYPES[case["dtype"]])
    if kind == "linear":
        if not case["train"]:
            with torch.no_grad():
                return sg.mxfp4_linear(s["x"], sg.MXFP4(*s["w"], (case["N"], case["K"])))
        y = sg.mxfp4_linear(s["x"], s["w"])
        dx, dw = torch.autograd.grad(y, [s["x"], s["w"]], s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    w_gu, w_down = s["w_gu"], s["w_down"]
    if case["weights"] == "mxfp4":
        E, D, I = case["E"], case["D"], case["I"]
        w_gu, w_down = sg.MXFP4(*w_gu, (E, 2 * I, D)), sg.MXFP4(*w_down, (E, D, I))
    with torch.no_grad():
        out, selected = sg.decode_routed_experts(s["x"], s["router"], w_gu, w_down, case["k"], score=case["score"],
                                                 bias=s["bias"], mask=s["mask"], renormalize=case["renorm"],
                                                 scale=case["scale"])
    return {"out": out, "selected": selected}


# ------------------------------------------------------------------ the plain form
def _plain_quantize(x):
    """(codes, scales) of [..., R, C]: the 64 bytes of 128 values of a row side by side for all rows (rounded up to 16),
    [..., C / 128, rows, 64], the lower value in the lower half of a byte, and their four scales [..., C / 128, rows, 4].
    A scale is 2 to the exponent of the block's largest value less 2 (the exponent of the largest code), in an 8-bit
    exponent; values round to nearest, ties to the even code, and what is past 6 becomes 6."""
    R, C = x.shape[-2:]
    S, rows = -(-C // 128), -(-R // 16) * 16
    full = torch.zeros(*x.shape[:-2], rows, S * 128, device=x.device)
    full[..., :R, :C] = x
    v = full.view(*full.shape[:-1], S * 4, 32)
    exponent = v.abs().amax(-1).view(torch.int32) >> 23
    scale = torch.where(exponent == 255, 255, (exponent - 2).clamp(min=0))
    factor = ((254 - scale.clamp(max=252)) << 23).view(torch.float32)[..., None]
    m = v.abs() * factor
    code = ((m > 0.25).byte() + (m >= 0.75).byte() + (m > 1.25).byte() + (m >= 1.75).byte() + (m > 2.5).byte()
            + (m >= 3.5).byte() + (m > 5).byte() + 8 * (v < 0).byte())
    code = code.view(*full.shape[:-1], S, 64, 2)
    code = code[..., 0] + 16 * code[..., 1]  # [..., rows, S, 64]
    scale = scale.to(torch.uint8).view(*full.shape[:-1], S, 4)
    return code.transpose(-3, -2).contiguous(), scale.transpose(-3, -2).contiguous()


def _plain_values(q, R, C, grid):
    """What (codes, scales) stand for, in 32 bits: [..., R, C]."""
    codes, scales = q
    pair = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1)  # [..., S, rows, 64, 2]
    e = scales.int()
    bits = torch.where(e == 255, 0x7FC00000, torch.where(e == 0, 0x00400000, e << 23))
    v = pair.view(*codes.shape[:-1], 4, 32) * bits.view(torch.float32)[..., None]
    v = v.transpose(-4, -3)  # [..., rows, S, 4, 32]
    return v.reshape(*v.shape[:-3], -1)[..., :R, :C]


def _plain_both(x, along):
    return [_plain_quantize(x) if d == "rows" else _plain_quantize(x.t())
            for d in (("rows", "columns") if along == "both" else (along,))]


def _plain_quant(s, case):
    R, C = case["R"], case["C"]
    out = {"rows": [(R, C)], "columns": [(C, R)], "both": [(R, C), (C, R)]}[case["along"]]
    return [_plain_values(q, r, c, s["grid"]).to(torch.bfloat16)
            for q, (r, c) in zip(_plain_both(s["x"], case["along"]), out)]


def _plain_matmul(s, case):
    M, N, K = case["M"], case["N"], case["K"]
    a, b = _plain_values(s["a"], M, K, s["grid"]), _plain_values(s["b"], N, K, s["grid"])
    return (a @ b.t()).to(DTYPES[case["dtype"]])


def _plain_linear(s, case):
    T, N, K, dtype, grid = case["T"], case["N"], case["K"], DTYPES[case["dtype"]], s["grid"]
    x = _plain_values(_plain_quantize(s["x"]), T, K, grid)
    if not case["train"]:
        return (x @ _plain_values(s["w"], N, K, grid).t()).to(dtype)
    y = x @ _plain_values(_plain_quantize(s["w"]), N, K, grid).t()
    # each gradient's product has its own blocks, along the dimension that it sums over
    dy = _plain_values(_plain_quantize(s["dy"]), T, N, grid)
    dx = dy @ _plain_values(_plain_quantize(s["w"].t()), K, N, grid).t()
    dyt = _plain_values(_plain_quantize(s["dy"].t()), N, T, grid)
    dw = dyt @ _plain_values(_plain_quantize(s["x"].t()), K, T, grid).t()
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw}


def _plain_experts(s, case):
    T, E, k, D, I = (case[n] for n in ("T", "E", "k", "D", "I"))
    x = s["x"].float()
    low = s["x"].double() @ s["router"].double().t()  # two scores may differ by less than 32 bits hold
    if case["score"] == "softmax":
        p = torch.exp(low - low.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-low))
    order = low if s["bias"] is None else p + s["bias"].double()
    selected = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
    weights = p.gather(1, selected)
    if case["renorm"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = (case["scale"] * weights).float()
    at = selected.reshape(-1)
    if case["weights"] == "mxfp4":
        w_gu = _plain_values([t[at] for t in s["w_gu"]], 2 * I, D, s["grid"])
        w_down = _plain_values([t[at] for t in s["w_down"]], D, I, s["grid"])
    else:
        w_gu, w_down = s["w_gu"][at].float(), s["w_down"][at].float()
    gu = torch.matmul(w_gu, x.repeat_interleave(k, 0)[:, :, None])[:, :, 0]
    g, u = gu[:, :I], gu[:, I:]
    h = g / (1 + torch.exp(-g)) * u
    rows = torch.matmul(w_down, h[:, :, None]).view(T, k, D)
    if s["mask"] is not None:
        weights = weights * s["mask"][:, None]
        selected = torch.where(s["mask"][:, None], selected, -1)
    return {"out": (rows * weights[:, :, None]).sum(1).to(torch.bfloat16), "selected": selected}


PLAIN = {"quant": _plain_quant, "matmul": _plain_matmul, "linear": _plain_linear, "experts": _plain_experts}


# ------------------------------------------------------------------ what a pass needs
def work(case):
    kind, four = case["kind"], SIZES["mxfp4"]
    if kind == "quant":  # the values in, codes and scales, the values that they stand for
        n = case["R"] * case["C"]
        ways = 2 if case["along"] == "both" else 1
        return {"bytes": n * (SIZES[case["dtype"]] + ways * (four + 2)), "flops": 3.0 * n * ways}
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": four * K * (M + N) + SIZES[case["dtype"]] * M * N, "flops": 2.0 * M * N * K}
    if kind == "linear":
        T, N, K, size = case["T"], case["N"], case["K"], SIZES[case["dtype"]]
        if not case["train"]:
            return {"bytes": size * T * (K + N) + four * N * K, "flops": 2.0 * T * N * K}
        # x, w and dy; y, dx and dw
        return {"bytes": size * T * 2 * (K + N) + 8.0 * N * K, "flops": 6.0 * T * N * K}
    T, E, k, D, I = (case[n] for n in ("T", "E", "k", "D", "I"))
    live = E * (1 - (1 - k / E) ** T)  # experts that some token is expected to take
    return {"bytes": live * 3 * D * I * SIZES[case["weights"]] + 2 * E * D + 4 * T * D + 8 * T * k,
            "flops": 2.0 * T * (3 * k * D * I + E * D)}


# ------------------------------------------------------------------ the same in 64 bits
def _quantized(x):
    """The values that the codes of x's rows stand for, from the definition: 2 ** (floor(log2(largest)) - 2) times the
    nearest of the grid."""
    x = x.double()
    R, C = x.shape[-2:]
    blocks = torch.nn.functional.pad(x, (0, -C % 32)).unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    power = torch.frexp(top).exponent - 3  # top = mantissa * 2 ** exponent, mantissa from 0.5 up
    unit = torch.exp2(power.clamp(min=-127).double())
    v = (blocks / unit).abs()
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(max=6.0)  # torch.round takes ties to even
    return (torch.copysign(v, blocks) * unit).flatten(-2)[..., :C]


def _decoded(q, R, C):
    """The values of given codes, byte by byte."""
    codes, scales = q
    grid = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    out = torch.empty(*codes.shape[:-1], 128, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        nibble = torch.bitwise_right_shift(codes, 4 * half).bitwise_and(15).long()
        out[..., half::2] = grid[nibble % 8] * torch.where(nibble >= 8, -1.0, 1.0)
    out *= torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    return out.movedim(-3, -2).flatten(-2)[..., :R, :C]


def exact(case, seed):
    v, kind = _inputs(case, seed), case["kind"]
    if kind == "quant":
        ways = ("rows", "columns") if case["along"] == "both" else (case["along"],)
        return [_quantized(v["x"] if d == "rows" else v["x"].t()) for d in ways]
    if kind == "matmul":
        return torch.mm(_decoded(v["a"], case["M"], case["K"]), _decoded(v["b"], case["N"], case["K"]).t())
    if kind == "linear":
        if not case["train"]:
            return torch.mm(_quantized(v["x"]), _decoded(v["w"], case["N"], case["K"]).t())
        x, w, dy = v["x"], v["w"], v["dy"]
        return {"y": torch.mm(_quantized(x), _quantized(w).t()), "dx": torch.mm(_quantized(dy), _quantized(w.t()).t()),
                "dw": torch.mm(_quantized(dy.t()), _quantized(x.t()).t())}
    T, k, D, I = (case[n] for n in ("T", "k", "D", "I"))
    low = torch.mm(v["x"].double(), v["router"].double().t())
    logp = torch.log_softmax(low, 1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(low)
    order = low if v["bias"] is None else logp.exp() + v["bias"]
    selected = order.topk(k, dim=1).indices
    picked = logp.gather(1, selected)
    weights = case["scale"] * (torch.softmax(picked, 1) if case["renorm"] else picked.exp())
    out = torch.zeros(T, D, dtype=torch.float64, device=low.device)
    for t in range(T):
        if v["mask"] is not None and not bool(v["mask"][t]):
            continue
        for j, e in enumerate(selected[t].tolist()):
            if case["weights"] == "mxfp4":
                w_gu = _decoded([c[e] for c in v["w_gu"]], 2 * I, D)
                w_down = _decoded([c[e] for c in v["w_down"]], D, I)
            else:
                w_gu, w_down = v["w_gu"][e].double(), v["w_down"][e].double()
            gate, up = torch.mv(w_gu, v["x"][t].double()).chunk(2)
            out[t] += weights[t, j] * torch.mv(w_down, torch.nn.functional.silu(gate) * up)
    return {"out": out, "selected": None}
