"""A mixture-of-experts training step around the experts' products, as cases that can be timed and compared.

Four operators, each in a plain torch form (``own`` false) and through the package's entry points (``own`` true):

* ``route``    scores, selection of the top experts and their weights, and in training the gradient of the logits
               (``route_tokens``)
* ``order``    the rows' order by expert that the experts read (``expert_order``)
* ``combine``  the weighted sum of each token's expert rows, and in training the gradients of rows and weights
               (``combine_experts``)
* ``clip``     the global norm of many gradients and their scaling to a largest norm (``clip_grads``)
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CLIP_EPS = 1e-6  # what a clipped norm is divided by beyond itself
LARGEST = {"route": 65536 * 256, "combine": 65536 * 2 * 1024, "clip": 8 * 3 * 2048 * 6144}


def listed():
    route = {"kind": "route", "mask": False, "groups": 1, "top_groups": 1, "group_best": 1, "bias": False,
             "renorm": True, "scale": 1.0, "score": "softmax", "dtype": "fp32"}
    return [
        # generation, four sequences at once: one token each
        {**route, "name": "route_decode", "T": 4, "E": 64, "k": 6, "train": False},
        # the benchmark's experts, top-2 of 8, at its batch, bf16 logits
        {**route, "name": "route_8x2", "T": 65536, "E": 8, "k": 2, "train": True, "dtype": "bf16"},
        # sigmoid scores with a bias for balance, the best 4 of 8 groups by their two best experts
        {**route, "name": "route_groups", "T": 16384, "E": 256, "k": 8, "train": True, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_best": 2, "scale": 2.5},
        # a short, padded micro-batch, an odd number of experts, the probabilities themselves as weights
        {**route, "name": "route_ragged", "T": 5003, "E": 60, "k": 4, "train": True, "mask": True, "renorm": False,
         "dtype": "bf16"},
        # many small experts at the benchmark's batch
        {**route, "name": "route_256x8", "T": 65536, "E": 256, "k": 8, "train": True},
        # generation: a few tokens of many experts
        {"name": "order_decode", "kind": "order", "T": 8, "E": 128, "k": 8, "mask": False},
        # many small experts at the benchmark's batch
        {"name": "order_256x8", "kind": "order", "T": 65536, "E": 256, "k": 8, "mask": False},
        # generation, eight sequences at once
        {"name": "combine_decode", "kind": "combine", "T": 8, "k": 8, "D": 2048, "E": 64, "train": False,
         "mask": False, "dtype": "bf16"},
        # the benchmark's experts: two rows of each of 65536 tokens
        {"name": "combine_8x2", "kind": "combine", "T": 65536, "k": 2, "D": 1024, "E": 8, "train": True,
         "mask": False, "dtype": "bf16"},
        # a padded micro-batch of uneven length, a width that is no multiple of the wave
        {"name": "combine_ragged", "kind": "combine", "T": 5003, "k": 6, "D": 1000, "E": 60, "train": True,
         "mask": True, "dtype": "bf16"},
        # the weight gradients of 20 layers of the muP base width, below the largest norm, in place
        {"name": "clip_base", "kind": "clip", "layers": 20, "D": 256, "I": 1024, "dtype": "fp32", "over": 0.5,
         "in_place": True},
        # the weight gradients of eight wide layers, scaled down, into the optimizer's own buffers
        {"name": "clip_wide", "kind": "clip", "layers": 8, "D": 2048, "I": 6144, "dtype": "fp32", "over": 3.0,
         "in_place": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "route", "route", "order", "combine", "combine", "clip"])
    if kind == "clip":
        D = 8 * rng.randint(16, 256) + rng.choice([0, 0, 1])
        I = rng.randint(2 * D, 3 * D)
        layers = _log(rng, 1, max(1, min(20, LARGEST[kind] // (3 * D * I))))
        over = rng.choice([0.5, 2.0, 10.0])
        return {"kind": kind, "layers": layers, "D": D, "I": I, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                "over": over, "in_place": over < 1}
    if kind == "combine":
        k, D = rng.randint(1, 8), rng.choice([1, 2, 8, 8, 8]) * _log(rng, 32, 512)
        T = _log(rng, 1, min(65536, LARGEST[kind] // (k * D)))
        return {"kind": kind, "T": T, "k": k, "D": D, "E": rng.choice([8, 60, 128]), "train": T > 64,
                "mask": rng.random() < 0.3, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "order":
        k, E = rng.randint(1, 8), rng.randint(8, 512)
        return {"kind": kind, "T": _log(rng, 1, 65536), "E": E, "k": k, "mask": rng.random() < 0.3}
    groups = rng.choice([1, 1, 1, 2, 4, 6, 8])
    E = groups * rng.randint(-(-8 // groups), 384 // groups)
    top_groups = rng.randint(1, groups)
    k = rng.randint(1, min(8, top_groups * (E // groups)))
    T = _log(rng, 1, min(65536, LARGEST[kind] // E))
    return {"kind": kind, "T": T, "E": E, "k": k, "train": T > 64, "mask": rng.random() < 0.3, "groups": groups,
            "top_groups": top_groups, "group_best": rng.choice([1, 2]) if groups > 1 else 1,
            "bias": rng.random() < 0.4, "renorm": rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]),
            "score": rng.choice(["softmax", "sigmoid"]), "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Logits N(0, 1) with experts that are liked more and less, a bias of the
    size that balance steps reach, rows N(0, 1), upstream gradients N(0, 1e-3)."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=dev, generator=gen).mul_(std)

    kind, v = case["kind"], {}
    if kind == "clip":
        D, I, n = case["D"], case["I"], case["layers"] * (3 * case["D"] * case["I"] + case["D"])
        std = case["over"] / math.sqrt(n)  # the norm comes out as `over` times the largest, which is 1
        shapes = [(2 * I, D), (D, I), (D,)] * case["layers"]
        v["grads"] = [normal(*s, std=std).to(DTYPES[case["dtype"]]) for s in shapes]
        return v
    T, k, E = case["T"], case["k"], case["E"]
    v["mask"] = None
    if case["mask"]:  # the padding of a batch: about an eighth of its tokens
        v["mask"] = torch.rand(T, device=dev, generator=gen) >= 0.125
    if kind == "route":
        v["logits"] = (normal(T, E) + normal(E, std=0.5)).to(DTYPES[case["dtype"]])
        v["bias"] = normal(E, std=0.05) if case["bias"] else None
        v["dw"] = normal(T, k, std=1e-3)
        return v
    chosen = torch.rand(T, E, device=dev, generator=gen).topk(min(k, E), dim=-1).indices
    if v["mask"] is not None:
        chosen = torch.where(v["mask"][:, None], chosen, -1)
    v["selected"] = chosen
    if kind == "combine":
        dtype = DTYPES[case["dtype"]]
        v["inverse"], v["offsets"] = _plain_order(chosen, E)[1:]
        v["rows"] = normal(T * k, case["D"]).to(dtype)
        w = torch.rand(T, k, device=dev, generator=gen) + 0.1
        v["weights"] = w / w.sum(1, keepdim=True)
        if v["mask"] is not None:
            v["weights"] *= v["mask"][:, None]
        v["dout"] = normal(T, case["D"], std=1e-3).to(dtype)
    return v


def prepare(case, seed):
    v = _inputs(case, seed)
    v["case"] = case
    if case["kind"] == "route":
        v["logits"].requires_grad_(case["train"])
    if case["kind"] == "combine":
        v["rows"].requires_grad_(case["train"])
        v["weights"].requires_grad_(case["train"])
    if case["kind"] == "clip":
        v["out"] = None if case["in_place"] else [torch.empty_like(g) for g in v["grads"]]
    return v


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        with torch.no_grad():
            return PLAIN[kind](s, case)
    import spark_gpt_amd as sg

    if kind == "route":
        with torch.set_grad_enabled(case["train"]):
            w, sel = sg.route_tokens(s["logits"], case["k"], score=case["score"], bias=s["bias"], mask=s["mask"],
                                     groups=case["groups"], top_groups=case["top_groups"],
                                     group_best=case["group_best"], renormalize=case["renorm"], scale=case["scale"])
        out = {"weights": w.detach(), "selected": sel}
        if case["train"]:
            out["dlogits"], = torch.autograd.grad(w, [s["logits"]], s["dw"])
        return out
    if kind == "order":
        token_index, inverse, offsets = sg.expert_order(s["selected"], case["E"])
        return {"token_index": token_index, "inverse": inverse, "offsets": offsets}
    if kind == "combine":
        with torch.set_grad_enabled(case["train"]):
            y = sg.combine_experts(s["rows"], s["weights"], s["inverse"], s["offsets"])
        out = {"y": y.detach()}
        if case["train"]:
            out["drows"], out["dweights"] = torch.autograd.grad(y, [s["rows"], s["weights"]], s["dout"])
        return out
    norm = sg.clip_grads(s["grads"], 1.0, out=s["out"])
    return {"norm": norm, "grads": s["grads"] if s["out"] is None else s["out"]}


# ------------------------------------------------------------------ the plain form
def _best(value, n):
    """Indices of the n largest of each row, the lowest first among equals, and
    whether each is there to be taken (a value above -inf)."""
    v, i = torch.sort(value, dim=-1, descending=True, stable=True)
    return i[:, :n], v[:, :n] != -math.inf


def _plain_route(s, case):
    # the order of the experts in 64 bits: two scores may differ by less than 32 bits hold
    low = s["logits"].double()
    T, E = low.shape
    if case["score"] == "softmax":
        p = torch.exp(low - low.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-low))
    there = low != -math.inf
    score = p if s["bias"] is None else p + s["bias"].double()
    value = torch.where(there, low if s["bias"] is None else score, -math.inf)
    if case["groups"] > 1:
        G = case["groups"]
        if case["group_best"] == 1:
            of_group = value.view(T, G, -1).amax(2)
        else:
            two = torch.where(there, score, -math.inf).view(T, G, -1).sort(2, descending=True).values[:, :, :2]
            of_group = torch.where(two[:, :, 0] == -math.inf, -math.inf, two.masked_fill(two == -math.inf, 0).sum(2))
        g, ok = _best(of_group, case["top_groups"])
        keep = torch.zeros(T, G + 1, dtype=torch.bool, device=low.device)
        keep.scatter_(1, torch.where(ok, g, G), True)
        value = torch.where(keep[:, :G].repeat_interleave(E // G, 1), value, -math.inf)
    selected, ok = _best(value, case["k"])
    if s["mask"] is not None:
        ok = ok & s["mask"][:, None]
    at = torch.where(ok, selected, 0)
    chosen = p.gather(1, at).float() * ok
    total = chosen.sum(1, keepdim=True)
    share = chosen / torch.where(total > 0, total, 1) if case["renorm"] else chosen
    out = {"weights": case["scale"] * share, "selected": torch.where(ok, selected, -1)}
    if case["train"]:
        g = case["scale"] * s["dw"] * ok
        if case["renorm"]:
            d = share * (g - (g * share).sum(1, keepdim=True))
            if case["score"] == "sigmoid":
                d = d * (1 - p.gather(1, at)).float()
        elif case["score"] == "sigmoid":
            d = g * chosen * (1 - p.gather(1, at)).float()
        else:
            d = g * chosen
        dl = torch.zeros(T, E, device=low.device).scatter_add_(1, at, d)
        if case["score"] == "softmax" and not case["renorm"]:
            dl -= p.float() * (g * chosen).sum(1, keepdim=True)
        out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _plain_order(selected, E):
    k = selected.shape[1]
    flat = selected.reshape(-1)
    _, permutation = torch.sort(torch.where(flat < 0, E, flat), stable=True)
    inverse = torch.empty_like(permutation)
    inverse[permutation] = torch.arange(permutation.numel(), device=flat.device)
    inverse = torch.where(flat < 0, -1, inverse)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=flat.device)
    counts.scatter_add_(0, torch.where(flat < 0, E, flat), torch.ones_like(flat))
    return permutation // k, inverse, torch.cumsum(counts[:E], 0).to(torch.int32)


def _plain_combine(s, case):
    rows, w = s["rows"].float(), s["weights"]
    T, k = w.shape
    inv = s["inverse"].view(T, k)
    there = inv >= 0
    of_token = rows[inv.clamp(min=0)]  # [T, k, D]
    w = torch.where(there, w, 0)
    out = {"y": (of_token * w[:, :, None]).masked_fill(~there[:, :, None], 0).sum(1).to(s["rows"].dtype)}
    if case["train"]:
        dy = s["dout"].float()
        drows = torch.zeros(T * k + 1, dy.shape[1], device=dy.device)
        at = torch.where(there, inv, T * k).reshape(-1)
        drows[at] = (w[:, :, None] * dy[:, None, :]).reshape(T * k, -1)
        out["drows"] = drows[:-1].to(s["rows"].dtype)
        out["dweights"] = (of_token * dy[:, None, :]).sum(2) * there
    return out


def _plain_clip(s, case):
    # a sum over up to 10^9 squares: in 64 bits
    norm = sum(g.double().square().sum() for g in s["grads"]).sqrt().float()
    c = torch.clamp(1.0 / (norm + CLIP_EPS), max=1.0)
    out = s["grads"] if s["out"] is None else s["out"]
    for g, o in zip(s["grads"], out):
        o.copy_((g.float() * c).to(g.dtype))
    return {"norm": norm, "grads": out}


PLAIN = {"route": _plain_route, "order": lambda s, case: dict(zip(("token_index", "inverse", "offsets"),
                                                                 _plain_order(s["selected"], case["E"]))),
         "combine": _plain_combine, "clip": _plain_clip}


# ------------------------------------------------------------------ what a pass needs
def work(case):
    kind = case["kind"]
    size = 2 if case.get("dtype") in ("bf16", "fp16") else 4
    if kind == "clip":  # each gradient read; written where the norm is above the largest, or elsewhere
        n = case["layers"] * (3 * case["D"] * case["I"] + case["D"])
        return {"bytes": float(size * n * (1 if case["in_place"] and case["over"] < 1 else 2)), "flops": 3.0 * n}
    T, k, E = case["T"], case["k"], case["E"]
    if kind == "order":  # the selection; token_index, inverse_permutation and offsets
        return {"bytes": 24.0 * T * k + 4 * E, "flops": 0.0}
    if kind == "route":  # logits, bias, mask; weights and selection; their gradient and the logits'
        n = size * T * E + (4 * E if case["bias"] else 0) + (T if case["mask"] else 0) + 12 * T * k
        flops = 4.0 * T * E
        if case["train"]:
            n, flops = n + 4 * T * k + size * T * E, 2 * flops
        return {"bytes": float(n), "flops": flops}
    R, D = T * k, case["D"]
    n, flops = size * (R * D + T * D) + 12 * R, 2.0 * R * D
    if case["train"]:  # the rows count once, though forward and backward read them
        n, flops = n + size * (T * D + R * D) + 4 * R, 3 * flops
    return {"bytes": float(n), "flops": flops}


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    v, kind = _inputs(case, seed), case["kind"]
    if kind == "order":
        return None  # whole numbers alone
    if kind == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in v["grads"]]))
        if float(norm) + CLIP_EPS <= 1:
            return {"norm": norm, "grads": [g.double() for g in v["grads"]]}
        return {"norm": norm, "grads": [g.double() / (norm + CLIP_EPS) for g in v["grads"]]}
    if kind == "combine":
        T, k = case["T"], case["k"]
        rows = v["rows"].double().requires_grad_(True)
        w = v["weights"].double().requires_grad_(True)
        y = 0
        for j in range(k):
            at = v["inverse"].view(T, k)[:, j]
            live = (at >= 0).nonzero()[:, 0]
            part = rows.index_select(0, at[live]) * w[live, j, None]
            y = y + torch.zeros(T, case["D"], dtype=torch.float64, device=part.device).index_add(0, live, part)
        out = {"y": y.detach()}
        if case["train"]:
            out["drows"], out["dweights"] = torch.autograd.grad(y, [rows, w], v["dout"].double())
        return out
    # route: log scores, one choice at a time
    low = v["logits"].double().requires_grad_(True)
    T, E = low.shape
    logp = torch.log_softmax(low, 1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(low)
    with torch.no_grad():
        score = logp.exp() + (v["bias"].double() if case["bias"] else 0)
        left = score.clone() if case["bias"] else low.detach().clone()
        if case["groups"] > 1:
            size = E // case["groups"]
            blocks = left if case["group_best"] == 1 else score
            of_group = torch.stack([b.topk(min(case["group_best"], size), 1).values.sum(1)
                                    for b in blocks.split(size, 1)], 1)
            for _ in range(case["groups"] - case["top_groups"]):
                worst = of_group.argmin(1)
                of_group.scatter_(1, worst[:, None], math.inf)
                left.masked_fill_((torch.arange(E, device=low.device) // size)[None] == worst[:, None], -math.inf)
        at = []
        for _ in range(case["k"]):
            first = (left == left.amax(1, keepdim=True)).byte().argmax(1)
            at.append(first)
            left.scatter_(1, first[:, None], -math.inf)
        selected = torch.stack(at, 1)
    picked = logp.gather(1, selected)
    weights = case["scale"] * (torch.softmax(picked, 1) if case["renorm"] else picked.exp())
    if v["mask"] is not None:
        weights = weights * v["mask"][:, None]
        selected = torch.where(v["mask"][:, None], selected, -1)
    out = {"weights": weights.detach(), "selected": None}
    if case["train"]:
        out["dlogits"], = torch.autograd.grad(weights, [low], v["dw"].double())
    return out
