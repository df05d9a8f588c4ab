"""GPU tests of the routing operators against a plain restatement in 64 bits
(oracle/routing.py): selection (equal, ties and borders included), weights and
gradients, the expert order, the combine, and the layer that runs them around
the FP8 experts.

Tolerances.  A score is exp of an argument d = l - max (softmax) or -|l|
(sigmoid): the argument's rounding, the product with log2(e) and that constant
give |d| * 2.5 * 2^-24, exp2 and the reciprocal 2 * 2^-24 each; sums of up to
1024 positive terms in lanes' order 22 * 2^-24, the scale 2^-24.  With D the
largest |d| of the row: (32 + 5 D) * 2^-24 relative, below 2^-100 nothing is
asked.  A gradient is a product of such weights: twice that, of the sum of the
absolute products, and half a step of its type."""
import threading

import pytest
import torch

import spark_gpt_amd as sg
from oracle import routing as O
from spark_gpt_amd import _lib

pytestmark = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
INF, NAN = float("inf"), float("nan")


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _row_tol(low, score):
    x = low.detach().cpu().double()
    x = torch.where(x.isfinite(), x, 0.0)
    span = (x.amax(1, keepdim=True) - x.amin(1, keepdim=True)) if score == "softmax" else x.abs().amax(1, keepdim=True)
    return (32 + 5 * span) * 2.0 ** -24


def _check_weights(w, ref, tol):
    w = w.detach().cpu().double()
    assert torch.equal(w.isnan(), ref.isnan())
    ok = ref.isnan() | ((w - ref).abs() <= tol * ref.abs() + 2.0 ** -100)
    assert ok.all(), (w[~ok][:4], ref[~ok][:4])


def _run(low, k, dw=None, mask=None, bias=None, **kw):
    """route_tokens against the oracle: selection, weights and, with dw, the gradient."""
    leaf = low.detach().requires_grad_(dw is not None)
    w, sel = sg.route_tokens(leaf, k, mask=mask, bias=bias, **kw)
    rw, rsel = O.route(low, k, mask=mask, bias=bias, **kw)
    assert sel.dtype == torch.int64 and torch.equal(sel.cpu(), rsel), kw
    score = kw.get("score", "softmax")
    tol = _row_tol(low, score)
    _check_weights(w, rw, tol)
    if dw is not None:
        d, = torch.autograd.grad(w, leaf, dw)
        kg = {x: kw[x] for x in ("score", "renormalize", "scale") if x in kw}
        rd, size = O.route_grad(low, rsel, dw, **kg)
        assert d.dtype == low.dtype and d.shape == low.shape
        x = d.cpu().double()
        assert torch.equal(x.isnan(), rd.isnan())
        # the smallest step of the type (fp16 has a large one) bounds the rounding of tiny values;
        # a score below 2^-126 is subnormal in 32 bits, off by up to its own size where it is flushed
        # to zero, and a gradient is a score times at most the sum of the row's |g|, or that of two
        tiny = torch.finfo(low.dtype).tiny * torch.finfo(low.dtype).eps
        g = (kw.get("scale", 1.0) * dw.cpu().double()).abs().sum(1, keepdim=True)
        tiny = tiny + 2.0 ** -125 * g
        bound = 2 * tol * size + _half_step(low.dtype) * rd.abs() * (1 + 2.0 ** -8) + tiny
        ok = rd.isnan() | ((x - rd).abs() <= bound)
        assert ok.all(), (x[~ok][:4], rd[~ok][:4], bound[~ok][:4])
    return w, sel


def _logits(dev, T, E, dtype, seed, spread=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(T, E, device=dev, generator=g) * spread + 0.5 * torch.randn(E, device=dev, generator=g)).to(dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 8, 8), (130, 16, 5), (65, 60, 4), (33, 64, 6), (5, 100, 64),
                                   (41, 128, 8), (19, 256, 8), (3, 257, 1), (9, 384, 8), (4, 1000, 10), (2, 1024, 64)])
def test_route_and_gradient(dev, T, E, k, score, renorm, dtype):
    low = _logits(dev, T, E, DTYPES[dtype], T + E)
    dw = torch.randn(T, k, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    _run(low, k, dw, score=score, renormalize=renorm, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,best", [(8, 4, 2), (8, 3, 1), (4, 1, 2), (6, 5, 2), (3, 2, 1), (1, 1, 1),
                                                    (64, 20, 1), (16, 16, 2)])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_route_groups_and_bias(dev, score, groups, top_groups, best, with_bias, dtype):
    T = 70
    for per in (1, 3, 8, 20, 32):
        E = groups * per
        if E > 1024:
            continue
        k = min(8, top_groups * per)
        low = _logits(dev, T, E, DTYPES[dtype], E + best)
        g = torch.Generator(device=dev).manual_seed(E)
        bias = torch.randn(E, device=dev, generator=g) * 0.05 if with_bias else None
        dw = torch.randn(T, k, device=dev, generator=g)
        mask = torch.rand(T, device=dev, generator=g) > 0.2
        _run(low, k, dw, mask=mask, bias=bias, score=score, groups=groups, top_groups=top_groups, group_best=best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups,k", [(1023, 3, 2, 8), (1023, 33, 9, 10), (1000, 20, 7, 64), (1020, 5, 1, 6),
                                                   (1024, 64, 32, 3), (1024, 8, 4, 8), (126, 63, 20, 33), (992, 31, 30, 1)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_route_many_experts_in_groups(dev, score, E, groups, top_groups, k, dtype):
    """Group counts that are no power of two, of up to 1024 experts."""
    low = _logits(dev, 23, E, DTYPES[dtype], E + groups)
    bias = torch.randn(E, device=dev, generator=torch.Generator(device=dev).manual_seed(E)) * 0.05
    for best in (1, 2):
        for b in (None, bias):
            _run(low, k, torch.ones(23, k, device=dev), bias=b, score=score, groups=groups, top_groups=top_groups,
                 group_best=best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(8, 1), (64, 4), (256, 8)])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_route_special_rows(dev, score, E, groups, with_bias, dtype):
    """Rows that are equal, tied, nearly tied, masked by -inf in part, but for
    one expert or whole, NaN and infinite ones, far apart and tiny."""
    k, per = 6, E // groups
    base = torch.randn(E, generator=torch.Generator().manual_seed(E))
    rows = [torch.zeros(E), torch.full((E,), -3.5), base.sign(), base.round()]
    up = torch.full((E,), 1.0)
    up[E // 2:] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0))  # one step of fp32 apart
    rows += [up, torch.where(torch.arange(E) % 3 == 0, up, up.flip(0))]
    x = base.clone()
    x[::2] = -INF
    rows += [x, torch.full((E,), -INF)]
    x = torch.full((E,), -INF)
    x[E - 1] = 0.25
    rows.append(x)
    x = torch.full((E,), -INF)
    x[per - 1:per + 2] = torch.tensor([1.0, -2.0, 1.0])[:len(x[per - 1:per + 2])]
    rows.append(x)
    for at, v in ((3, NAN), (0, INF), (5, -INF)):
        x = base.clone()
        x[at] = v
        rows.append(x)
    x = base.clone()
    x[1], x[2], x[4] = NAN, INF, NAN
    rows += [x, base * 1e4, base * 1e-6, base * 60, base - 200, base + 200, base * 1e-3 + 1]
    x = base.clone()
    x[2] = 3e4
    rows.append(x)
    low = torch.stack(rows).to(dev).to(DTYPES[dtype])
    low = torch.cat([low, low.flip(0), low.flip(1)])
    for bias in ([torch.zeros(E, device=dev), (torch.arange(E, device=dev) % 4) * 0.25] if with_bias else [None]):
        for best in ((1, 2) if groups > 1 else (1,)):
            kw = dict(score=score, groups=groups, top_groups=max(1, groups // 2), group_best=best)
            _run(low, k, None, bias=bias, **kw)
            fine = low.isfinite().all(1) & (low.float().abs().amax(1) < 1e3)
            dw = torch.randn(int(fine.sum()), k, device=dev)
            for renorm in (True, False):
                _run(low[fine], k, dw, bias=bias, renormalize=renorm, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups,k", [(8, 1, 1, 2), (60, 1, 1, 4), (1000, 1, 1, 10), (1023, 33, 9, 10),
                                                   (1000, 20, 7, 64), (126, 63, 20, 33), (96, 3, 2, 8)])
def test_route_tiny_and_huge_differences(dev, score, E, groups, top_groups, k):
    """Rows whose largest difference is subnormal, or so large that its reciprocal is."""
    g = torch.Generator().manual_seed(E + k)
    step = torch.randint(0, 4, (6, E), generator=g).float()
    one = torch.zeros(2, E)
    one[0, E - 1] = one[1, E // 2] = 1.0
    step = torch.cat([step, one])
    low = torch.cat([step * v for v in (2.0 ** -149, 2.0 ** -140, 2.0 ** -128, 2.0 ** -126, 2.0 ** -101, 2.0 ** -99,
                                        2.0 ** 99, 2.0 ** 101, 2.0 ** 125)])
    low = torch.cat([low, low - 2.0 ** 126]).to(dev)
    _run(low, k, score=score, groups=groups, top_groups=top_groups)
    # scores that are all 0, so that biases alone differ, by the smallest steps and the largest
    if score == "sigmoid":
        flat = torch.full((5, E), -1e30, device=dev)
        for v in (2.0 ** -149, 2.0 ** -128, 2.0 ** -101, 2.0 ** 125):
            for best in (1, 2) if groups > 1 else (1,):
                _run(flat, k, bias=step[0].to(dev) * v, score=score, groups=groups, top_groups=top_groups, group_best=best)


def test_route_bias_special(dev):
    """A bias of -inf takes an expert out, +inf puts it first, NaN ranks above."""
    low = _logits(dev, 20, 16, torch.float32, 5)
    bias = torch.zeros(16, device=dev)
    bias[3], bias[7], bias[9] = -INF, INF, INF
    _run(low, 4, torch.ones(20, 4, device=dev), bias=bias, score="sigmoid")
    bias[12] = NAN
    _run(low, 4, bias=bias, score="sigmoid")
    _run(low, 14, bias=torch.full((16,), -INF, device=dev), score="sigmoid")
    _run(low, 4, bias=torch.linspace(-1e6, 1e6, 16, device=dev), score="softmax")


def test_route_close_scores(dev):
    """Biased scores that differ by less than fp32 holds: the order is the 64-bit one."""
    g = torch.Generator(device=dev).manual_seed(2)
    E, T = 64, 256
    low = torch.randn(T, E, device=dev, generator=g)
    # every score within a few 1e-8 of 1/2 (of 1/64), in steps of 2^-30 (2^-34), and biases in
    # steps that have no common measure with them: two experts are the same or differ by more
    # than a twentieth of a step, far above the errors of 64 bits
    low = torch.round(low * 8) * 2.0 ** -28
    steps = torch.randint(-4, 4, (E,), device=dev, generator=g) * 2.0 ** 0.5
    # sums of two such scores do tie: e^a + e^b and e^c + e^d with a + b = c + d differ by 2^-57 of
    # themselves at these sizes, which 64 bits (2^-53) do not hold.  For sums the logits are
    # continuous: two of them come within 2^-41 in a thousand borders, 2^12 times what 64 bits hold
    loose = torch.randn(T, E, device=dev, generator=g) * 2.0 ** -26
    for groups, best in ((1, 1), (8, 1), (8, 2)):
        x = low if best == 1 else loose
        kw = dict(groups=groups, top_groups=max(1, groups // 2), group_best=best)
        _run(x, 8, bias=steps * 2.0 ** -31, score="sigmoid", **kw)
        _run(x, 8, bias=steps * 2.0 ** -35, score="softmax", **kw)
        _run(x, 8, torch.ones(T, 8, device=dev), score="softmax", **kw)
    far = torch.randn(T, E, device=dev, generator=g) * 1e-3 + 20.0  # 1 - s of about 2e-9
    _run(far, 8, bias=torch.zeros(E, device=dev), score="sigmoid")
    _run(far, 8, score="sigmoid")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(64, 2), (60, 3), (256, 8), (1000, 10)])
@pytest.mark.parametrize("mixed", [False, True])
def test_route_neighbours_of_many_equal_experts(dev, score, E, k, mixed):
    """k - 1 clear winners, many experts with one logit and bias, and one whose
    other logit and bias give the same biased score but for about 1e-9 either
    way: fewer than 32 bits hold, a hundred times what 64 bits do and more.  `mixed`:
    between the rows are some with hardly an expert."""
    g = torch.Generator().manual_seed(E + k)
    T, win = 96, [7 + 2 * j for j in range(k - 1)]
    down = 0.19 if score == "sigmoid" else 0.25 / E
    for at in (0, 1, E // 2, E - 1):
        x = (0.8 + 0.2 * torch.rand(T, generator=g)).float()
        low = x[:, None].repeat(1, E)
        low[:, win] = 3.0 + 0.02 * torch.arange(k - 1)
        bias = torch.full((E,), -0.037174962)
        bias[at] = bias[at] + down
        b = bias.double()
        drop = b[at] - b[at - 1]
        xd = x.double()
        if score == "sigmoid":
            p = torch.sigmoid(xd) - drop
            y = torch.log(p / (1 - p))
        else:
            y = xd.clone()
            top = float(low[0, win].max())
            fixed = torch.exp(low[0, win].double() - top).sum()
            for _ in range(60):  # e^(y - top) = e^(x - top) - drop * z, z the row's sum
                z = fixed + (E - k) * torch.exp(xd - top) + torch.exp(y - top)
                y = top + torch.log(torch.exp(xd - top) - drop * z)
        low[:, at] = y.float()
        if mixed:
            low[::3] = -INF
            low[::3, E - 2] = 1.0
        _run(low.to(dev), k, torch.ones(T, k, device=dev), bias=bias.to(dev), score=score)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_route_strides(dev, dtype):
    """Any row stride and offset, a transposed view, an expanded row, no tokens."""
    big = _logits(dev, 40, 77, DTYPES[dtype], 11)
    dw = torch.randn(40, 3, device=dev)
    for low in (big[:, 5:69], big[:, 1:65], big[:, :64]):
        _run(low, 3, dw)
        _run(low, 3, dw, renormalize=False)
    _run(big[::2, 3:35], 3, dw[::2])
    _run(big.t(), 3, torch.randn(77, 3, device=dev))
    _run(big[:1, :64].expand(9, 64), 3, dw[:9], renormalize=False)
    w, sel = sg.route_tokens(big[:0], 2)
    assert w.shape == sel.shape == (0, 2)
    leaf = big[:0].detach().requires_grad_(True)
    d, = torch.autograd.grad(sg.route_tokens(leaf, 2)[0].sum(), leaf)
    assert d.shape == (0, 77)


def test_route_deterministic_and_large(dev):
    """Twice the same bits; token counts past one pass of the chip against a
    second call on parts of the rows."""
    for T, E, k, kw in ((70001, 8, 2, {}), (50001, 64, 6, dict(score="sigmoid")),
                        (30001, 256, 8, dict(score="sigmoid", groups=8, top_groups=4, group_best=2,
                                             bias=torch.linspace(-0.1, 0.1, 256, device=dev)))):
        low = _logits(dev, T, E, torch.float32, T).requires_grad_(True)
        dw = torch.randn(T, k, device=dev)
        w, sel = sg.route_tokens(low, k, **kw)
        d, = torch.autograd.grad(w, low, dw)
        w2, sel2 = sg.route_tokens(low, k, **kw)
        assert torch.equal(w, w2) and torch.equal(sel, sel2)
        for a, b in ((0, 100), (T // 2, T // 2 + 333), (T - 50, T)):
            part = low.detach()[a:b].clone().requires_grad_(True)
            pw, psel = sg.route_tokens(part, k, **kw)
            pd, = torch.autograd.grad(pw, part, dw[a:b])
            assert torch.equal(psel, sel[a:b]) and torch.equal(pw, w[a:b]) and torch.equal(pd, d[a:b])
        _run(low.detach()[-64:], k, dw[-64:], **kw)


def test_route_refusals(dev):
    low = torch.zeros(4, 12, device=dev)
    one = torch.ones(12, device=dev)
    for kw in (dict(score="tanh"), dict(groups=5), dict(groups=0), dict(groups=3, top_groups=4), dict(top_groups=0),
               dict(group_best=3), dict(bias=one.double()), dict(bias=one[:5]), dict(bias=one.cpu()),
               dict(mask=torch.ones(5, dtype=torch.bool, device=dev)), dict(mask=torch.ones(4, device=dev)),
               dict(mask=torch.ones(4, dtype=torch.bool)), dict(groups=4, top_groups=1)):
        with pytest.raises(ValueError):
            sg.route_tokens(low, 4, **kw)
    for bad, k in ((low, 0), (low, 13), (low[0], 1), (low.double(), 1), (torch.zeros(2, 1025, device=dev), 1),
                   (torch.zeros(2, 0, device=dev), 1), (torch.zeros(2, 128, device=dev), 65)):
        with pytest.raises(ValueError):
            sg.route_tokens(bad, k)
    sel = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    for args in ((sel.int(), 8), (sel[0], 8), (sel, 0), (sel, 1025), (sel[:, :0], 8)):
        with pytest.raises(ValueError):
            sg.expert_order(*args)
    rows, w, inv = torch.zeros(8, 16, device=dev), torch.zeros(4, 2, device=dev), sel.view(-1)
    off = torch.zeros(8, dtype=torch.int32, device=dev)
    for args in ((rows.double(), w, inv, off), (rows, w, inv[:-1], off), (rows, w, inv.int(), off),
                 (rows[0], w, inv, off), (rows[:, :0], w, inv, off), (rows, w.cpu(), inv, off)):
        with pytest.raises(ValueError):
            sg.combine_experts(*args)
    with pytest.raises(ValueError):
        sg.ops.moe_combine_bwd(rows[:4], rows, w, inv, off.long())
    with pytest.raises(ValueError):
        sg.ops.moe_combine_bwd(rows, rows, w, inv, off)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ expert order
@pytest.mark.parametrize("T,k,E", [(0, 2, 8), (1, 1, 1), (1, 8, 128), (8, 8, 128), (63, 3, 7), (1000, 2, 8), (4096, 1, 1),
                                   (4097, 1, 3), (5003, 6, 60), (9001, 8, 256), (2049, 4, 1023), (3000, 7, 1024)])
@pytest.mark.parametrize("fill", ["random", "some unrouted", "one expert", "none"])
def test_expert_order(dev, T, k, E, fill):
    g = torch.Generator().manual_seed(T + E)
    sel = torch.randint(0, E, (T, k), generator=g)
    if fill == "some unrouted":
        sel[torch.rand(T, k, generator=g) < 0.2] = -1
        sel[torch.rand(T, k, generator=g) < 0.05] = E + 3
        sel[torch.rand(T, k, generator=g) < 0.05] = -(2 ** 40)
    elif fill == "one expert":
        sel[:] = E - 1
    elif fill == "none":
        sel[:] = -1
    got = sg.expert_order(sel.to(dev), E)
    for name, a, b in zip(("token_index", "inverse", "offsets"), got, O.expert_order(sel, E)):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), name


def test_expert_order_large_matches_sort(dev):
    """More slots than one pass of the work-groups, against torch's stable sort."""
    T, k, E = 300007, 5, 200
    sel = torch.randint(-1, E, (T, k), device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    tok, inv, off = sg.expert_order(sel, E)
    flat = sel.view(-1).cpu()
    key = torch.where(flat < 0, E, flat)
    order = torch.sort(key, stable=True).indices
    assert torch.equal(tok.cpu(), order // k)
    want = torch.empty_like(order)
    want[order] = torch.arange(T * k)
    assert torch.equal(inv.cpu(), torch.where(flat < 0, -1, want))
    assert torch.equal(off.cpu(), torch.cumsum(torch.bincount(key, minlength=E + 1)[:E], 0).int())


# ------------------------------------------------------------------ combine
def _sum_steps(n):
    """Roundings on the way of one product through a sum of n terms spread over
    the lanes of a wave: its lane's chain and the tree."""
    return n / 16 + 24


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,k,D", [(1, 1, 1), (1, 8, 2048), (5, 2, 7), (64, 2, 8), (33, 6, 1000), (50, 3, 130), (9, 8, 4096),
                                   (17, 64, 24), (300, 2, 256), (12, 4, 5003)])
@pytest.mark.parametrize("unrouted", [False, True])
def test_combine_and_gradients(dev, T, k, D, dtype, unrouted):
    g = torch.Generator().manual_seed(T * k + D)
    E, dt = 16, DTYPES[dtype]
    sel = torch.randint(0, E, (T, k), generator=g)
    if unrouted:
        sel[torch.rand(T, k, generator=g) < 0.3] = -1
    _, inv, off = O.expert_order(sel, E)
    rows = torch.randn(T * k, D, generator=g).to(dt)
    n = int(off[-1])
    rows[n:] = NAN  # what no slot names is not read
    w = torch.rand(T, k, generator=g)
    w[sel < 0] = NAN if unrouted else 0.0
    dout = torch.randn(T, D, generator=g).to(dt)
    r, ww = rows.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = sg.combine_experts(r, ww, inv.to(dev), off.to(dev))
    dr, dw = torch.autograd.grad(y, [r, ww], dout.to(dev))
    step, tiny = _half_step(dt), torch.finfo(dt).tiny * torch.finfo(dt).eps
    ref, size = O.combine(rows, w, inv)
    assert y.dtype == dt and ((y.cpu().double() - ref).abs()
                              <= (k + 1) * 2.0 ** -24 * size + step * (1 + 2.0 ** -8) * ref.abs() + tiny).all()
    rdr, rdw, dsize = O.combine_grad(dout, rows, w, inv)
    assert dr.dtype == dt and ((dr.cpu().double() - rdr).abs() <= (2.0 ** -24 + step * 1.01) * rdr.abs() + tiny).all()
    assert (dr[n:] == 0).all()
    assert dw.dtype == torch.float32
    assert ((dw.cpu().double() - rdw).abs() <= _sum_steps(D) * 2.0 ** -24 * dsize + 2.0 ** -120).all()


def test_combine_layouts(dev):
    """Rows at an odd offset of their storage, strided views, bf16 weights, one
    gradient alone, row indices beyond the rows, no tokens."""
    g = torch.Generator(device=dev).manual_seed(8)
    T, k, D, E = 40, 2, 64, 4
    sel = torch.randint(0, E, (T, k), device=dev, generator=g)
    _, inv, off = sg.expert_order(sel, E)
    store = torch.randn(T * k * D + 1, device=dev, generator=g).to(torch.bfloat16)
    w = torch.rand(T, k, device=dev, generator=g)
    odd = store[1:].view(T * k, D)
    want = sg.combine_experts(odd.clone(), w, inv, off)
    assert torch.equal(sg.combine_experts(odd, w, inv, off), want)
    wide = torch.randn(T * k, 2 * D, device=dev, generator=g).to(torch.bfloat16)
    assert torch.equal(sg.combine_experts(wide[:, ::2], w, inv, off), sg.combine_experts(wide[:, ::2].clone(), w, inv, off))
    wb = w.to(torch.bfloat16).requires_grad_(True)
    y = sg.combine_experts(odd, wb, inv, off)
    gw, = torch.autograd.grad(y, wb, torch.ones_like(y))
    assert gw.dtype == torch.bfloat16 and torch.equal(y, sg.combine_experts(odd, wb.float(), inv, off))
    dout = torch.randn(T, D, device=dev, generator=g).to(torch.bfloat16)
    dr, dw = sg.ops.moe_combine_bwd(dout, odd, w, inv, off)
    only, none = sg.ops.moe_combine_bwd(dout, odd, w, inv, off, True, False)
    assert none is None and torch.equal(only, dr)
    none, only = sg.ops.moe_combine_bwd(dout, odd, w, inv, off, False, True)
    assert none is None and torch.equal(only, dw)
    far = inv.clone()
    far[::3] = T * k + 5
    want, size = O.combine(odd, torch.where((far < T * k).view(T, k), w, 0.0), torch.where(far < T * k, far, -1))
    got = sg.combine_experts(odd, w, far, off).cpu().double()
    assert ((got - want).abs() <= 3 * 2.0 ** -24 * size + 2.0 ** -8 * 1.01 * want.abs()).all()
    empty = sg.combine_experts(odd[:0], w[:0], inv[:0], torch.zeros(E, dtype=torch.int32, device=dev))
    assert empty.shape == (0, D)


def _any_slots(T, k, how, g):
    """inverse_permutation of T * k slots over T * k rows, changed after the order was made."""
    R = T * k
    inv = torch.randperm(R, generator=g)
    if how == "dropped":
        inv[torch.rand(R, generator=g) < 0.3] = -1
    elif how == "out of range":
        inv[torch.rand(R, generator=g) < 0.3] = R + 2
        inv[torch.rand(R, generator=g) < 0.1] = -(2 ** 40)
    elif how == "shared":
        inv[torch.rand(R, generator=g) < 0.4] = inv[0].clone()
        inv[torch.rand(R, generator=g) < 0.2] = inv[-1].clone()
        inv[torch.rand(R, generator=g) < 0.2] = -1
    elif how == "two each":
        inv //= 2
    elif how == "one row":
        inv[:] = R - 1
    elif how == "none":
        inv[:] = -1
    return inv


def _any_slots_reference(dout, rows, weights, inv):
    """(drows, sum of the absolute products, most slots of a row) in float64."""
    R, (T, k) = rows.shape[0], weights.shape
    live = ((inv >= 0) & (inv < R)).nonzero()[:, 0]
    part = weights.double().view(-1)[live, None] * dout.double()[live // k]
    zero = torch.zeros(rows.shape, dtype=torch.float64)
    n = int(torch.bincount(inv[live], minlength=1).max())
    return zero.index_add(0, inv[live], part), zero.index_add(0, inv[live], part.abs()), n


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("how", ["dropped", "out of range", "shared", "two each", "one row", "none"])
@pytest.mark.parametrize("T,k,D", [(1, 2, 1), (40, 3, 5), (200, 1, 24), (33, 64, 8), (70, 6, 130), (300, 4, 64), (21, 2, 1500)])
def test_combine_gradients_of_any_slots(dev, dtype, how, T, k, D):
    """Whatever rows the slots name: a row that no slot names gets zeros, one that
    several name the sum of theirs in slot order (n products and sums in 32 bits,
    2^-24 each, rounded once), the same bits from call to call."""
    dt, R = DTYPES[dtype], T * k
    g = torch.Generator().manual_seed(R + D)
    inv = _any_slots(T, k, how, g)
    rows, dout = torch.randn(R, D, generator=g).to(dt), torch.randn(T, D, generator=g).to(dt)
    w = torch.rand(T, k, generator=g)
    off = torch.full((4,), R, dtype=torch.int32, device=dev)
    args = [x.to(dev) for x in (dout, rows, w, inv)]
    want, size, n = _any_slots_reference(dout, rows, w, inv)
    step, tiny = _half_step(dt), torch.finfo(dt).tiny * torch.finfo(dt).eps
    first = None
    for _ in range(3):
        stale = torch.full((R, D), NAN, device=dev, dtype=dt)  # what a gradient's memory may hold
        del stale
        leaf = args[1].clone().requires_grad_(True)
        y = sg.combine_experts(leaf, args[2], args[3], off)
        got, = torch.autograd.grad(y, leaf, args[0])
        bound = n * 2.0 ** -24 * size + step * (1 + 2.0 ** -8) * want.abs() + tiny
        assert ((got.cpu().double() - want).abs() <= bound).all()
        first = got if first is None else first
        assert torch.equal(got, first)
    _, dw = sg.ops.moe_combine_bwd(*args, off, False, True)
    there = (inv >= 0) & (inv < R)
    dots = torch.where(there[:, None], rows.double()[inv.where(there, torch.zeros_like(inv))], 0.0) \
        * dout.double().repeat_interleave(k, 0)
    assert ((dw.cpu().double().view(-1) - dots.sum(1)).abs()
            <= _sum_steps(D) * 2.0 ** -24 * dots.abs().sum(1) + 2.0 ** -120).all()


def test_combine_gradients_whatever_the_workspace_holds(dev):
    """The C entries: the workspace's contents do not matter, slots in a proper
    order get the same bits from both, and what lies behind the workspace stays."""
    T, k, D = 150, 4, 72
    R, g = T * k, torch.Generator().manual_seed(5)
    rows, dout = torch.randn(R, D, generator=g).to(dev), torch.randn(T, D, generator=g).to(dev)
    w = torch.rand(T, k, generator=g).to(dev)
    ints = _lib.query("sfp8_moe_combine_bwd_any_workspace_ints", R, T, k)
    st = torch.cuda.current_stream().cuda_stream

    def any_slots(inv, ws):
        dr, dw = torch.full_like(rows, NAN), torch.full_like(w, NAN)
        _lib.call("sfp8_moe_combine_bwd_any", dout.data_ptr(), rows.data_ptr(), 0, R, D, w.data_ptr(), inv.data_ptr(), T,
                  k, dr.data_ptr(), dw.data_ptr(), ws.data_ptr(), ints, st)
        assert bool((ws[ints:] == 77).all())
        return dr, dw

    for how in ("order", "dropped", "shared", "two each", "one row", "none"):
        if how == "order":
            sel = torch.randint(-1, 8, (T, k), generator=g).to(dev)
            _, inv, off = sg.expert_order(sel, 8)
        else:
            inv = _any_slots(T, k, how, g).to(dev)
        outs = []
        for fill in ("zeros", "ones", "stale", "slots", "again"):
            if fill != "again":
                ws = torch.full((ints + 8,), 77, dtype=torch.int32, device=dev)
                ws[:ints] = {"zeros": 0, "ones": -1}.get(fill, 0)
            if fill == "stale":
                ws[:ints] = torch.randint(-2 ** 31, 2 ** 31 - 1, (ints,), generator=g).to(dev)
            elif fill == "slots":  # each row's first slot, where it has one
                for s in reversed(range(R)):
                    r = int(inv[s])
                    if 0 <= r < R:
                        ws[r] = s
            outs.append(any_slots(inv, ws))
        assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0])), how
        if how == "order":
            dr, dw = torch.full_like(rows, NAN), torch.full_like(w, NAN)
            _lib.call("sfp8_moe_combine_bwd", dout.data_ptr(), rows.data_ptr(), 0, R, D, w.data_ptr(), inv.data_ptr(), T,
                      k, off.data_ptr(), 8, dr.data_ptr(), dw.data_ptr(), st)
            assert torch.equal(dr, outs[0][0]) and torch.equal(dw, outs[0][1])
        want, size, n = _any_slots_reference(dout.cpu(), rows.cpu(), w.cpu(), inv.cpu())
        assert ((outs[0][0].cpu().double() - want).abs() <= (n + 1) * 2.0 ** -24 * size).all()


def test_combine_gradients_of_any_slots_captured(dev):
    """Captured with slots of one kind and replayed with those of others: the
    workspace then holds what the replay before left."""
    T, k, D = 90, 3, 136
    R, g = T * k, torch.Generator().manual_seed(6)
    rows, dout = torch.randn(R, D, generator=g).to(dev), torch.randn(T, D, generator=g).to(dev)
    w, off = torch.rand(T, k, generator=g).to(dev), torch.full((1,), R, dtype=torch.int32, device=dev)
    inv = _any_slots(T, k, "dropped", g).to(dev)
    sg.ops.moe_combine_bwd(dout, rows, w, inv, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sg.ops.moe_combine_bwd(dout, rows, w, inv, off)
    for how in ("shared", "none", "one row", "two each", "dropped", "shared", "dropped"):
        inv.copy_(_any_slots(T, k, how, g))
        graph.replay()
        want = sg.ops.moe_combine_bwd(dout, rows, w, inv, off)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), how


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_combine_beyond_the_last_level_cache(dev, dtype):
    """Rows beyond the caches, which are read another way: the same bits as in parts."""
    T, k, D, E = (70001, 2, 1024, 8) if dtype == "bf16" else (20001, 3, 1280, 8)
    g = torch.Generator(device=dev).manual_seed(3)
    sel = torch.randint(-1, E, (T, k), device=dev, generator=g)
    _, inv, off = sg.expert_order(sel, E)
    rows = torch.randn(T * k, D, device=dev, generator=g).to(DTYPES[dtype])
    w, dout = torch.rand(T, k, device=dev, generator=g), torch.randn(T, D, device=dev, generator=g).to(DTYPES[dtype])
    assert rows.numel() * rows.element_size() > 256 << 20
    y = sg.ops.moe_combine(rows, w, inv)
    dr, dw = sg.ops.moe_combine_bwd(dout, rows, w, inv, off)
    n = int(off[-1])
    assert 0 < n < T * k and bool((dr[n:] == 0).all())
    for a in range(0, T, 9000):
        b = min(a + 9000, T)
        part = inv[a * k:b * k]
        own = part[part >= 0]
        few = rows[own].contiguous()  # the rows of these tokens alone
        pinv = torch.full_like(part, -1)
        pinv[part >= 0] = torch.arange(own.numel(), device=dev)
        assert torch.equal(sg.ops.moe_combine(few, w[a:b], pinv), y[a:b])
        poff = torch.tensor([own.numel()], dtype=torch.int32, device=dev)
        pdr, pdw = sg.ops.moe_combine_bwd(dout[a:b], few, w[a:b], pinv, poff)
        assert torch.equal(pdr, dr[own]) and torch.equal(pdw, dw[a:b])


# ------------------------------------------------------------------ together
class _Experts(torch.nn.Module):
    def __init__(self, E, D, I, dev, seed=0):
        super().__init__()
        g = torch.Generator(device=dev).manual_seed(seed)
        self.gate_up_proj = torch.nn.Parameter(torch.randn(E, 2 * I, D, device=dev, generator=g) * D ** -0.5)
        self.down_proj = torch.nn.Parameter(torch.randn(E, D, I, device=dev, generator=g) * I ** -0.5)
        self.register_buffer("fp8_scale", torch.ones(5, device=dev), persistent=False)
        self.register_buffer("fp8_amax", torch.zeros(5, device=dev), persistent=False)


@pytest.mark.parametrize("padded", [False, True])
def test_routed_layer_matches_its_parts(dev, padded):
    """fp8_routed_experts, forward and backward, against torch's sort and
    products around _FP8Experts on the same scales: the rows, and so dx and the
    experts' gradients, are equal to the bit; a padded batch gives its valid
    tokens what they get without the padding."""
    T, D, I, E, k = 600, 256, 384, 8, 2
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(T, D, device=dev, generator=g).to(torch.bfloat16)
    low = torch.randn(T, E, device=dev, generator=g)
    low[:, 5] = -INF  # an expert that nothing reaches
    dout = (torch.randn(T, D, device=dev, generator=g) * 1e-3).to(torch.bfloat16)
    mask = (torch.arange(T, device=dev) % 5 != 0) if padded else None
    m = _Experts(E, D, I, dev).train()
    m.fp8_scale.copy_(torch.tensor([32.0, 32, 16, 2.0 ** 20, 2.0 ** 20], device=dev))
    xx, ll = x.clone().requires_grad_(True), low.clone().requires_grad_(True)
    y, sel = sg.fp8_routed_experts(xx, ll, m, k, mask=mask)
    params = [m.gate_up_proj, m.down_proj]
    dx, dl, dgu, dd = torch.autograd.grad(y, [xx, ll] + params, dout)
    amax = m.fp8_amax.clone()

    # the same on the valid tokens alone, in torch around the experts
    keep = mask if padded else torch.ones(T, dtype=torch.bool, device=dev)
    n = int(keep.sum())
    m.fp8_amax.zero_()
    xv, lv = x[keep].clone().requires_grad_(True), low[keep].double().requires_grad_(True)
    p = torch.softmax(lv, 1)
    want_sel = torch.sort(low[keep], dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(sel[keep], want_sel) and bool((sel[~keep] == -1).all())
    w = p.gather(1, want_sel)
    w = w / w.sum(1, keepdim=True)
    flat = want_sel.reshape(-1)
    perm = torch.sort(flat, stable=True).indices
    inv = torch.empty_like(perm)
    inv[perm] = torch.arange(n * k, device=dev)
    off = torch.cumsum(torch.bincount(flat, minlength=E), 0).int()
    rows = sg._FP8Experts.apply(xv, m.gate_up_proj, m.down_proj, perm // k, inv, off, k, m.fp8_scale, m.fp8_amax)
    yv = (rows.double()[inv].view(n, k, D) * w[:, :, None]).sum(1)
    # k products and sums in 32 bits of weights within (32 + 5 * 8) 2^-24, rounded to bf16
    size = (rows.double()[inv].view(n, k, D) * w[:, :, None]).abs().sum(1)
    assert ((y[keep].double() - yv).abs() <= 76 * 2.0 ** -24 * size + 2.0 ** -8 * 1.01 * yv.abs()).all()
    assert bool((y[~keep] == 0).all())
    drows = torch.empty_like(rows)
    w32 = sg.route_tokens(low[keep], k)[0]
    drows[inv] = (w32.reshape(-1, 1) * dout[keep].float().repeat_interleave(k, 0)).to(torch.bfloat16)
    vx, vgu, vd = torch.autograd.grad(rows, [xv] + params, drows, retain_graph=True)
    assert torch.equal(dx[keep], vx) and bool((dx[~keep] == 0).all())
    assert torch.equal(dgu, vgu) and torch.equal(dd, vd) and torch.equal(amax, m.fp8_amax)
    assert bool((dgu[5] == 0).all()) and bool((dd[5] == 0).all())
    vl, = torch.autograd.grad(yv, lv, dout[keep].double())
    # dweights: dot products of D terms, 2^-24 of their absolute sum a step; then the route's own bound
    dots = (rows.double()[inv].view(n, k, D) * dout[keep].double()[:, None]).abs().sum(2)
    bound = (2 * 72 + _sum_steps(D)) * 2.0 ** -24 * 2 * dots.sum(1, keepdim=True)
    assert ((dl[keep].double() - vl).abs() <= bound).all() and bool((dl[~keep] == 0).all())


def test_routed_layer_without_tokens_and_all_masked(dev):
    """No tokens, and a batch that is all padding: zeros, and zero gradients."""
    D, I, E, k = 128, 128, 4, 2
    m = _Experts(E, D, I, dev).train()
    for T, mask in ((0, None), (70, torch.zeros(70, dtype=torch.bool, device=dev))):
        x = torch.randn(T, D, device=dev).to(torch.bfloat16).requires_grad_(True)
        low = torch.randn(T, E, device=dev).requires_grad_(True)
        y, sel = sg.fp8_routed_experts(x, low, m, k, mask=mask)
        assert y.shape == (T, D) and bool((y == 0).all()) and bool((sel == -1).all())
        for g in torch.autograd.grad(y, [x, low, m.gate_up_proj, m.down_proj], torch.ones_like(y)):
            assert bool((g == 0).all())


def test_training_step(dev):
    """A router, the layer, clipping over its parameters and the momentum stage:
    the norm, the clipped gradients and the stage's results against torch."""
    T, D, I, E, k = 512, 256, 256, 4, 2
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(T, D, device=dev, generator=g).to(torch.bfloat16)
    router = torch.nn.Parameter(torch.randn(E, D, device=dev, generator=g) * D ** -0.5)
    m = _Experts(E, D, I, dev).train()
    params = [router, m.gate_up_proj, m.down_proj]
    for step in range(2):
        for p in params:
            p.grad = None
        y, sel = sg.fp8_routed_experts(x, torch.nn.functional.linear(x.float(), router), m, k, score="sigmoid", scale=1.5)
        (y.float().square().mean()).backward()
        assert all(bool(p.grad.isfinite().all()) and float(p.grad.abs().max()) > 0 for p in params)
        before = [p.grad.clone() for p in params]
        norm, factor = O.clip(before, 1e-3)
        assert factor < 1
        got = sg.clip_grad_norm_(params, 1e-3)
        assert abs(float(got) - norm) <= 2.0 ** -24 * 1.01 * norm
        for p, b in zip(params, before):
            assert ((p.grad.double() - b.double() * factor).abs() <= 5 * 2.0 ** -24 * (b.double() * factor).abs() + 1e-44).all()
        for p in params[1:]:
            v = torch.zeros_like(p)
            u = torch.empty(p.shape, dtype=torch.bfloat16, device=dev)
            sg._momentum_stage(p.grad, v, u, 0.95)
            rv = torch.zeros_like(p).lerp_(p.grad, 1 - 0.95)
            assert torch.equal(v, rv)
        sg.fp8_update_scales(m)


def test_side_stream_and_threads(dev):
    """Calls on another stream than the default, and from two threads at once,
    each on a stream of its own, give the same bits."""
    low = _logits(dev, 3000, 64, torch.float32, 3)
    rows = torch.randn(3000 * 4, 128, device=dev).to(torch.bfloat16)

    def work():
        w, sel = sg.route_tokens(low, 4)
        tok, inv, off = sg.expert_order(sel, 64)
        return w, sel, tok, inv, off, sg.combine_experts(rows, w, inv, off)

    want = work()
    torch.cuda.synchronize()
    got = {}

    def go(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = work()
        s.synchronize()

    go(0)
    threads = [threading.Thread(target=go, args=(i,)) for i in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want))


def test_captured_and_replayed(dev):
    """Route, order and combine captured into a graph: every replay on new data
    equals the eager call, with eager work between the replays; two graphs side
    by side do not disturb each other."""
    T, E, k, D = 700, 32, 4, 96

    def data(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return (torch.randn(T, E, device=dev, generator=g), torch.randn(T * k, D, device=dev, generator=g).to(torch.bfloat16),
                torch.randn(T, k, device=dev, generator=g), torch.randn(T, D, device=dev, generator=g).to(torch.bfloat16))

    def work(low, rows, dw, dout):
        w, sel, picked = sg.ops.moe_route(low, None, None, "sigmoid", 4, 2, 2, k, True, 1.0)
        dl = sg.ops.moe_route_bwd(dw, sel, picked, low, "sigmoid", True, 1.0)
        tok, inv, off = sg.ops.moe_expert_order(sel, E)
        y = sg.ops.moe_combine(rows, w, inv)
        dr, dwt = sg.ops.moe_combine_bwd(dout, rows, w, inv, off)
        return w, sel, dl, tok, inv, off, y, dr, dwt

    graphs = []
    for i in range(2):
        ins = data(100 + i)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work(*ins)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work(*ins)
        graphs.append((graph, ins, outs))
    for rep in range(4):
        for i, (graph, ins, outs) in enumerate(graphs):
            new = data(10 * rep + i)
            for a, b in zip(ins, new):
                a.copy_(b)
            graph.replay()
            want = work(*new)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), (rep, i)


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_gradients_captured_and_replayed(dev, score, renorm):
    """The layer's steps and their gradients, through autograd, captured into a
    graph: every replay on new data equals the eager gradients."""
    T, E, k, D = 500, 24, 3, 72

    def data(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return (torch.randn(T, E, device=dev, generator=g).requires_grad_(),
                torch.randn(T * k, D, device=dev, generator=g).to(torch.bfloat16).requires_grad_(),
                torch.randn(T, D, device=dev, generator=g).to(torch.bfloat16))

    def work(low, rows, dout):
        w, sel = sg.route_tokens(low, k, score=score, renormalize=renorm)
        tok, inv, off = sg.expert_order(sel, E)
        y = sg.combine_experts(rows, w, inv, off)
        return (y.detach(), sel) + torch.autograd.grad(y, (low, rows), dout)

    ins = data(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work(*ins)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(*ins)
    for rep in range(4):
        new = data(rep + 1)
        with torch.no_grad():
            for a, b in zip(ins, new):
                a.copy_(b)
        graph.replay()
        want = work(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep


def test_compiled_matches_eager(dev):
    T, E, k, D = 300, 16, 2, 64
    low = _logits(dev, T, E, torch.float32, 21)
    rows = torch.randn(T * k, D, device=dev).to(torch.bfloat16)
    dout = torch.randn(T, D, device=dev).to(torch.bfloat16)

    def f(low, rows):
        w, sel = sg.route_tokens(low, k, score="sigmoid")
        tok, inv, off = sg.expert_order(sel, E)
        return sg.combine_experts(rows, w, inv, off), sel

    outs = []
    for fn in (f, torch.compile(f, dynamic=False, fullgraph=True)):
        a, b = low.clone().requires_grad_(True), rows.clone().requires_grad_(True)
        y, sel = fn(a, b)
        outs.append((y, sel) + torch.autograd.grad(y, [a, b], dout))
    assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_operators_opcheck(dev):
    low = _logits(dev, 20, 16, torch.bfloat16, 2)
    args = (low, None, None, "softmax", 1, 1, 1, 3, False, 1.0)
    w, sel, picked = torch.ops.sparkfp8.route_fwd(*args)
    torch.library.opcheck(torch.ops.sparkfp8.route_fwd.default, args)
    torch.library.opcheck(torch.ops.sparkfp8.route_bwd.default, (w, sel, picked, low, "softmax", False, 1.0))
    torch.library.opcheck(torch.ops.sparkfp8.expert_order.default, (sel, 16))
    _, inv, off = torch.ops.sparkfp8.expert_order(sel, 16)
    rows = torch.randn(60, 24, device=dev)
    torch.library.opcheck(torch.ops.sparkfp8.combine_fwd.default, (rows, w, inv))
    torch.library.opcheck(torch.ops.sparkfp8.combine_bwd.default, (rows[:20], rows, w, inv, off))


def test_no_gradient_and_one_gradient(dev):
    """Nothing asked of the logits costs no backward; weights alone carry one."""
    low = _logits(dev, 10, 8, torch.float32, 6)
    with torch.no_grad():
        assert not sg.route_tokens(low, 2)[0].requires_grad
    leaf = low.clone().requires_grad_(True)
    w, sel = sg.route_tokens(leaf, 2)
    assert w.requires_grad and not sel.requires_grad
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(w.sum(), leaf, create_graph=True)
        torch.autograd.grad(d.sum(), leaf)


@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_bias_that_requires_a_gradient(dev, score, compiled):
    """A bias held as a Parameter has no gradient: a router whose logits need
    none gives weights that need none, and one whose logits do gets the same
    gradient as with a plain bias."""
    T, E, k, D = 60, 16, 3, 40
    low = _logits(dev, T, E, torch.float32, 12)
    bias = torch.nn.Parameter(torch.linspace(-0.2, 0.2, E, device=dev))
    rows = torch.randn(T * k, D, device=dev)
    dout = torch.randn(T, D, device=dev)

    def f(low, bias, rows):
        w, sel = sg.route_tokens(low, k, score=score, bias=bias)
        tok, inv, off = sg.expert_order(sel, E)
        return sg.combine_experts(rows, w, inv, off), w

    run = torch.compile(f, dynamic=False, fullgraph=True) if compiled else f
    # a frozen router
    r = rows.clone().requires_grad_(True)
    y, w = run(low, bias, r)
    assert not w.requires_grad
    y.backward(dout)
    want, = torch.autograd.grad(f(low, bias.detach(), r)[0], r, dout)
    assert bias.grad is None and torch.equal(r.grad, want)
    y, w = run(low, bias, rows)  # nothing needs a gradient
    assert not y.requires_grad and not w.requires_grad
    # a router that learns
    a, b = low.clone().requires_grad_(True), low.clone().requires_grad_(True)
    y, w = run(a, bias, rows)
    y.backward(dout)
    z, _ = f(b, bias.detach(), rows)
    z.backward(dout)
    assert bias.grad is None and torch.equal(y, z) and torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("sigmoid", True), ("sigmoid", False), ("softmax", False)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_logits_after_routing(dev, score, renorm, dtype):
    """The gradient needs the logits' values for the plain softmax alone: else
    they may be written, and their memory is free, once the tokens are routed.
    For the plain softmax a write is refused."""
    T, E, k = 4096, 256, 4
    leaf = _logits(dev, T, E, DTYPES[dtype], 31).requires_grad_(True)
    dw = torch.randn(T, k, device=dev)
    kw = dict(score=score, renormalize=renorm)
    want, = torch.autograd.grad(sg.route_tokens(leaf * 1, k, **kw)[0], leaf, dw)
    low = leaf * 1
    w, sel = sg.route_tokens(low, k, **kw)
    low.detach().zero_()
    dense = score == "softmax" and not renorm
    if dense:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(w, leaf, dw)
    else:
        assert torch.equal(torch.autograd.grad(w, leaf, dw)[0], want)
    del low, w, sel
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    w, sel = sg.route_tokens(leaf * 1, k, **kw)
    held = torch.cuda.memory_allocated() - start
    assert (held >= T * E * leaf.element_size()) == dense
    assert torch.equal(torch.autograd.grad(w, leaf, dw)[0], want)


def test_rows_after_the_combine(dev):
    """The rows' values are needed for the gradient of the weights alone: with
    weights that need none the rows may be written, and their memory is free,
    once they are combined.  Else a write is refused."""
    T, k, D = 1000, 4, 256
    sel = torch.randint(-1, 8, (T, k), device=dev)
    _, inv, off = sg.expert_order(sel, 8)
    leaf = torch.randn(T * k, D, device=dev, requires_grad=True)
    dout = torch.randn(T, D, device=dev)
    for learns in (False, True):
        w = torch.rand(T, k, device=dev, requires_grad=learns)
        want, = torch.autograd.grad(sg.combine_experts(leaf * 1, w, inv, off), leaf, dout)
        rows = leaf * 1
        y = sg.combine_experts(rows, w, inv, off)
        rows.detach().zero_()
        if learns:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, leaf, dout)
        else:
            assert torch.equal(torch.autograd.grad(y, leaf, dout)[0], want)
        del rows, y
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        y = sg.combine_experts(leaf * 1, w, inv, off)
        held = torch.cuda.memory_allocated() - start
        assert (held >= T * k * D * 4) == learns
        assert torch.equal(torch.autograd.grad(y, leaf, dout)[0], want)
        del y
    w = torch.rand(T, k, device=dev, requires_grad=True)
    got, = torch.autograd.grad(sg.combine_experts(leaf.detach(), w, inv, off), w, dout)
    assert torch.equal(got, sg.ops.moe_combine_bwd(dout, leaf.detach(), w.detach(), inv, off, False, True)[1])


def test_second_derivatives_are_refused(dev):
    """The first gradient with create_graph is the plain one; a derivative of it
    raises, whole or in one leaf, and alone or in a sum where its part would
    otherwise be missing."""
    T, E, k, D = 12, 8, 2, 24
    sel = torch.randint(0, E, (T, k), device=dev)
    _, inv, off = sg.expert_order(sel, E)
    low, rows, w = (torch.randn(s, device=dev, requires_grad=True) for s in ((T, E), (T * k, D), (T, k)))
    calls = [(lambda kw=kw: sg.route_tokens(low, k, **kw)[0], (low,), (T, k))
             for kw in (dict(), dict(renormalize=False), dict(score="sigmoid"))]
    calls.append((lambda: sg.combine_experts(rows, w, inv, off), (rows, w), (T, D)))
    for call, leaves, shape in calls:
        for upstream_learns in (False, True):
            dy = torch.randn(shape, device=dev, requires_grad=upstream_learns)
            want = torch.autograd.grad(call(), leaves, dy.detach())
            got = torch.autograd.grad(call(), leaves, dy, create_graph=True)
            for d, x in zip(got, want):
                assert d.requires_grad and torch.equal(d, x)
                with pytest.raises(RuntimeError, match="differentiable once"):
                    d.square().sum().backward(retain_graph=True)
                for leaf in leaves + ((dy,) if upstream_learns else ()):
                    loss = (leaf * 3).sum() + d.square().sum()
                    with pytest.raises(RuntimeError, match="differentiable once"):
                        torch.autograd.grad(loss, leaf, retain_graph=True)
        assert all(leaf.grad is None for leaf in leaves)
