"""GPU tests of the experts' layer for a few tokens against its formulas in 64
bits: the selection equal to the routing oracle's on 64-bit logits, the output
within a bound that the sums' lengths and sizes give."""
import pytest
import torch

import spark_gpt_amd as sg
from oracle import mxfp4 as Q
from oracle import routing as O

pytestmark = pytest.mark.gpu


def _randn(dev, *shape, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)


def _layer(dev, T, E, D, I, seed=0, router=torch.bfloat16):
    return (_randn(dev, T, D, seed=seed), _randn(dev, E, D, seed=seed + 1, std=D ** -0.5, dtype=router),
            _randn(dev, E, 2 * I, D, seed=seed + 2, std=D ** -0.5), _randn(dev, E, D, I, seed=seed + 3, std=I ** -0.5))


def _reference(x, weights, selected, w_gu, w_down):
    """(out, bound) in 64 bits.  A sum of n products in 32 bits is off by n 2^-23 of the sum of their sizes (twice the
    rounding bound, for adders that truncate); silu's slope is at most 1.1, its exponential is off by |g| + 8 steps; the
    two bf16 parts of h hold it to 2^-17; the waves' and slots' sums are part of n."""
    T, k = selected.shape
    I = w_down.shape[2]
    out = torch.zeros(T, w_down.shape[1], dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    eps = 2.0 ** -23
    for t in range(T):
        for j in range(k):
            e = int(selected[t, j])
            if e < 0:
                continue
            w, xt = float(weights[t, j]), x[t].double()
            gu, size = w_gu[e].double() @ xt, w_gu[e].double().abs() @ xt.abs()
            g, u = gu[:I], gu[I:]
            dg, du = xt.numel() * eps * size[:I], xt.numel() * eps * size[I:]
            s = g * torch.sigmoid(g)
            h = s * u
            dh = 1.1 * dg * u.abs() + s.abs() * du + 1.1 * dg * du + ((g.abs() + 8) * eps + 2.0 ** -17) * h.abs()
            wd = w_down[e].double()
            out[t] += w * (wd @ h)
            err[t] += abs(w) * (wd.abs() @ dh + (2 * I + 16) * eps * (wd.abs() @ h.abs())) * (1 + 2.0 ** -20)
    return out, err + 2.0 ** -8 * (out.abs() + err) + 2.0 ** -126


def _check(x, router, w_gu, w_down, k, values=None, **kw):
    """values: the weights that the reference multiplies by (of codes)."""
    out, selected = sg.decode_routed_experts(x, router, w_gu, w_down, k, **kw)
    low = x.double() @ router.double().T
    w, sel = O.route(low, k, **kw)
    assert out.dtype == torch.bfloat16 and out.shape == x.shape
    assert selected.dtype == torch.int64 and torch.equal(selected.cpu(), sel)
    ref, bound = _reference(x, w, sel, *(values or (w_gu, w_down)))
    bad = ~((out.double() - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), out[bad][:4], ref[bad][:4], bound[bad][:4])
    # all errors together are a rounding to bf16 and little more
    norm = float(ref.norm())
    if norm:
        assert float((out.double() - ref).norm()) / norm < 2.0 ** -8
    return out, selected


SIZES = [(1, 1, 1, 8, 8), (1, 8, 2, 64, 24), (2, 4, 4, 40, 16), (1, 128, 8, 512, 96), (3, 16, 3, 264, 72),
         (16, 8, 2, 128, 200), (17, 8, 2, 128, 64), (33, 60, 4, 96, 136), (64, 64, 6, 256, 88), (64, 4, 1, 72, 40),
         (64, 2, 2, 200, 64), (20, 8, 2, 4096, 40), (10, 8, 2, 4104, 16), (40, 3, 2, 8200, 8),
         (5, 300, 10, 64, 32), (2, 1024, 64, 64, 16), (64, 70, 64, 32, 8), (8, 8, 2, 1024, 1536)]


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("T,E,k,D,I", SIZES)
def test_layer(dev, T, E, k, D, I, four):
    x, router, w_gu, w_down = _layer(dev, T, E, D, I, seed=T + E)
    if not four:
        _check(x, router, w_gu, w_down, k)
        return
    q_gu, q_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
    values = (Q.quantized(w_gu).to(dev), Q.quantized(w_down).to(dev))
    _check(x, router, q_gu, q_down, k, values=values)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("T,E,k,D,I", [(2, 1, 1, 16384, 32768), (18, 40, 1, 4096, 8192)])
def test_largest_matrices_and_offsets(dev, T, E, k, D, I, four):
    """A matrix of the largest size (2 GiB in bf16), and experts that lie past 4 GiB."""
    x, router, w_gu, w_down = _layer(dev, T, E, D, I, seed=3)
    if E > 1:  # token t takes expert 39 - t
        x[:, :E] = torch.eye(E, device=dev)[E - 1 - torch.arange(T, device=dev)].bfloat16()
        router.zero_()[:, :E] = 4 * torch.eye(E, device=dev)
    if four:
        q_gu, q_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
        del w_gu, w_down
        values = (sg.mxfp4_dequantize(q_gu), sg.mxfp4_dequantize(q_down))
        _, selected = _check(x, router, q_gu, q_down, k, values=values)
    else:
        _, selected = _check(x, router, w_gu, w_down, k)
    assert selected[:, 0].tolist() == ([39 - t for t in range(T)] if E > 1 else [0, 0])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("groups,top_groups,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2), (12, 5, 2), (6, 6, 1)])
def test_routing_options(dev, score, renorm, with_bias, groups, top_groups, best):
    for T, E, k, router in ((9, 12, 3, torch.float32), (40, 120, 8, torch.bfloat16)):
        k = min(k, top_groups * (E // groups))
        x, r, w_gu, w_down = _layer(dev, T, E, 64, 24, seed=E, router=router)
        bias = _randn(dev, E, seed=5, std=0.3, dtype=torch.float32) if with_bias else None
        mask = torch.rand(T, device=dev, generator=torch.Generator(device=dev).manual_seed(2)) > 0.25
        _check(x, r, w_gu, w_down, k, score=score, renormalize=renorm, bias=bias, groups=groups,
               top_groups=top_groups, group_best=best, mask=mask, scale=2.5)


def test_special_tokens_and_scores(dev):
    """Ties, masked and NaN tokens, infinite ones, experts that cannot be taken; each token by itself."""
    T, E, k, D, I = 12, 20, 4, 64, 24
    x, router, w_gu, w_down = _layer(dev, T, E, D, I)
    # exact logits: multiples of a quarter
    x.copy_((x.float() * 2).round().clamp(-4, 4) / 2)
    router.copy_((router.float() * 16).round().clamp(-4, 4) / 2)
    router[7] = router[3]
    router[11] = router[3]
    x[4] = 0
    clean, chosen = _check(x, router, w_gu, w_down, k)
    assert chosen[4].tolist() == [0, 1, 2, 3]
    live = [t for t in range(T) if t not in (2, 6)]
    broken = x.clone()
    broken[2, 9] = float("nan")
    broken[6, 1] = float("inf")
    out, sel = sg.decode_routed_experts(broken, router, w_gu, w_down, k)
    assert sel[2].tolist() == [0, 1, 2, 3] and out[2].isnan().all()
    assert torch.equal(out[live], clean[live]) and torch.equal(sel[live], chosen[live])
    low = broken.double() @ router.double().T
    assert torch.equal(sel.cpu(), O.route(low, k)[1])
    for score in ("softmax", "sigmoid"):
        bias = torch.full((E,), -float("inf"), device=dev)
        bias[5], bias[13] = 0.0, 0.1
        out, sel = _check(x, router, w_gu, w_down, k, bias=bias, score=score)
        assert (sel[:, 2:] == -1).all() and (sel[:, :2] >= 0).all()
        bias.fill_(-float("inf"))
        out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, k, bias=bias, score=score)
        assert (sel == -1).all() and not out.any()
    none = torch.zeros(T, dtype=torch.bool, device=dev)
    out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, k, mask=none)
    assert (sel == -1).all() and not out.any()
    # a masked token may hold anything
    some = torch.ones(T, dtype=torch.bool, device=dev)
    some[[2, 6]] = False
    out, sel = sg.decode_routed_experts(broken, router, w_gu, w_down, k, mask=some)
    assert torch.equal(out[live], clean[live]) and not out[[2, 6]].any() and (sel[[2, 6]] == -1).all()
    # an expert with broken weights reaches the tokens that take it alone
    bad = w_gu.clone()
    e = int(chosen[0, 0])
    bad[e, 3, 5] = float("nan")
    out, _ = sg.decode_routed_experts(x, router, bad, w_down, k)
    takes = (chosen == e).any(1)
    assert out[takes].isnan().all() and torch.equal(out[~takes], clean[~takes])


def test_overflowing_h(dev):
    """h past bf16's largest value is an infinity, as the product in 32 bits rounded to bf16 would be; no NaN comes of
    the second part."""
    x, router, w_gu, w_down = _layer(dev, 2, 4, 64, 16)
    x.fill_(1.0)
    router.zero_()
    w_gu.fill_(2.0 ** 60)
    w_down.fill_(1.0)
    out, _ = sg.decode_routed_experts(x, router, w_gu, w_down, 1)
    assert (out == float("inf")).all()


def test_strides_types_and_no_tokens(dev):
    x, router, w_gu, w_down = _layer(dev, 6, 8, 128, 40)
    out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, 3)
    wide = torch.full((6, 300), float("nan"), device=dev, dtype=torch.bfloat16)
    wide[:, 11:139] = x
    for other in (wide[:, 11:139], x.t().contiguous().t(), x.repeat_interleave(2, 0)[::2]):
        o, s = sg.decode_routed_experts(other, router, w_gu, w_down, 3)
        assert torch.equal(o, out) and torch.equal(s, sel)
    o, s = sg.decode_routed_experts(x, router.float(), w_gu, w_down, 3)
    assert torch.equal(o, out) and torch.equal(s, sel)
    same = x[:1].expand(5, -1)
    o, s = sg.decode_routed_experts(same, router, w_gu, w_down, 3)
    assert torch.equal(s, sel[:1].expand(5, -1)) and all(torch.equal(o[t], o[0]) for t in range(5))
    o, s = sg.decode_routed_experts(x[:0], router, w_gu, w_down, 3)
    assert o.shape == (0, 128) and s.shape == (0, 3)


def test_token_alone_or_among_others(dev):
    """A token's experts do not depend on the batch, and its output is that of the same formula."""
    x, router, w_gu, w_down = _layer(dev, 40, 16, 256, 72)
    out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, 4)
    for t in (0, 17, 39):
        o, s = sg.decode_routed_experts(x[t:t + 1], router, w_gu, w_down, 4)
        assert torch.equal(s[0], sel[t])
        assert float((o[0].float() - out[t].float()).norm() / out[t].float().norm()) < 2.0 ** -7


def test_refusals(dev):
    x, router, w_gu, w_down = _layer(dev, 4, 8, 64, 16)
    call = lambda **kw: sg.decode_routed_experts(kw.pop("x", x), kw.pop("router", router), kw.pop("w_gu", w_gu),
                                                 kw.pop("w_down", w_down), kw.pop("k", 2), **kw)
    for kw in (dict(x=x.float()), dict(x=_randn(dev, 65, 64)), dict(x=x[:, :32]), dict(router=router[:, :32]),
               dict(router=router.half()), dict(router=router[:4]), dict(w_gu=w_gu[:, :30]), dict(w_gu=w_gu.float()),
               dict(w_down=w_down[:4]), dict(w_gu=w_gu[0]), dict(k=0), dict(k=9), dict(k=65), dict(score="tanh"),
               dict(groups=3), dict(groups=4, top_groups=5), dict(groups=4, top_groups=1, k=3), dict(group_best=3),
               dict(bias=torch.zeros(7, device=dev)), dict(bias=torch.zeros(8, device=dev, dtype=torch.bfloat16)),
               dict(mask=torch.ones(3, device=dev, dtype=torch.bool)), dict(mask=torch.ones(4, device=dev)),
               dict(router=router.cpu()), dict(w_gu=w_gu.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**kw)
    q = sg.mxfp4_quantize(w_gu)
    with pytest.raises(TypeError):
        call(w_gu=q)
    with pytest.raises(ValueError):
        call(w_gu=sg.MXFP4(q.codes[:4], q.scales[:4], q.shape), w_down=sg.mxfp4_quantize(w_down))
    with pytest.raises(ValueError, match="multiples of 8"):
        sg.decode_routed_experts(x[:, :60], router[:, :60].contiguous(), w_gu[:, :, :60].contiguous(),
                                 w_down[:, :60].contiguous(), 2)
    with pytest.raises(ValueError, match="no gradient"):
        call(x=x.clone().requires_grad_(True))
    with torch.no_grad():
        call(x=x.clone().requires_grad_(True))


def _stack(dev, layers, E, D, I):
    out = []
    for i in range(layers):
        _, router, w_gu, w_down = _layer(dev, 1, E, D, I, seed=10 * i)
        if i % 2:
            w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
        out.append((router, w_gu, w_down, sg.mxfp4_quantize(_randn(dev, D, D, seed=i, std=D ** -0.5))))
    return out


def _generation_step(x, stack, k):
    """Layers as generation runs them: a 4-bit projection, the experts (bf16 and 4-bit in turn), residuals."""
    picked = []
    for router, w_gu, w_down, proj in stack:
        x = x + sg.mxfp4_linear(x, proj)
        out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, k)
        x = x + out
        picked.append(sel)
    return x, torch.stack(picked)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_generation_captured_and_replayed(dev, T):
    E, D, I, k = 16, 256, 72, 3
    stack = _stack(dev, 3, E, D, I)
    with torch.no_grad():
        x = torch.zeros(T, D, device=dev, dtype=torch.bfloat16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _generation_step(x, stack, k)
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = _generation_step(x, stack, k)
            graphs.append((graph, out))
        for seed in range(4):
            fresh = _randn(dev, T, D, seed=20 + seed)
            x.copy_(fresh)
            ref = _generation_step(fresh, stack, k)
            for graph, out in graphs:
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
                _generation_step(fresh.flip(0), stack, k)
        assert bool(torch.isfinite(ref[0].float()).all())


def test_two_streams_at_once(dev):
    x, router, w_gu, w_down = _layer(dev, 20, 16, 512, 136)
    xs = [x, x.flip(0).contiguous()]
    ref = [sg.decode_routed_experts(v, router, w_gu, w_down, 4) for v in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sg.decode_routed_experts(xs[i], router, w_gu, w_down, 4))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i][0]) and torch.equal(s, ref[i][1]) for o, s in got[i])


def test_compiled_matches_eager(dev):
    x, router, w_gu, w_down = _layer(dev, 3, 8, 128, 40)
    f = torch.compile(lambda v: sg.decode_routed_experts(v, router, w_gu, w_down, 2, scale=1.5), fullgraph=True,
                      dynamic=False)
    with torch.no_grad():
        got, want = f(x), sg.decode_routed_experts(x, router, w_gu, w_down, 2, scale=1.5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_same_layer_as_the_grouped_experts(dev):
    """Beside route_tokens, expert_order, the experts in torch and combine_experts: the same experts, and outputs that
    differ by that path's bf16 rows."""
    T, E, k, D, I = 24, 8, 2, 128, 64
    x, router, w_gu, w_down = _layer(dev, T, E, D, I, router=torch.float32)
    out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, k)
    weights, selected = sg.route_tokens(x.float() @ router.T, k)
    assert torch.equal(selected, sel)
    token, inverse, offsets = sg.expert_order(selected, E)
    owner = torch.searchsorted(offsets, torch.arange(T * k, device=dev), right=True)
    gu = (w_gu[owner].float() @ x[token].float()[:, :, None])[:, :, 0]
    h = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
    rows = (w_down[owner].float() @ h[:, :, None])[:, :, 0].to(torch.bfloat16)
    ref = sg.combine_experts(rows, weights, inverse, offsets)
    assert float((out.float() - ref.float()).norm() / ref.float().norm()) < 2.0 ** -7


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("T,D", [(1, 64), (1, 2048), (1, 4096), (9, 64), (9, 2048), (24, 64)])
def test_h_keeps_its_32_bits(dev, T, D, four):
    """Two columns of h, 64 (1 + 2^-8 + 2^-17) and 64 (1 + 2^-8), whose difference is the output: 2^-11, which the 17
    bits of two bf16 parts do not hold.  In steps of 2^-23 of 65, which h stays below: a sum of three products is off
    by 3, the sigmoid by 1, the two products by 1 together; the difference of what two columns' three parts give, six
    products, by 12: 2 * 5 + 12 in all."""
    x, router, w_gu, w_down = _layer(dev, T, 2, D, 16)
    for t in (x, router, w_gu, w_down):
        t.zero_()
    x[:, :4] = torch.tensor([64.0, 1.0, 2.0 ** -8, 2.0 ** -17], device=dev).bfloat16()
    w_gu[:, :2, 0] = 1  # the gate
    w_gu[:, 16:18, 1:3] = 1
    w_gu[:, 16, 3] = 1
    w_down[:, :, 0], w_down[:, :, 1] = 1, -1
    if four:
        w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
    out, _ = sg.decode_routed_experts(x, router, w_gu, w_down, 1)
    off = (out.double() - 2.0 ** -11).abs().max()
    assert float(off) <= 22 * 65 * 2.0 ** -23 + 2.0 ** -8 * 2.0 ** -11, float(off)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("T", [1, 9, 24])
def test_infinities_in_h(dev, T, four):
    """An infinity in one column of h is one in the output, of either sign; both, or a weight of zero beside it, are a
    NaN."""
    def run(columns, zero_weight=False):
        x, router, w_gu, w_down = (torch.zeros_like(t) for t in _layer(dev, T, 2, 64, 16))
        x[:, 0] = 1
        w_down.fill_(1)
        if zero_weight:
            w_down[:, :, 5] = 0
        for column, sign in columns:
            w_gu[:, column, 0], w_gu[:, 16 + column, 0] = 2.0 ** 100, sign * 2.0 ** 100
        if four:
            w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
        return sg.decode_routed_experts(x, router, w_gu, w_down, 1)[0]

    assert (run([(2, 1)]) == float("inf")).all() and (run([(3, -1)]) == -float("inf")).all()
    assert run([(2, 1), (3, -1)]).isnan().all() and run([(5, 1)], zero_weight=True).isnan().all()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("T", [1, 6, 24])
def test_silu_of_large_gates(dev, T, four):
    """silu(g) less 64 v, v the fp32 value nearest to silu(g) / 64, for gates whose product with log2(e) rounds badly
    (off by 26 steps of 2^-23 in the exponential).  In those steps of silu(g): the exponential is off by 1, the sum and the
    quotient by 1 together, v's three parts by 2, the down sums' six products by 6: 10."""
    x, router, w_gu, w_down = (torch.zeros_like(t) for t in _layer(dev, T, 2, 64, 16))
    g = -torch.tensor([61.25, 58.0, 54.75, 51.5, 48.25, 45.0], dtype=torch.float64, device=dev)
    g = g[torch.arange(T, device=dev) % 6]
    silu = g / (1 + torch.exp(-g))
    left = (silu / 64).float()
    v = left.double()
    x[:, 0], x[:, 1], x[:, 2] = g.bfloat16(), 64, 1
    for part in range(3):
        x[:, 3 + part] = left.bfloat16()
        left = left - x[:, 3 + part].float()
    assert not left.any()
    w_gu[:, 0, 0] = w_gu[:, 1, 1] = w_gu[:, 16, 2] = 1
    w_gu[:, 17, 3:6] = 1
    w_down[:, :, 0], w_down[:, :, 1] = 1, -1
    if four:
        w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
    out, _ = sg.decode_routed_experts(x, router, w_gu, w_down, 1)
    ref, err = (silu - 64 * v)[:, None], (10 * 2.0 ** -23 * silu.abs())[:, None]
    off = (out.double() - ref).abs()
    assert (off <= err + 2.0 ** -8 * (ref.abs() + err)).all(), (off / silu.abs()[:, None]).max() * 2.0 ** 23


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("groups,top_groups,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2), (12, 5, 2), (6, 6, 1)])
def test_routing_options_of_one_to_four_tokens(dev, score, renorm, with_bias, groups, top_groups, best):
    """Few enough tokens and candidates that gate and up selects by itself, up to 256 experts, bf16 and 4-bit."""
    for T, E, k, router, four in ((1, 12, 3, torch.float32, False), (3, 12, 3, torch.bfloat16, True),
                                  (4, 120, 8, torch.bfloat16, False), (4, 252, 6, torch.float32, True)):
        k = min(k, top_groups * (E // groups))
        x, r, w_gu, w_down = _layer(dev, T, E, 64, 24, seed=E + T, router=router)
        bias = _randn(dev, E, seed=5, std=0.3, dtype=torch.float32) if with_bias else None
        values = None
        if four:
            values = (Q.quantized(w_gu).to(dev), Q.quantized(w_down).to(dev))
            w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
        for masked in ((), (0,), tuple(range(T))) if T > 1 else ((), (0,)):
            mask = torch.ones(T, dtype=torch.bool, device=dev)
            mask[list(masked)] = False
            out, sel = _check(x, r, w_gu, w_down, k, values=values, score=score, renormalize=renorm, bias=bias,
                              groups=groups, top_groups=top_groups, group_best=best, mask=mask, scale=2.5)
            assert not out[~mask].any() and (sel[~mask] == -1).all() and (sel[mask] >= 0).all()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("E", [20, 150])
def test_special_tokens_and_scores_of_four_tokens(dev, E, four):
    """Ties, NaN and infinite tokens, experts that cannot be taken, masks, where gate and up selects by itself."""
    T, k, D, I = 4, 4, 64, 24
    x, router, w_gu, w_down = _layer(dev, T, E, D, I)
    x.copy_((x.float() * 2).round().clamp(-4, 4) / 2)  # exact logits, multiples of a quarter
    router.copy_((router.float() * 16).round().clamp(-4, 4) / 2)
    router[7] = router[3]
    router[11] = router[3]
    x[3] = 0
    values = None
    if four:
        values = (Q.quantized(w_gu).to(dev), Q.quantized(w_down).to(dev))
        w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
    clean, chosen = _check(x, router, w_gu, w_down, k, values=values)
    assert chosen[3].tolist() == [0, 1, 2, 3]
    for value in (float("nan"), float("inf")):
        broken = x.clone()
        broken[1, 9] = value
        out, sel = sg.decode_routed_experts(broken, router, w_gu, w_down, k)
        low = broken.double() @ router.double().T
        assert torch.equal(sel.cpu(), O.route(low, k)[1]) and out[1].isnan().all()
        assert torch.equal(out[[0, 2, 3]], clean[[0, 2, 3]])
        some = torch.tensor([True, False, True, True], device=dev)
        out, sel = sg.decode_routed_experts(broken, router, w_gu, w_down, k, mask=some)
        assert torch.equal(out[some], clean[some]) and not out[1].any() and (sel[1] == -1).all()
    for score in ("softmax", "sigmoid"):
        bias = torch.full((E,), -float("inf"), device=dev)
        bias[5], bias[13] = 0.0, 0.1
        _, sel = _check(x, router, w_gu, w_down, k, values=values, bias=bias, score=score)
        assert (sel[:, 2:] == -1).all() and (sel[:, :2] >= 0).all()
        out, sel = sg.decode_routed_experts(x, router, w_gu, w_down, k, bias=bias.fill_(-float("inf")), score=score)
        assert (sel == -1).all() and not out.any()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("T,E,k,D,I", [(64, 1024, 16, 64, 16), (40, 1024, 12, 64, 16), (64, 600, 64, 32, 8),
                                       (50, 1024, 20, 40, 24)])
def test_many_candidates(dev, T, E, k, D, I, four):
    """More candidates than down's work-groups take in a turn (512), as experts and as slots, and slots past 256."""
    x, router, w_gu, w_down = _layer(dev, T, E, D, I, seed=T)
    if not four:
        _check(x, router, w_gu, w_down, k)
        return
    values = (Q.quantized(w_gu).to(dev), Q.quantized(w_down).to(dev))
    _check(x, router, sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down), k, values=values)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("groups,top_groups,best", [(1, 1, 1), (8, 3, 2), (64, 20, 1)])
def test_routing_options_of_many_experts(dev, score, with_bias, groups, top_groups, best):
    """Past 256 experts a lane of the selection holds sixteen of them."""
    for T, E, k in ((3, 512, 8), (30, 960, 12)):
        x, router, w_gu, w_down = _layer(dev, T, E, 64, 16, seed=E, router=torch.float32)
        bias = _randn(dev, E, seed=5, std=0.3, dtype=torch.float32) if with_bias else None
        mask = torch.rand(T, device=dev, generator=torch.Generator(device=dev).manual_seed(3)) > 0.25
        _check(x, router, w_gu, w_down, k, score=score, renormalize=False, bias=bias, groups=groups,
               top_groups=top_groups, group_best=best, mask=mask, scale=0.5)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("D,I", [(64, 72), (2048, 136), (4096, 264)])
def test_every_number_of_slots(dev, D, I, four):
    """An expert of 1 .. 18 tokens, and of 33 and 64: each way that down has of putting slots in a product's columns."""
    x, router, w_gu, w_down = _layer(dev, 64, 1, D, I, seed=D)
    values = (w_gu, w_down)
    if four:
        values = (Q.quantized(w_gu).to(dev), Q.quantized(w_down).to(dev))
        w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
    one = torch.ones(64, 1, device=dev)
    ref, bound = _reference(x, one, torch.zeros(64, 1, dtype=torch.int64), *values)
    for T in (*range(1, 19), 33, 64):
        out, sel = sg.decode_routed_experts(x[:T], router, w_gu, w_down, 1)
        bad = ~((out.double() - ref[:T]).abs() <= bound[:T])
        assert not bad.any() and not sel.any(), (T, int(bad.sum()), out[bad][:4], ref[:T][bad][:4])


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("which,least", [("x", -128), ("w_gu", -128), ("w_down", -128), ("w_gu", -124),
                                         ("w_down", -124)])
@pytest.mark.parametrize("T", [1, 9, 24])
def test_subnormal_values(dev, T, which, least, four):
    """Subnormal tokens and weights (4-bit: scales from 2^-127 on) beside large ones count as what they are.  Gate and
    up weights N(0, 2^-6) 2^-128 are nearly all zeros in 4 bits, below 2^-129, half the smallest code; no other case's
    are."""
    x, router, w_gu, w_down = _layer(dev, T, 4, 64, 40, seed=T)
    tiny = {"x": x, "w_gu": w_gu, "w_down": w_down}[which]
    tiny.copy_((tiny.double() * 2.0 ** least).to(torch.bfloat16))
    for t, power in ((x, {"w_gu": 100}.get(which, 0)), (w_gu, {"x": 100, "w_down": 60}.get(which, 0))):
        if power and t is not tiny:
            t.copy_((t.double() * 2.0 ** power).to(torch.bfloat16))
    if which in ("x", "w_gu"):  # h is tiny then: about 2^-60
        w_down.copy_((w_down.double() * 2.0 ** 60).to(torch.bfloat16))
    values = (w_gu, w_down)
    if four:
        values = (Q.quantized(w_gu).to(dev), Q.quantized(w_down).to(dev))
        w_gu, w_down = sg.mxfp4_quantize(w_gu), sg.mxfp4_quantize(w_down)
    out, _ = _check(x, router, w_gu, w_down, 2, values=values)
    assert out.any(1).all() or (four and (which, least) == ("w_gu", -128))
