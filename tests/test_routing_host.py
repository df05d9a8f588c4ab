"""CPU tests of the routing and clipping operators: the oracle's formulas
against differences, the refusals of the C ABI and of the wrappers before
anything is launched, workspace sizes, and the shapes that a compiled graph is
told."""
import ctypes

import pytest
import torch

import spark_gpt_amd as sg
from oracle import routing as O
from spark_gpt_amd import _lib, ops, torch_ops


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_oracle_gradient_matches_differences(score, renorm):
    """Central differences of the weights, the selection held: with h = 1e-5 the
    difference's own error is h^2 times a third derivative (below 1) over 6 and
    2^-53 / h of rounding, 3e-11 in all, times the |dw| of about 4."""
    g = torch.Generator().manual_seed(3)
    T, E, k, scale, h = 3, 7, 3, 2.5, 1e-5
    low = torch.randn(T, E, generator=g, dtype=torch.float64)
    dw = torch.randn(T, k, generator=g, dtype=torch.float64)
    _, sel = O.route(low, k, score=score, renormalize=renorm, scale=scale)
    grad, size = O.route_grad(low, sel, dw, score=score, renormalize=renorm, scale=scale)
    for t in range(T):
        for e in range(E):
            ends = []
            for d in (h, -h):
                x = low[t].numpy().copy()
                x[e] += d
                ends.append(scale * float((torch.from_numpy(O.shares(x, sel[t].tolist(), score, renorm)) * dw[t]).sum()))
            assert abs((ends[0] - ends[1]) / (2 * h) - float(grad[t, e])) < 1e-9
    assert (size >= grad.abs() - 1e-12).all()


def test_oracle_selection_rules():
    """Ties to the lowest index, NaN first, -inf never, groups by their best."""
    inf, nan = float("inf"), float("nan")
    sel = O.route(torch.tensor([[1.0, 3.0, 3.0, 2.0], [-inf, 0.0, nan, inf], [-inf] * 4, [-inf, 5.0, -inf, -inf]]), 2)[1]
    assert sel.tolist() == [[1, 2], [2, 3], [-1, -1], [1, -1]]
    low = torch.tensor([[9.0, 0.0, 7.0, 7.0, 8.0, 1.0]])
    kw = dict(groups=3, top_groups=1, score="sigmoid")
    assert O.route(low, 2, group_best=1, **kw)[1].tolist() == [[0, 1]]
    assert O.route(low, 2, group_best=2, **kw)[1].tolist() == [[2, 3]]
    assert O.route(low, 1, score="sigmoid", bias=torch.tensor([-1.0, 0, 0, 0, 0, 0]))[1].tolist() == [[4]]
    tok, inv, off = O.expert_order(torch.tensor([[2, 0], [-1, 2], [0, 9]]), 3)
    assert tok.tolist() == [0, 2, 0, 1, 1, 2] and inv.tolist() == [2, 0, -1, 3, 1, -1] and off.tolist() == [2, 2, 4]


def test_c_abi_refuses_before_launch():
    lib = _lib.load()

    def route(logits=16, dtype=0, T=4, E=64, ld=64, bias=None, mask=None, score=0, groups=1, top_groups=1, best=1, k=4,
              renorm=1, scale=1.0, w=16, sel=16, picked=16):
        return lib.sfp8_moe_route(logits, dtype, T, E, ld, bias, mask, score, groups, top_groups, best, k, renorm,
                                  scale, w, sel, picked, None)

    assert route(logits=None) == route(w=None) == route(sel=None) == -1
    for bad in (dict(dtype=3), dict(T=-1), dict(T=2 ** 25 + 1), dict(E=0), dict(E=1025), dict(ld=-1), dict(score=2),
                dict(groups=0), dict(groups=3), dict(groups=65, E=65), dict(groups=4, top_groups=5),
                dict(top_groups=0), dict(best=3), dict(k=0), dict(k=65), dict(groups=16, top_groups=2, k=9)):
        assert route(**bad) == -2, bad
    assert route(T=0, logits=None, w=None, sel=None) == 0  # no tokens: nothing is launched

    def bwd(dw=16, sel=16, picked=16, logits=16, dtype=0, T=4, E=64, score=0, k=4, renorm=0, d=16):
        return lib.sfp8_moe_route_bwd(dw, sel, picked, logits, dtype, T, E, E, score, k, renorm, 1.0, d, None)

    assert bwd(dw=None) == bwd(sel=None) == bwd(picked=None) == bwd(logits=None) == bwd(d=None) == -1
    for bad in (dict(dtype=-1), dict(E=1025), dict(k=65), dict(E=3), dict(score=-1), dict(T=-1)):
        assert bwd(**bad) == -2, bad

    order = lib.sfp8_moe_expert_order
    assert order(None, 8, 2, 4, 16, 16, 16, None, 0, None) == -1
    assert order(16, 8, 2, 4, 16, 16, None, None, 0, None) == -1
    for R, k, E in ((9, 2, 4), (8, 0, 4), (8, 2, 0), (8, 2, 1025), (2 ** 30 + 2, 2, 4), (-2, 2, 4)):
        assert order(16, R, k, E, 16, 16, 16, 16, 0, None) == -2
    assert order(16, 1 << 20, 2, 256, 16, 16, 16, None, 0, None) == -4
    assert order(16, 1 << 20, 2, 256, 16, 16, 16, 16, 100, None) == -4

    comb = lib.sfp8_moe_combine
    assert comb(None, 1, 8, 64, 16, 16, 4, 2, 16, None) == comb(16, 1, 8, 64, None, 16, 4, 2, 16, None) == -1
    assert comb(16, 7, 8, 64, 16, 16, 4, 2, 16, None) == comb(16, 1, 8, 0, 16, 16, 4, 2, 16, None) == -2
    assert comb(16, 1, 8, 64, 16, 16, 4, 65, 16, None) == comb(16, 1, -1, 64, 16, 16, 4, 2, 16, None) == -2
    cb = lib.sfp8_moe_combine_bwd
    assert cb(None, 16, 1, 8, 64, 16, 16, 4, 2, 16, 4, 16, 16, None) == -1
    assert cb(16, 16, 1, 8, 64, 16, 16, 4, 2, None, 4, 16, 16, None) == -1  # drows needs the offsets
    assert cb(16, 16, 1, 8, 64, 16, 16, 4, 2, 16, 0, 16, 16, None) == -2
    assert cb(16, 16, 1, 8, 64, 16, 16, 4, 2, None, 4, None, None, None) == 0  # nothing asked for

    n = (ctypes.c_int64 * 2)(4, 4)
    dt = (ctypes.c_int * 2)(0, 1)
    p = (ctypes.c_void_p * 2)(16, 32)
    addr = ctypes.addressof
    norm = lambda count=2, g=addr(p), nn=addr(n), d=addr(dt), out=16, ws=16, wsn=1 << 20: \
        lib.sfp8_grad_norm(count, g, nn, d, out, ws, wsn, None)
    assert norm(g=None) == norm(nn=None) == norm(out=None) == norm(ws=None) == -1
    assert norm(count=-1) == -2 and norm(wsn=10) == -4
    assert norm(d=addr((ctypes.c_int * 2)(0, 3))) == -2
    assert norm(nn=addr((ctypes.c_int64 * 2)(4, -1))) == -2
    assert norm(g=addr((ctypes.c_void_p * 2)(16, 33))) == -3
    assert norm(g=addr((ctypes.c_void_p * 2)(16, None))) == -1
    clip = lambda out=addr(p), mx=1.0: lib.sfp8_grad_clip(2, addr(p), out, addr(n), addr(dt), mx, 16, 16, 1 << 20, None)
    assert clip(out=None) == -1 and clip(mx=-1.0) == -2 and clip(mx=float("nan")) == -2
    assert clip(out=addr((ctypes.c_void_p * 2)(18, 32))) == -3


def test_workspace_sizes():
    q = lambda R, E: _lib.query("sfp8_moe_expert_order_workspace_ints", R, E)
    assert q(0, 8) == q(4096, 8) == 0  # one work-group needs none
    assert q(4097, 8) == 3 * 12 and q(65536 * 8, 256) == 256 * 260  # rows of E + 1 bins, in fours
    assert q(65536 * 8, 1023) == 128 * 1024
    assert q(1 << 30, 1024) == 256 * 1028  # never more than 256 work-groups
    assert q(-1, 8) == q(8, 0) == q(8, 1025) == q((1 << 30) + 1, 8) == -1
    assert _lib.query("sfp8_grad_norm_workspace_doubles", -1) == -1
    assert _lib.query("sfp8_grad_norm_workspace_doubles", 0) > 0


def test_wrappers_refuse_host_tensors():
    f, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    w = torch.zeros(4, 2)
    off = torch.zeros(8, dtype=torch.int32)
    calls = {"moe_route": (f, None, None, "softmax", 1, 1, 1, 2, True, 1.0),
             "moe_route_bwd": (w, i, w, f, "softmax", True, 1.0), "moe_expert_order": (i, 8),
             "moe_combine": (f, w, i.view(-1)), "moe_combine_bwd": (f, f, w, i.view(-1), off),
             "grad_norm": ([f],), "clip_grads": ([f], 1.0)}
    for name, args in calls.items():
        with pytest.raises(ValueError, match="ROCm device tensor"):
            getattr(ops, name)(*args)
    assert set(calls) == set(ops._NATIVE_STEP)
    for call in (lambda: sg.route_tokens(f, 2), lambda: sg.expert_order(i, 8),
                 lambda: sg.combine_experts(f, w, i.view(-1), off), lambda: sg.grad_norm([f]),
                 lambda: sg.clip_grads([f], 1.0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: sg.grad_norm([]), lambda: sg.clip_grads([], 1.0)):
        with pytest.raises(ValueError, match="at least one"):
            call()
    p = torch.nn.Parameter(f.clone())
    assert float(sg.clip_grad_norm_([p], 1.0)) == 0.0  # no gradient yet
    p.grad = f
    with pytest.raises(ValueError):
        sg.clip_grad_norm_(p, 1.0)


def test_routed_experts_refuse_other_shapes():
    """One row of logits for each token and one column for each expert: a plan of
    more experts than there are weights would read past them."""
    m = torch.nn.Module()
    m.gate_up_proj = torch.nn.Parameter(torch.zeros(4, 256, 128))
    x = torch.zeros(6, 128, dtype=torch.bfloat16)
    for shape in ((6, 5), (6, 3), (5, 4), (4,)):
        with pytest.raises(ValueError, match="one row for each token"):
            sg.fp8_routed_experts(x, torch.zeros(shape), m, 2)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        low = torch.empty(6, 12, dtype=torch.bfloat16, device="cuda")
        w, sel, picked = torch.ops.sparkfp8.route_fwd(low, None, None, "sigmoid", 3, 2, 2, 4, True, 1.0)
        assert w.shape == sel.shape == picked.shape == (6, 4)
        assert (w.dtype, sel.dtype, picked.dtype) == (torch.float32, torch.int64, torch.float32)
        d = torch.ops.sparkfp8.route_bwd(w, sel, picked, low, "sigmoid", True, 1.0)
        assert d.shape == low.shape and d.dtype == low.dtype
        tok, inv, off = torch.ops.sparkfp8.expert_order(sel, 12)
        assert tok.shape == inv.shape == (24,) and off.shape == (12,)
        assert (tok.dtype, inv.dtype, off.dtype) == (torch.int64, torch.int64, torch.int32)
        rows = torch.empty(24, 40, dtype=torch.bfloat16, device="cuda")
        out = torch.ops.sparkfp8.combine_fwd(rows, w, inv)
        assert out.shape == (6, 40) and out.dtype == torch.bfloat16
        dr, dw = torch.ops.sparkfp8.combine_bwd(out, rows, w, inv, off)
        assert dr.shape == rows.shape and dr.dtype == rows.dtype and dw.shape == w.shape and dw.dtype == torch.float32
    assert torch_ops.route_fwd is not None


def test_combine_of_any_slots_refuses_before_launch():
    q = lambda *a: _lib.query("sfp8_moe_combine_bwd_any_workspace_ints", *a)
    assert q(8, 4, 2) == 8 + 2 and q(9, 3, 3) == 9 + 3 and q(0, 0, 1) == 0 and q(5, 0, 2) == 5
    assert q(-1, 4, 2) == q(8, -1, 2) == q(8, 2 ** 25 + 1, 2) == q(8, 4, 0) == q(8, 4, 65) == -1
    cb = _lib.load().sfp8_moe_combine_bwd_any

    def call(dout=16, rows=16, dtype=1, R=8, D=64, w=16, inv=16, T=4, k=2, dr=16, dw=16, ws=16, ints=10):
        return cb(dout, rows, dtype, R, D, w, inv, T, k, dr, dw, ws, ints, None)

    assert call(dout=None) == call(rows=None) == call(w=None) == call(inv=None) == -1
    for bad in (dict(dtype=3), dict(R=-1), dict(D=0), dict(T=-1), dict(T=2 ** 25 + 1), dict(k=0), dict(k=65)):
        assert call(**bad) == -2, bad
    assert call(ws=None) == call(ints=9) == call(ws=None, dw=None) == -4
    assert call(dr=None, dw=None) == call(T=0, R=0) == call(R=0, dw=None, T=4) == 0  # nothing to write
