"""CPU tests of the experts' layer for a few tokens: workspace sizes, the
refusals of the C ABI and of the wrapper before anything is launched, and the
shapes that a compiled graph is told."""
import pytest
import torch

import spark_gpt_amd as sg
from spark_gpt_amd import _lib


def test_workspace_sizes():
    q = lambda *a: _lib.query("sfp8_moe_decode_workspace_bytes", *a)
    # logits [T, E] in 64 bits, weights [T, k], the plan, beyond 16 tokens a counter for each 32 columns and sums in 32
    # bits for each share of the work, h in two parts of whole 512s; each from a 256-byte boundary
    assert q(4, 128, 8, 2048, 768) == 4096 + 256 + 8448 + 32 * 2 * 1024 * 2
    assert q(64, 8, 2, 1024, 16) == 4096 + 512 + 2304 + 256 + 8 * 64 * 1024 * 4 + 128 * 2 * 512 * 2
    assert q(64, 8, 2, 8192, 16) == 4096 + 512 + 2304 + 128 * 2 * 512 * 2  # 256 column blocks: no sharing
    assert q(0, 8, 2, 64, 16) >= 0
    for bad in ((65, 8, 2, 64, 16), (-1, 8, 2, 64, 16), (4, 0, 1, 64, 16), (4, 1025, 2, 64, 16), (4, 8, 0, 64, 16),
                (4, 8, 9, 64, 16), (4, 100, 65, 64, 16), (4, 8, 2, 64, 12), (4, 8, 2, 64, 0), (4, 8, 2, 60, 16),
                (4, 8, 2, 8, (1 << 20) + 8), (4, 8, 2, 1 << 16, 1 << 14)):
        assert q(*bad) == -1, bad


def test_c_abi_refuses_before_launch():
    lib = _lib.load()

    def call(x=16, ldx=64, T=4, D=64, router=16, rt=1, E=8, gu=16, gs=None, down=16, ds=None, I=16, bias=None, mask=None,
             score=0, groups=1, top_groups=1, best=1, k=2, sel=16, out=16, ws=16, n=1 << 20):
        return lib.sfp8_moe_decode(x, ldx, T, D, router, rt, E, gu, gs, down, ds, I, bias, mask, score, groups, top_groups,
                                   best, k, 1, 1.0, sel, out, ws, n, None)

    for name in ("x", "router", "gu", "down", "sel", "out", "ws"):
        assert call(**{name: None}) == -1, name
    for bad in (dict(T=65), dict(T=-1), dict(D=60), dict(D=0), dict(I=12), dict(I=0), dict(E=0), dict(E=1025), dict(k=0),
                dict(k=9), dict(rt=2), dict(rt=-1), dict(ldx=-1), dict(score=2), dict(groups=3), dict(groups=0),
                dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(groups=4, top_groups=1, k=3),
                dict(best=0), dict(gs=16), dict(ds=16), dict(E=65, groups=65),
                dict(D=1 << 16, I=1 << 14)):
        assert call(**bad) == -2, bad
    for bad in (dict(x=17), dict(router=17), dict(rt=0, router=18), dict(gu=8), dict(down=24), dict(gs=18, ds=16),
                dict(out=8), dict(ws=8), dict(sel=4), dict(bias=18)):
        assert call(**bad) == -3, bad
    assert call(n=100) == -4
    assert call(T=0, x=None) == 0


def test_wrapper_refuses_host_tensors_and_misfits():
    x, router = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(4, 64)
    w_gu, w_down = torch.zeros(4, 32, 64, dtype=torch.bfloat16), torch.zeros(4, 64, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        sg.decode_routed_experts(x, router, w_gu, w_down, 2)
    with pytest.raises(ValueError, match="do not fit"):
        sg.decode_routed_experts(x, router, w_gu[:, :30], w_down, 2)
    with pytest.raises(ValueError, match="router"):
        sg.decode_routed_experts(x, router[:3], w_gu, w_down, 2)
    with pytest.raises(ValueError, match="no gradient"):
        sg.decode_routed_experts(x, router.requires_grad_(True), w_gu, w_down, 2)
    q = sg.MXFP4.from_rows(torch.zeros(4, 32, 32, dtype=torch.uint8), torch.zeros(4, 32, 2, dtype=torch.uint8), 64)
    with pytest.raises(TypeError, match="both"):
        sg.decode_routed_experts(x, router.detach(), q, w_down, 2)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, router = torch.empty(3, 64, dtype=torch.bfloat16), torch.empty(8, 64)
        out, sel = torch.ops.sparkfp8.moe_decode(x, router, torch.empty(8, 32, 64, dtype=torch.bfloat16), None,
                                                 torch.empty(8, 64, 16, dtype=torch.bfloat16), None, 16, None, None,
                                                 "softmax", 1, 1, 1, 2, True, 1.0)
        assert out.shape == (3, 64) and out.dtype == torch.bfloat16 and sel.shape == (3, 2) and sel.dtype == torch.int64


def test_refuses_tangents():
    """A dual tensor requires no gradient: its tangent is refused, not dropped."""
    from torch.autograd import forward_ad

    x, router = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(4, 64)
    w_gu, w_down = torch.zeros(4, 32, 64, dtype=torch.bfloat16), torch.zeros(4, 64, 16, dtype=torch.bfloat16)
    args, bias = [x, router, w_gu, w_down], torch.zeros(4)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for i in range(4):
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                sg.decode_routed_experts(*args[:i], dual(args[i]), *args[i + 1:], 2)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sg.decode_routed_experts(*args, 2, bias=dual(bias))
        with pytest.raises(ValueError, match="ROCm device"):
            sg.decode_routed_experts(*args, 2, bias=bias)
