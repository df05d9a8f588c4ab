"""CPU tests of the 4-bit operators: the oracle's rounding, the layout's way
from and to rows, the refusals of the C ABI and of the wrappers before anything
is launched, and the shapes that a compiled graph is told."""
import pytest
import torch

import spark_gpt_amd as sg
from oracle import mxfp4 as O
from spark_gpt_amd import _lib, ops, torch_ops


def test_oracle_rounds_ties_to_even_codes():
    x = torch.zeros(1, 32)
    x[0, :14] = torch.tensor([4.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.0, 7.99, -0.75, -0.1])
    codes, scales = O.quantize(x)
    assert scales.tolist() == [[127]]
    assert O.values(codes, scales)[0, :14].tolist() == [4, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, 6, -1, 0]
    assert O.quantize(torch.tensor([[0.0, 2.0 ** -140]]))[1].tolist() == [[0]]
    assert O.quantize(torch.tensor([[float("inf"), 1.0]]))[1].tolist() == [[255]]


@pytest.mark.parametrize("shape", [(1, 1), (16, 128), (17, 129), (5, 63), (2, 33, 260), (3, 0, 40)])
def test_layout_round_trip(shape):
    g = torch.Generator().manual_seed(sum(shape))
    columns = shape[-1]
    codes = torch.randint(0, 256, (*shape[:-1], -(-columns // 2)), generator=g, dtype=torch.uint8)
    if columns % 2:
        codes[..., -1] &= 15
    scales = torch.randint(0, 256, (*shape[:-1], -(-columns // 32)), generator=g, dtype=torch.uint8)
    q = sg.MXFP4.from_rows(codes, scales, columns)
    assert q.shape == shape and q.codes.shape[-3:] == (-(-columns // 128), -(-shape[-2] // 16) * 16, 64)
    back = q.rows()
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)
    for r, c in ((0, 0), (shape[-2] - 1, columns - 1)):
        if 0 in shape:
            continue
        byte = q.codes.reshape(-1, *q.codes.shape[-3:])[0, c // 128, r, c % 128 // 2]
        assert (int(byte) >> 4 * (c % 2)) & 15 == (int(codes.reshape(-1, *codes.shape[-2:])[0, r, c // 2]) >> 4 * (c % 2)) & 15
    assert int(q.codes.sum()) == int(codes.sum()) and int(q.scales.sum()) == int(scales.sum())  # the padding is zero


def test_c_abi_refuses_before_launch():
    lib = _lib.load()
    assert lib.sfp8_mxfp4_code_bytes(17, 129) == 2 * 32 * 64
    assert lib.sfp8_mxfp4_code_bytes(0, 5) == lib.sfp8_mxfp4_code_bytes(5, 0) == 0
    assert lib.sfp8_mxfp4_code_bytes(-1, 5) == lib.sfp8_mxfp4_code_bytes(5, 2 ** 31 + 1) == -1

    def quant(x=16, dtype=1, batch=1, R=4, C=64, ld=64, bs=0, codes=16, scales=16, ct=None, st=None):
        return lib.sfp8_mxfp4_quantize(x, dtype, batch, R, C, ld, bs, codes, scales, ct, st, None)

    assert quant(x=None) == quant(codes=None) == quant(scales=None) == quant(ct=16) == -1
    for bad in (dict(dtype=3), dict(dtype=-1), dict(batch=-1), dict(R=-1), dict(C=2 ** 31 + 1), dict(ld=-1), dict(bs=-1),
                dict(batch=2 ** 20, R=2 ** 20, C=2 ** 20)):
        assert quant(**bad) == -2, bad
    assert quant(x=17) == quant(codes=8) == quant(scales=2) == quant(dtype=0, x=18) == -3
    assert quant(R=0, x=None) == quant(C=0) == quant(batch=0) == quant(codes=None, scales=None) == 0

    deq = lambda codes=16, scales=16, R=4, C=64, out=16, dtype=0: \
        lib.sfp8_mxfp4_dequantize(codes, scales, 1, R, C, out, dtype, None)
    assert deq(codes=None) == deq(scales=None) == deq(out=None) == -1
    assert deq(dtype=3) == deq(R=-1) == deq(C=-1) == -2
    assert deq(codes=8) == deq(scales=2) == deq(out=8) == -3
    assert deq(R=0) == deq(C=0) == 0

    gemm = lambda a=16, sa=16, b=16, sb=16, M=4, N=4, K=64, out=16, dtype=1, ws=None, bytes=0: \
        lib.sfp8_mxfp4_gemm(a, sa, b, sb, M, N, K, out, dtype, ws, bytes, None)
    assert gemm(a=None) == gemm(sa=None) == gemm(b=None) == gemm(sb=None) == gemm(out=None) == -1
    for bad in (dict(M=-1), dict(N=-1), dict(K=-1), dict(dtype=3), dict(M=2 ** 31 + 1)):
        assert gemm(**bad) == -2, bad
    assert gemm(a=8) == gemm(sb=2) == gemm(out=8) == -3
    assert gemm(M=0) == gemm(N=0) == 0

    space = lib.sfp8_mxfp4_gemm_workspace_bytes
    assert space(4, 4, 64) == space(0, 4, 1 << 20) == space(4, 0, 1 << 20) == space(16384, 4096, 65536) == 0
    assert space(128, 128, 65536) == 16 * 128 * 128 * 4 and space(3, 3, 49152) == 12 * 12 * 4
    assert space(-1, 4, 4) == space(4, 2 ** 31 + 1, 4) == -1
    shared = dict(M=128, N=128, K=65536)
    assert gemm(**shared) == -1 and gemm(**shared, ws=8, bytes=1 << 30) == -3
    assert gemm(**shared, ws=16, bytes=space(128, 128, 65536) - 1) == -4

    rows = lambda x=16, xt=1, ld=64, b=16, sb=16, M=4, N=4, K=64, out=16, dtype=1: \
        lib.sfp8_mxfp4_gemm_rows(x, xt, ld, b, sb, M, N, K, out, dtype, None)
    assert rows(x=None) == rows(b=None) == rows(sb=None) == rows(out=None) == -1
    for bad in (dict(M=17), dict(M=-1), dict(N=1 << 27), dict(xt=3), dict(dtype=-1), dict(ld=-1), dict(N=-1)):
        assert rows(**bad) == -2, bad
    assert rows(x=17) == rows(b=8) == rows(sb=2) == rows(out=8) == -3
    assert rows(M=0) == 0


def test_wrappers_refuse_host_tensors_and_misfits():
    x = torch.zeros(4, 64)
    q = sg.MXFP4.from_rows(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 64)
    for f in (lambda: sg.mxfp4_quantize(x), lambda: sg.mxfp4_dequantize(q), lambda: sg.mxfp4_matmul(q, q),
              lambda: sg.mxfp4_linear(x, q), lambda: sg.mxfp4_linear(x, x), lambda: ops.mxfp4_quantize(x, True, False)):
        with pytest.raises(ValueError, match="ROCm device"):
            f()
    with pytest.raises(ValueError, match="along"):
        sg.mxfp4_quantize(x, along="diagonal")
    with pytest.raises(ValueError, match="rows of one length"):
        sg.mxfp4_matmul(q, sg.MXFP4(q.codes, q.scales, (4, 32)))
    with pytest.raises(TypeError, match="MXFP4"):
        sg.mxfp4_matmul(x, q)
    with pytest.raises(TypeError, match="MXFP4"):
        sg.mxfp4_dequantize((q.codes, q.scales))
    with pytest.raises(ValueError, match="2-D"):
        sg.mxfp4_matmul(q, sg.MXFP4(q.codes[None], q.scales[None], (1, 4, 64)))
    for other in (sg.MXFP4(q.codes, q.scales, (1, 4, 64)), sg.MXFP4(q.codes[None], q.scales[None], (4, 64)),
                  sg.MXFP4(q.codes[None], q.scales[None], (2, 4, 64))):
        with pytest.raises(ValueError, match="do not fit"):
            sg.mxfp4_dequantize(other)
    with pytest.raises(ValueError, match=r"\[\.\.\., 64\]"):
        sg.mxfp4_linear(x[:, :32], q)
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        sg.mxfp4_linear(x, x[0])
    with pytest.raises(ValueError, match="no gradient"):
        sg.mxfp4_linear(x.requires_grad_(True), q)
    for codes, scales in ((torch.zeros(4, 32), torch.zeros(4, 2)), (q.rows()[0][:3], q.rows()[1]),
                          (q.rows()[0], q.rows()[1][:, :1]), (q.rows()[0][0], q.rows()[1][0])):
        with pytest.raises(ValueError):
            sg.MXFP4.from_rows(codes, scales, 64)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(3, 17, 130)
        parts = torch.ops.sparkfp8.mxfp4_quantize(x, True, True)
        assert [tuple(p.shape) for p in parts] == [(3, 2, 32, 64), (3, 2, 32, 4), (3, 1, 144, 64), (3, 1, 144, 4)]
        assert len(torch.ops.sparkfp8.mxfp4_quantize(x, False, True)) == 2
        out = torch.ops.sparkfp8.mxfp4_dequantize(parts[0], parts[1], 17, 130, torch.bfloat16)
        assert out.shape == (3, 17, 130) and out.dtype == torch.bfloat16
        a, s = torch.ops.sparkfp8.mxfp4_quantize(x[0], True, False)
        y = torch.ops.sparkfp8.mxfp4_matmul(a, s, a, s, 17, 17, 130, torch.float16)
        assert y.shape == (17, 17) and y.dtype == torch.float16
        assert torch.ops.sparkfp8.mxfp4_rows_matmul(x[0, :5], a, s, 17, torch.float32).shape == (5, 17)


def test_linear_refuses_tangents():
    """A dual tensor requires no gradient: its tangent is refused, not dropped."""
    from torch.autograd import forward_ad

    x = torch.zeros(4, 64)
    q = sg.MXFP4.from_rows(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for args in ((dual, q), (dual, x), (x, dual)):
            for on in (True, False):
                with torch.set_grad_enabled(on), pytest.raises(NotImplementedError, match="forward-mode"):
                    sg.mxfp4_linear(*args)
        with pytest.raises(ValueError, match="ROCm device"):
            sg.mxfp4_linear(x, q)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: sg.mxfp4_linear(v, q), (x,), (x,))


def test_rows_product_refuses_grids_past_the_limit():
    """16 columns take 512 threads, and a grid has less than 2^32 of them."""
    rows = lambda N: _lib.load().sfp8_mxfp4_gemm_rows(16, 1, 64, 16, 16, 4, N, 64, 16, 1, None)
    assert rows((1 << 27) - 1) == rows((1 << 27) - 15) == -2
    assert sg.mxfp4.ROWS_MAX_N == (1 << 27) - 16


def test_product_refuses_grids_past_the_limit():
    """Tiles of 256 x 256 take 512 threads: one row of them reaches 2^32 before those of 128 x 128 are too many."""
    gemm = lambda N, K: _lib.load().sfp8_mxfp4_gemm(16, 16, 16, 16, 1, N, K, 16, 1, None, 0, None)
    assert gemm((1 << 31) - 1024, 2560) == gemm((1 << 31) - 2047, 2560) == -2
    assert gemm((1 << 31) - 1023, 64) == -2
