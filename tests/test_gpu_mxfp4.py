"""GPU tests of the 4-bit operators against their 64-bit restatement.

Codes and scales are compared as they are.  Products are compared exactly where
32 bits hold every partial sum: with all scales 2^0 a product of two values is a
multiple of 1/4 of at most 36, so sums of up to 2^17 of them are exact in any
order.  Elsewhere a sum of K products in 32 bits is off by at most (K - 1) 2^-24
of the sum of their sizes in any order, twice that where the adders truncate, and
the result once more by half a step of its type."""
import pytest
import torch

import spark_gpt_amd as sg
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _randn(dev, *shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


def _check_codes(q, x):
    """q is the quantised x, padding zero, and its values come back."""
    codes, scales = O.quantize(x)
    assert tuple(q.shape) == tuple(x.shape)
    packed = torch.nn.functional.pad(codes, (0, codes.shape[-1] % 2))
    packed = packed[..., ::2] + 16 * packed[..., 1::2]
    want = sg.MXFP4.from_rows(packed, scales, x.shape[-1])
    bad = (scales == 255).repeat_interleave(32, -1)[..., :x.shape[-1]]  # a NaN block's codes stand for nothing
    if not bad.any():
        assert torch.equal(q.codes.cpu(), want.codes)
    assert torch.equal(q.scales.cpu(), want.scales)
    values = O.values(codes, scales)
    for dtype in DTYPES.values():
        got = sg.mxfp4_dequantize(q, dtype).cpu()
        ref = values.to(dtype)
        assert got.dtype == dtype and torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got.nan_to_num(0.0), ref.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 32), (3, 31), (16, 128), (17, 129), (128, 128), (130, 260), (1, 1000),
                                 (257, 40), (300, 1001), (64, 4096), (4100, 1000), (33000, 130)])
def test_quantize(dev, R, C, dtype):
    x = _randn(dev, R, C, seed=R + C, dtype=DTYPES[dtype]) * torch.exp(2 * _randn(dev, C, seed=1)).to(DTYPES[dtype])
    rows, columns = sg.mxfp4_quantize(x, along="both")
    _check_codes(rows, x)
    _check_codes(columns, x.t())
    for along, want in (("rows", rows), ("columns", columns)):
        one = sg.mxfp4_quantize(x, along=along)
        assert torch.equal(one.codes, want.codes) and torch.equal(one.scales, want.scales) and one.shape == want.shape


def test_quantize_every_bf16_pattern(dev):
    """All bit patterns beside largest values of every exponent: subnormal blocks, the largest, infinities and NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    _check_codes(sg.mxfp4_quantize(bits.view(-1, 32).to(dev)), bits.view(-1, 32))
    finite = bits[torch.isfinite(bits.float())]
    for e in (-133, -127, -126, -125, -60, 0, 1, 60, 126, 127):
        x = torch.full((finite.numel(), 32), 0.0, dtype=torch.bfloat16)
        x[:, 0] = 2.0 ** e
        x[:, 1:] = torch.where(finite.float().abs() < 2.0 ** min(e + 1, 127), finite, 0)[:, None]
        x = x.unique(dim=0)
        q = sg.mxfp4_quantize(x.to(dev))
        codes, scales = O.quantize(x)
        assert torch.equal(q.rows()[1].cpu(), scales)
        assert torch.equal(q.rows()[0].cpu(), codes[:, ::2] + 16 * codes[:, 1::2])


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_quantize_special_values(dev, dtype):
    t = DTYPES[dtype]
    x = _randn(dev, 40, 256, seed=3).to(t)
    x[1] = 0.0
    x[2] = -0.0
    x[3, 5] = float("inf")
    x[4, 40] = float("nan")
    x[5, 64:96] = -float("inf")
    x[6] *= torch.finfo(t).tiny
    x[7] = torch.finfo(t).tiny * torch.finfo(t).eps  # the smallest subnormal
    x[8] = torch.finfo(t).max
    x[9, 0] = torch.finfo(t).max
    rows, columns = sg.mxfp4_quantize(x, along="both")
    _check_codes(rows, x)
    _check_codes(columns, x.t())


def test_quantize_strides_offsets_and_batches(dev):
    base = _randn(dev, 70, 300, seed=5, dtype=torch.bfloat16)
    for x in (base[3:60, 7:250], base[::3], base[:, ::2], base.t(), base[5], base[:, :1], base[:1, 1:34]):
        x = x if x.dim() == 2 else x[None].expand(20, -1)
        _check_codes(sg.mxfp4_quantize(x), x)
        _check_codes(sg.mxfp4_quantize(x, along="columns"), x.t())
    batch = _randn(dev, 3, 50, 140, seed=6)
    for x in (batch, batch[:, 1:, 3:], batch.transpose(0, 1), batch.transpose(1, 2)):
        rows, columns = sg.mxfp4_quantize(x, along="both")
        _check_codes(rows, x)
        _check_codes(columns, x.transpose(1, 2))
    for shape in ((0, 64), (5, 0), (2, 0, 3), (0, 4, 4)):
        q = sg.mxfp4_quantize(torch.zeros(shape, device=dev))
        assert sg.mxfp4_dequantize(q).shape == shape
    q = sg.mxfp4_quantize(base)
    again = sg.MXFP4.from_rows(*q.rows(), 300)
    assert torch.equal(again.codes, q.codes) and torch.equal(again.scales, q.scales)


def _operand(dev, R, K, seed, exponents=(0, 0)):
    """Random codes with scales 2^exponents."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (R, K), generator=g, dtype=torch.uint8)
    scales = torch.randint(127 + exponents[0], 128 + exponents[1], (R, -(-K // 32)), generator=g, dtype=torch.uint8)
    packed = torch.nn.functional.pad(codes, (0, K % 2))
    q = sg.MXFP4.from_rows(packed[:, ::2] + 16 * packed[:, 1::2], scales, K)
    return sg.MXFP4(q.codes.to(dev), q.scales.to(dev), q.shape), O.values(codes, scales)


SHAPES = [(1, 1, 1), (1, 16, 32), (3, 17, 129), (16, 64, 128), (8, 4096, 512), (17, 33, 4096), (64, 64, 640),
          (65, 130, 200), (128, 128, 256), (100, 1000, 1000), (256, 256, 384), (257, 255, 1024), (300, 700, 130),
          (513, 511, 2304), (1003, 2050, 1000), (2048, 1536, 256), (40, 3, 8192), (2, 20000, 96), (4100, 24, 4096),
          (2300, 2304, 2048),
          # every tile shape: 256 x 256 with an odd number of slabs, 64 x 64, 64 x 32, 32 x 32, 16 x 32 and 16 x 16
          (4100, 4100, 4100), (1030, 1000, 2003), (100, 4100, 300), (20, 8200, 130), (7, 8200, 520), (9, 300, 5000)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul_exact(dev, M, N, K):
    """All scales 2^0: every partial sum is exact in 32 bits."""
    (a, av), (b, bv) = _operand(dev, M, K, M + K), _operand(dev, N, K, N + 1)
    ref = (av.to(dev) @ bv.to(dev).T).cpu()
    for dtype in DTYPES.values():
        got = sg.mxfp4_matmul(a, b, dtype)
        assert got.shape == (M, N) and got.dtype == dtype and torch.equal(got.cpu(), ref.to(dtype))


@pytest.mark.parametrize("M,N,K", [(5, 40, 1000), (200, 300, 4000), (700, 900, 2000), (16, 2048, 8192)])
def test_matmul_scales(dev, M, N, K):
    (a, av), (b, bv) = _operand(dev, M, K, 7, (-9, 9)), _operand(dev, N, K, 8, (-14, 3))
    av, bv = av.to(dev), bv.to(dev)
    ref, size = av @ bv.T, av.abs() @ bv.abs().T
    got = sg.mxfp4_matmul(a, b, torch.float32).double()
    assert ((got - ref).abs() <= K * 2.0 ** -23 * size + 2.0 ** -24 * ref.abs()).all()
    # rounding errors that do not add up in one direction: far below the bound over all elements
    assert float((got - ref).norm() / ref.norm()) < 2.0 ** -20
    half = sg.mxfp4_matmul(a, b).double()
    assert ((half - ref).abs() <= K * 2.0 ** -23 * size + 2.0 ** -8 * (1 + 2.0 ** -8) * ref.abs()).all()


def test_matmul_extreme_scales(dev):
    """One block of one operand is NaN: so are its row's results alone.  The smallest and the largest scales."""
    for M, N in ((9, 50), (300, 300)):
        (a, av), (b, bv) = _operand(dev, M, 256, 1), _operand(dev, N, 256, 2)
        a.scales[1, 5, 2] = 255
        got = sg.mxfp4_matmul(a, b, torch.float32).cpu()
        ref = av @ bv.T
        assert got[5].isnan().all() and torch.equal(got[:5].double(), ref[:5]) and torch.equal(got[6:].double(), ref[6:])
        a.scales[1, 5, 2] = 127
        for low, high in ((0, 254), (60, 220), (127 - 100, 127 + 80)):
            a.scales[:, :M] = low
            b.scales[:, :N] = high
            got = sg.mxfp4_matmul(a, b, torch.float32).cpu().double()
            assert torch.equal(got, ref * 2.0 ** (low + high - 254))


@pytest.mark.parametrize("M,N,K", [(1, 8, 49153), (130, 70, 49183), (3, 5, 65536), (700, 768, 16500), (128, 257, 70000)])
def test_matmul_shared(dev, M, N, K):
    """Work-groups that share K: exact sums where every one is exact, again and again and from a graph, a NaN where it is
    one, and the bound of one sum (the shares' sums are as many additions fewer)."""
    assert sg._lib.load().sfp8_mxfp4_gemm_workspace_bytes(M, N, K) > 0
    (a, av), (b, bv) = _operand(dev, M, K, 3), _operand(dev, N, K, 4)
    ref = av.to(dev) @ bv.to(dev).T
    assert torch.equal(sg.mxfp4_matmul(a, b, torch.float32).double(), ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = sg.mxfp4_matmul(a, b, torch.float32)
    for dtype in DTYPES.values():
        got = sg.mxfp4_matmul(a, b, dtype)
        assert got.shape == (M, N) and torch.equal(got, ref.to(dtype))
        graph.replay()
        assert torch.equal(replayed.double(), ref)
    a.scales[-1, 0, 0] = 255
    got = sg.mxfp4_matmul(a, b, torch.float32)
    assert got[0].isnan().all() and torch.equal(got[1:].double(), ref[1:])
    (a, av), (b, bv) = _operand(dev, M, K, 7, (-9, 9)), _operand(dev, N, K, 8, (-14, 3))
    av, bv = av.to(dev), bv.to(dev)
    ref, size = av @ bv.T, av.abs() @ bv.abs().T
    got = sg.mxfp4_matmul(a, b, torch.float32)
    assert ((got.double() - ref).abs() <= K * 2.0 ** -23 * size + 2.0 ** -24 * ref.abs()).all()
    assert torch.equal(got, sg.mxfp4_matmul(a, b, torch.float32))


def test_matmul_shared_unevenly(dev):
    """8300 slabs for 256 work-groups of 33: the last of them have none."""
    K, g = 8300 * 128 - 5, torch.Generator().manual_seed(1)
    signs = lambda rows: 1 - 2 * torch.randint(0, 2, (rows, K), generator=g)
    a, b = signs(2), signs(3)
    quantized = lambda t: sg.mxfp4_quantize(t.to(dev, torch.bfloat16))
    assert torch.equal(sg.mxfp4_matmul(quantized(a), quantized(b), torch.float32).cpu(), (a @ b.T).float())


def test_linear_of_many_tokens(dev):
    """The weight gradient of a small weight over many tokens is the product of the two quantised transposes."""
    x, dy = _randn(dev, 50000, 96, seed=1).bfloat16().requires_grad_(True), _randn(dev, 50000, 40, seed=2).bfloat16()
    w = _randn(dev, 40, 96, seed=3).requires_grad_(True)
    dw, = torch.autograd.grad(sg.mxfp4_linear(x, w), [w], dy)
    columns = lambda t: sg.mxfp4_quantize(t.detach(), along="columns")
    assert torch.equal(dw, sg.mxfp4_matmul(columns(dy), columns(x), torch.float32))


def test_matmul_of_nothing(dev):
    empty = lambda r, c: sg.mxfp4_quantize(torch.zeros(r, c, device=dev))
    assert sg.mxfp4_matmul(empty(0, 64), empty(5, 64)).shape == (0, 5)
    assert sg.mxfp4_matmul(empty(5, 64), empty(0, 64)).shape == (5, 0)
    for M in (3, 300):
        assert torch.equal(sg.mxfp4_matmul(empty(M, 0), empty(4, 0), torch.float32).cpu(), torch.zeros(M, 4))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (1, 4096, 4096), (4, 1000, 77), (16, 130, 300), (13, 33, 64), (17, 512, 40),
                                   (200, 1030, 100), (0, 64, 32)])
def test_linear_serving(dev, T, K, N, dtype):
    """Weights in codes: the same result, bit for bit, as quantising the tokens and multiplying, whose sums agree to
    the order of the sum; from a master without a gradient the same again."""
    x, w = _randn(dev, T, K, seed=T, dtype=DTYPES[dtype]), _randn(dev, N, K, seed=2) * K ** -0.5
    q = sg.mxfp4_quantize(w)
    y = sg.mxfp4_linear(x, q)
    xv, wv = O.quantized(x).to(dev), O.quantized(w).to(dev)
    ref, size = xv @ wv.T, xv.abs() @ wv.abs().T
    half = torch.finfo(DTYPES[dtype]).eps / 2
    tiny = torch.finfo(DTYPES[dtype]).tiny * torch.finfo(DTYPES[dtype]).eps  # the step of results below the normal ones
    assert y.dtype == DTYPES[dtype] and y.shape == (T, N)
    assert ((y.double() - ref).abs() <= K * 2.0 ** -23 * size + half * (1 + 2.0 ** -8) * ref.abs() + tiny).all()
    assert torch.equal(sg.mxfp4_linear(x, w), y)
    with torch.no_grad():
        assert torch.equal(sg.mxfp4_linear(x, w.clone().requires_grad_(True)), y)
    if T:
        assert torch.equal(sg.mxfp4_linear(x[0], q), sg.mxfp4_linear(x[:1], q)[0])
    assert torch.equal(sg.mxfp4_linear(x[None, :, None], q), y[None, :, None])
    wide = torch.full((T, K + 7), float("nan"), device=dev, dtype=DTYPES[dtype])
    wide[:, 3:K + 3] = x
    assert torch.equal(sg.mxfp4_linear(wide[:, 3:K + 3], q), y)
    assert torch.equal(sg.mxfp4_linear(x.t().contiguous().t(), q), y)


def test_linear_serving_special_tokens(dev):
    """A token with a NaN or an infinity is NaN, the others are as without it."""
    x, q = _randn(dev, 6, 300, seed=1, dtype=torch.bfloat16), sg.mxfp4_quantize(_randn(dev, 40, 300, seed=2))
    clean = sg.mxfp4_linear(x, q)
    x[2, 299] = float("nan")
    x[4, 0] = float("inf")
    y = sg.mxfp4_linear(x, q)
    live = [0, 1, 3, 5]
    assert y[[2, 4]].isnan().all() and torch.equal(y[live], clean[live])


def _on_grid(dev, R, C, seed):
    """Values that 4 bits hold exactly along rows and along columns: each block of 32 of either has a 4."""
    g = torch.Generator().manual_seed(seed)
    x = O.GRID[torch.randint(0, 8, (R, C), generator=g)] * (1 - 2 * torch.randint(0, 2, (R, C), generator=g))
    at = (torch.arange(R)[:, None] + torch.arange(C)) % 16 == 0
    return torch.where(at, 4.0, x).float().to(dev)


@pytest.mark.parametrize("T,K,N", [(32, 64, 32), (96, 160, 64), (300, 270, 520), (1030, 520, 260), (16, 32, 16)])
def test_linear_gradient_exact_and_against_differences(dev, T, K, N):
    """On values that the codes hold, the layer is a plain product: its results and gradients are exact, and a step of
    x or w to another such value changes sum(y dy) by gradient times step."""
    x, w, dy = _on_grid(dev, T, K, 1), _on_grid(dev, N, K, 2), _on_grid(dev, T, N, 3)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = sg.mxfp4_linear(xl, wl)
    dx, dw = torch.autograd.grad(y, [xl, wl], dy)
    X, W, D = x.double(), w.double(), dy.double()
    assert torch.equal(y.double(), X @ W.T) and torch.equal(dx.double(), D @ W) and torch.equal(dw.double(), D.T @ X)
    total = lambda a, b: float((sg.mxfp4_linear(a, b).double() * D).sum())
    base = total(x, w)
    for leaf, grad, f in ((x, dx, lambda v: total(v, w)), (w, dw, lambda v: total(x, v))):
        i, j = (leaf.abs() == 1).nonzero()[7].tolist()
        moved = leaf.clone()
        moved[i, j] += 0.5 if leaf[i, j] > 0 else -0.5
        step = float(moved[i, j] - leaf[i, j])
        assert f(moved) - base == float(grad[i, j]) * step


@pytest.mark.parametrize("wtype", ["fp32", "bf16"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", [(1, 40, 24), (7, 200, 130), (129, 1000, 257), (520, 300, 1030)])
def test_linear_gradient_formula(dev, T, K, N, dtype, wtype):
    x, w = _randn(dev, T, K, seed=1, dtype=DTYPES[dtype]), _randn(dev, N, K, seed=2, dtype=DTYPES[wtype])
    dy = _randn(dev, T, N, seed=3, dtype=DTYPES[dtype])
    x.requires_grad_(True)
    w.requires_grad_(True)
    got = sg.mxfp4_linear(x, w)
    dx, dw = torch.autograd.grad(got, [x, w], dy)
    a = lambda t: O.quantized(t).abs()
    sizes = (a(x) @ a(w).T, a(dy) @ a(w.T).T, a(dy.T) @ a(x.T).T)
    for out, ref, size, n, type_ in zip((got, dx, dw), O.linear(x, w, dy), sizes, (K, N, T), (x, x, w)):
        half = torch.finfo(type_.dtype).eps / 2
        assert out.dtype == type_.dtype and out.shape == ref.shape
        assert ((out.detach().cpu().double() - ref).abs()
                <= n * 2.0 ** -23 * size + half * (1 + 2.0 ** -8) * ref.abs() + 2.0 ** -24).all()


def test_linear_gradients_one_at_a_time(dev):
    x, w, dy = (_randn(dev, *s, seed=i, dtype=torch.bfloat16) for i, s in enumerate(((70, 96), (50, 96), (70, 50))))
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(sg.mxfp4_linear(xl, wl), [xl, wl], dy)
    assert torch.equal(torch.autograd.grad(sg.mxfp4_linear(xl, w), [xl], dy)[0], dx)
    assert torch.equal(torch.autograd.grad(sg.mxfp4_linear(x, wl), [wl], dy)[0], dw)
    # a gradient without strides of its own, leading dimensions, no tokens
    y = sg.mxfp4_linear(xl.view(7, 10, 96), wl)
    gx, gw = torch.autograd.grad(y.sum(), [xl, wl])
    ones = torch.autograd.grad(sg.mxfp4_linear(xl, wl), [xl, wl], torch.ones_like(dy))
    assert torch.equal(gx, ones[0]) and torch.equal(gw, ones[1])
    none = torch.zeros(0, 96, device=dev, requires_grad=True)
    gx, gw = torch.autograd.grad(sg.mxfp4_linear(none, wl).sum(), [none, wl])
    assert gx.shape == (0, 96) and torch.equal(gw, torch.zeros_like(w))
    # what the backward pass reads is kept in codes: the leaves may change
    y = sg.mxfp4_linear(xl, wl)
    with torch.no_grad():
        xl.zero_()
        wl.zero_()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, [xl, wl], dy), (dx, dw)))
    y = sg.mxfp4_linear(xl, wl)
    g, = torch.autograd.grad(y, [xl], dy.clone().requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_linear_of_no_tokens_and_no_width(dev):
    """A gradient over no tokens is zero at sizes of every kernel; no width gives zeros; leading dimensions of any kind."""
    for N, K in ((24, 40), (700, 700), (2100, 2000)):
        w = _randn(dev, N, K, seed=1).requires_grad_(True)
        x = torch.zeros(0, 3, K, device=dev, dtype=torch.bfloat16, requires_grad=True)
        y = sg.mxfp4_linear(x, w)
        dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
        assert y.shape == (0, 3, N) and dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))
    w = torch.zeros(5, 0, device=dev)
    for shape in ((4, 0), (2, 3, 0), (0,)):
        y = sg.mxfp4_linear(torch.zeros(shape, device=dev), w)
        assert torch.equal(y, torch.zeros(*shape[:-1], 5, device=dev))
    w = _randn(dev, 30, 64, seed=2).requires_grad_(True)
    x = _randn(dev, 64, seed=3).requires_grad_(True)
    y = sg.mxfp4_linear(x, w)
    assert y.shape == (30,)
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert dx.shape == (64,) and dw.shape == (30, 64)


def test_weights_kept_refuse_a_gradient(dev):
    q = sg.mxfp4_quantize(_randn(dev, 16, 64))
    with pytest.raises(ValueError, match="no gradient"):
        sg.mxfp4_linear(torch.zeros(2, 64, device=dev, requires_grad=True), q)
    with pytest.raises(ValueError, match="do not fit"):
        sg.mxfp4_linear(torch.zeros(2, 300, device=dev), sg.MXFP4(q.codes, q.scales, (16, 300)))
    with pytest.raises(ValueError, match="fp32|float"):
        sg.mxfp4_quantize(torch.zeros(4, 4, device=dev, dtype=torch.float64))
    with pytest.raises(ValueError, match="float"):
        sg.mxfp4_matmul(q, q, torch.float64)
    with pytest.raises(ValueError, match="2-D or 3-D"):
        sg.mxfp4_quantize(torch.zeros(4, device=dev))


def test_layer_of_projections_captured_and_replayed(dev):
    """Two 4-bit projections with a SwiGLU between them, forward and backward, as a training step uses them: captured
    once, replayed with new inputs between eager steps of the same size."""
    T, D, I = 130, 192, 160
    w_gu, w_down = _randn(dev, 2 * I, D, seed=1) * D ** -0.5, _randn(dev, D, I, seed=2) * I ** -0.5
    x, dy = torch.zeros(T, D, device=dev, dtype=torch.bfloat16), torch.zeros(T, D, device=dev, dtype=torch.bfloat16)

    def step(x, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w_gu, w_down)]
        gate, up = sg.mxfp4_linear(leaves[0], leaves[1]).chunk(2, -1)
        y = sg.mxfp4_linear(torch.nn.functional.silu(gate) * up, leaves[2])
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, dy)
    for seed in range(4):
        a, b = _randn(dev, T, D, seed=seed, dtype=torch.bfloat16), _randn(dev, T, D, seed=9 + seed, dtype=torch.bfloat16)
        x.copy_(a)
        dy.copy_(b)
        graph.replay()
        got = [t.clone() for t in out]
        ref = step(a, b)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
        assert all(bool(torch.isfinite(t.float()).all()) and float(t.float().norm()) > 0 for t in got)


def test_other_stream_and_repeats(dev):
    """On another stream, and again: the same bytes."""
    x, w = _randn(dev, 300, 1000, seed=1, dtype=torch.bfloat16), _randn(dev, 700, 1000, seed=2)
    first = sg.mxfp4_linear(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = sg.mxfp4_linear(x, w)
    side.synchronize()
    assert torch.equal(first, second) and torch.equal(first, sg.mxfp4_linear(x, w))


def test_compiled_linear_matches_eager(dev):
    w = _randn(dev, 200, 160, seed=1)

    def f(x, w):
        return torch.nn.functional.silu(sg.mxfp4_linear(x, w)) * 2

    for T in (8, 200):
        x, dy = _randn(dev, T, 160, seed=2, dtype=torch.bfloat16), _randn(dev, T, 200, seed=3, dtype=torch.bfloat16)
        grads = []
        for g in (f, torch.compile(f, fullgraph=True, dynamic=False)):
            leaves = [t.clone().requires_grad_(True) for t in (x, w)]
            y = g(*leaves)
            grads.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
        # silu is compiled by another route: its own rounding comes on top of bf16's
        for p, q in zip(*grads):
            assert float((p.float() - q.float()).norm() / q.float().norm()) < 2.0 ** -5
    codes = sg.mxfp4_quantize(w)
    serve = torch.compile(lambda x: sg.mxfp4_linear(x, codes), fullgraph=True, dynamic=False)
    with torch.no_grad():
        x = _randn(dev, 5, 160, seed=4, dtype=torch.bfloat16)
        assert torch.equal(serve(x), sg.mxfp4_linear(x, codes))


def test_large_offsets(dev):
    """More than 2^31 values and codes past 2^31 bytes: the last rows are right."""
    R, C = 70000, 65536
    x = torch.zeros(R, C, device=dev, dtype=torch.bfloat16)
    tail = _randn(dev, 40, C, seed=1, dtype=torch.bfloat16)
    x[-40:] = tail
    q = sg.mxfp4_quantize(x)
    want = sg.mxfp4_quantize(tail)
    # 70000 is a multiple of 16: the tail's 40 rows are the last of each slab
    assert torch.equal(q.codes[:, -40:], want.codes[:, :40]) and torch.equal(q.scales[:, -40:], want.scales[:, :40])
    assert int(q.codes[:, :-40].max()) == 0
    del x
    back = sg.mxfp4_dequantize(q)
    assert torch.equal(back[-40:], sg.mxfp4_dequantize(want))
    del back
    small = sg.mxfp4_quantize(_randn(dev, 20, C, seed=2))
    assert torch.equal(sg.mxfp4_matmul(q, small)[-40:], sg.mxfp4_matmul(want, small))


def test_no_forward_mode(dev):
    """Tangents are refused on every path; tensors without one pass inside a level."""
    from torch.autograd import forward_ad

    x, w = torch.randn(20, 64, device=dev, dtype=torch.bfloat16), torch.randn(32, 64, device=dev)
    q = sg.mxfp4_quantize(w)
    plain = [sg.mxfp4_linear(v, q) for v in (x, x[:3])]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for v in (dual, dual[:3]):
            for weights in (q, w, w.clone().requires_grad_(True)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    sg.mxfp4_linear(v, weights)
        assert all(torch.equal(sg.mxfp4_linear(v, q), p) for v, p in zip((x, x[:3]), plain))
