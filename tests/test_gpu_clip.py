"""GPU tests of the global gradient norm and clipping against 64 bits.

The squares are summed in 64 bits, so the norm is off by its rounding to fp32,
2^-24 relative (and 1e-9 for up to 10^7 additions of 2^-53).  The factor adds
that, the sum with 1e-6 and the quotient, 2^-24 each; a scaled gradient its
product and half a step of its type."""
import math
from fractions import Fraction

import pytest
import torch

import spark_gpt_amd as sg
from oracle import routing as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NORM_TOL = 2.0 ** -24 * 1.02


def _grads(dev, shapes, dtypes, seed, std=1e-2):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(s, device=dev, generator=g) * std).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def _check(before, after, norm, max_norm):
    ref, factor = O.clip(before, max_norm)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - ref) <= NORM_TOL * ref
    for b, a in zip(before, after):
        if factor == 1.0:
            assert torch.equal(a, b)
            continue
        want = b.double() * factor
        step = 5 * 2.0 ** -24 if b.dtype == torch.float32 else 5 * 2.0 ** -24 + torch.finfo(b.dtype).eps / 2
        tiny = torch.finfo(b.dtype).tiny * torch.finfo(b.dtype).eps
        assert a.dtype == b.dtype and ((a.double() - want).abs() <= step * want.abs() + tiny).all()


SHAPES = {"one": [(1,)], "scalars": [(), (1,), (3,)], "odd": [(7, 13), (1025,), (3, 5, 7), (16384,), (16385,), (32768 + 5,)],
          "weights": [(512, 256), (256, 1024), (256,)] * 3, "empty": [(0,), (4, 0), (5,)],
          "many": [(i % 97 + 1,) for i in range(500)], "large": [(3000, 1111)]}


@pytest.mark.parametrize("shapes", list(SHAPES))
@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES])
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_norm_and_clip(dev, shapes, dtypes, max_norm):
    grads = _grads(dev, SHAPES[shapes], dtypes, 3)
    before = [g.clone() for g in grads]
    ref, _ = O.clip(before, max_norm)
    assert abs(float(sg.grad_norm(grads)) - ref) <= NORM_TOL * ref
    out = [torch.full_like(g, 7.0) for g in grads]
    norm = sg.clip_grads(grads, max_norm, out=out)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    _check(before, out, norm, max_norm)
    norm2 = sg.clip_grads(grads, max_norm)
    assert torch.equal(norm2, norm)
    _check(before, grads, norm2, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))  # in place or not: the same bits


def test_parameters(dev):
    """clip_grad_norm_ on parameters, some without a gradient, some transposed,
    against torch's own on copies (its fp32 norm: 1e-5)."""
    params = [torch.nn.Parameter(torch.zeros(s, device=dev)) for s in ((40, 30), (7,), (9, 9), (64, 3))]
    other = [torch.nn.Parameter(torch.zeros_like(p)) for p in params]
    g = torch.Generator(device=dev).manual_seed(1)
    for i, (p, q) in enumerate(zip(params, other)):
        if i == 1:
            continue
        x = torch.randn(p.shape[::-1], device=dev, generator=g).t() if i == 0 else torch.randn(p.shape, device=dev, generator=g)
        p.grad, q.grad = x.clone(memory_format=torch.preserve_format), x.clone()
    assert not params[0].grad.is_contiguous()
    norm = sg.clip_grad_norm_(iter(params), 0.5)
    want = torch.nn.utils.clip_grad_norm_(other, 0.5)
    assert abs(float(norm) - float(want)) <= 1e-5 * float(want)
    for p, q in zip(params, other):
        if q.grad is not None:
            assert ((p.grad - q.grad).abs() <= 1e-5 * q.grad.abs()).all()
    single = sg.clip_grad_norm_(params[2], 100.0)
    assert float(single) > 0 and params[1].grad is None


def test_extremes(dev):
    """Squares beyond fp32's range on either side, infinite and NaN gradients,
    a largest norm of zero and of infinity."""
    for v in (1e25, 1e-25, 3e38, 1e-40):
        g = torch.full((1000,), v, device=dev)
        ref = min(float(g[0].double()) * 1000 ** 0.5, float("inf"))
        got = float(sg.grad_norm([g]))
        if ref > torch.finfo(torch.float32).max:
            assert got == float("inf")
        else:
            assert abs(got - ref) <= NORM_TOL * ref + 2.0 ** -150
    for bad in (float("inf"), float("nan")):
        a, b = torch.ones(10, device=dev), torch.ones(5000, device=dev)
        b[77] = bad
        want = torch.nn.Parameter(torch.zeros(5000, device=dev))
        want.grad = b.clone()
        torch.nn.utils.clip_grad_norm_([want], 1.0)
        norm = sg.clip_grads([a, b], 1.0)
        assert torch.equal(norm.isnan(), torch.tensor(bad != bad, device=dev)) and not bool(norm.isfinite())
        assert torch.equal(b.isnan(), want.grad.isnan()) and torch.equal(b.nan_to_num(3.0), want.grad.nan_to_num(3.0))
    g = torch.ones(10, device=dev)
    sg.clip_grads([g], 0.0)
    assert bool((g == 0).all())
    g = torch.ones(10, device=dev)
    assert float(sg.clip_grads([g], float("inf"))) > 3 and bool((g == 1).all())
    z = torch.zeros(10, device=dev)
    assert float(sg.clip_grads([z], 1.0)) == 0.0 and bool((z == 0).all())
    p = torch.nn.Parameter(torch.zeros(4, device=dev))
    p.grad = torch.full((4,), float("nan"), device=dev)
    with pytest.raises(RuntimeError):
        sg.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    p.grad = torch.ones(4, device=dev)
    assert abs(float(sg.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)) - 2.0) < 1e-6


def _at_a_border(n, dtype, seed):
    """n values whose exact norm lies halfway between two fp32 numbers to 2^-56:
    the last bits of the 64-bit sum, and so its order, decide the result."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g).to(dtype)
    x[:40] = 0
    exact = sum((Fraction(v) ** 2 for v in x.tolist()), Fraction(0))
    low = torch.tensor(math.sqrt(exact) * 1.001, dtype=torch.float32)
    half = (Fraction(float(low)) + Fraction(float(torch.nextafter(low, low + 1)))) / 2
    left, i = half ** 2 - exact, 0
    while i < 40 and left > half ** 2 / 2 ** 56:  # each takes most of what is left
        v = torch.tensor(math.sqrt(left) * (1 - 2.0 ** -12), dtype=torch.float64).to(dtype)
        while Fraction(float(v)) ** 2 > left:
            v = torch.nextafter(v, torch.zeros_like(v))
        x[i] = v
        left -= Fraction(float(v)) ** 2
        i += 1
    assert 0 <= left <= half ** 2 / 2 ** 56
    return x[torch.randperm(n, generator=g)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_does_not_depend_on_the_address(dev, dtype):
    """The same values at every offset in 16 bytes: the same sum, bit for bit,
    alone and among others, read only and clipped."""
    size = torch.empty((), dtype=dtype).element_size()
    for n, seed in ((1003, 1), (1003, 2), (20001, 3), (20001, 4), (70000, 5), (70000, 6)):
        x = _at_a_border(n, dtype, seed).to(dev)
        one, two = set(), set()
        for off in range(16 // size + 1):
            store = torch.zeros(n + 32, device=dev, dtype=dtype)
            v = store[off:off + n]
            v.copy_(x)
            assert v.data_ptr() % 16 == off * size % 16
            one.add(float(sg.grad_norm([v])))
            one.add(float(sg.clip_grads([v], 1e9, out=[torch.empty_like(v)])))
            a, b = v[:n // 3], v[n // 3:]
            two.add(float(sg.grad_norm([a, b])))
        assert len(one) == 1 and len(two) == 1, (n, one, two)


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_and_neighbours(dev, dtype):
    """Gradients at every offset of their storage; what lies beside them stays."""
    for off in range(0, 9):
        for n in (1, 5, 8, 40, 70000):
            store = torch.full((n + 32,), 3.0, device=dev, dtype=dtype)
            g = store[off:off + n]
            g.copy_(torch.randn(n, device=dev, generator=torch.Generator(device=dev).manual_seed(n)))
            before = g.clone()
            other = torch.full((n + 32,), 5.0, device=dev, dtype=dtype)
            o = other[3:3 + n]
            norm = sg.clip_grads([g], 0.1, out=[o])
            _check([before], [o], norm, 0.1)
            norm = sg.clip_grads([g], 0.1)
            assert torch.equal(g, o)
            assert bool((store[:off] == 3).all()) and bool((store[off + n:] == 3).all())
            assert bool((other[:3] == 5).all()) and bool((other[3 + n:] == 5).all())


def test_refusals(dev):
    a, b = torch.ones(64, device=dev), torch.ones(64, device=dev)
    store = torch.ones(100, device=dev)
    for grads in ([a, a], [store[:60], store[59:]], [store, store[10:20]]):
        with pytest.raises(ValueError, match="overlap"):
            sg.clip_grads(grads, 1.0)
        assert abs(float(sg.grad_norm(grads)) - O.clip(grads, 1.0)[0]) < 1e-5  # reading twice is fine
    assert bool((a == 1).all()) and bool((store == 1).all())
    for out in ([a], [a.double(), b], [a[:5], b], [b, b], [store[:64], store[1:65]], [b, a], [a.cpu(), b]):
        with pytest.raises(ValueError):
            sg.clip_grads([a, b], 1.0, out=out)
    for grads in ([a.double()], [a.int()], [a[:1].expand(8)], [store[::2]], [a.cpu()], []):
        with pytest.raises(ValueError):
            sg.clip_grads(grads, 1.0)
    for mx in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            sg.clip_grads([a], mx)
    torch.cuda.synchronize()
    assert bool((a == 1).all()) and bool((b == 1).all()) and bool((store == 1).all())


def test_written_tensors_count_a_version(dev):
    """Clipping is an in-place write to autograd too."""
    a, b, o = (torch.ones(8, device=dev) for _ in range(3))
    v = a._version, b._version, o._version
    sg.clip_grads([a, b], 1.0, out=[o, b])
    assert (a._version, b._version, o._version) == (v[0], v[1] + 1, v[2] + 1)
    x = torch.ones(8, device=dev, requires_grad=True)
    y = torch.ones(8, device=dev)
    z = (x * y).sum()  # saves y
    sg.clip_grads([y], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_deterministic_and_partly_in_place(dev):
    grads = _grads(dev, [(700, 900), (33,), (70000,)], DTYPES, 6)
    norms = {float(sg.grad_norm(grads)) for _ in range(5)}
    assert len(norms) == 1
    out = [torch.empty_like(grads[0]), grads[1], torch.empty_like(grads[2])]
    before = [g.clone() for g in grads]
    norm = sg.clip_grads(grads, 0.01, out=out)
    _check(before, out, norm, 0.01)
    assert torch.equal(grads[0], before[0]) and torch.equal(grads[2], before[2])


def test_beyond_the_last_level_cache(dev):
    """More gradients than the caches hold, in place and elsewhere, against torch in 64 bits."""
    grads = _grads(dev, [(9000, 8001), (33,), (6000, 7000)], [torch.float32, torch.bfloat16], 2)
    assert sum(g.numel() * g.element_size() for g in grads) > 300 << 20
    ref = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    before = [g.clone() for g in grads]
    out = [torch.empty_like(g) for g in grads]
    for got in (sg.grad_norm(grads), sg.clip_grads(grads, 0.5, out=out)):
        assert abs(float(got) - float(ref)) <= (2.0 ** -24 * 1.02 + 2e-8) * float(ref)  # 10^8 additions of 2^-53
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    sg.clip_grads(grads, 0.5)
    factor = 0.5 / (ref + 1e-6)
    for a, b, o in zip(grads, before, out):
        step = 5 * 2.0 ** -24 + 2e-8 + (0 if b.dtype == torch.float32 else torch.finfo(b.dtype).eps / 2)
        want = b.double() * factor
        assert torch.equal(a, o) and bool(((a.double() - want).abs() <= step * want.abs() + 1e-40).all())


def test_captured_and_replayed(dev):
    """A captured clip, replayed on new gradients between eager calls."""
    shapes = [(512, 256), (1000,), (64, 64)]
    static = _grads(dev, shapes, DTYPES, 1)
    out = [torch.empty_like(g) for g in static]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sg.clip_grads(static, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = sg.clip_grads(static, 1.0, out=out)
    for rep in range(4):
        new = _grads(dev, shapes, DTYPES, 50 + rep, std=10.0 ** (rep - 3))
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = [torch.empty_like(g) for g in new]
        wn = sg.clip_grads(new, 1.0, out=want)
        torch.cuda.synchronize()
        assert torch.equal(norm, wn) and all(torch.equal(a, b) for a, b in zip(out, want)), rep


def test_parameters_called_as_torch_is(dev):
    """The positions of torch.nn.utils.clip_grad_norm_: the third is the norm's
    type, of which only 2 is offered, the fourth whether a norm that is not finite
    raises, the fifth how torch goes about it."""
    def params(*values):
        out = []
        for v in values:
            out.append(torch.nn.Parameter(torch.zeros(50, device=dev)))
            out[-1].grad = torch.full((50,), v, device=dev)
        return out

    for args in ((1.0,), (1.0, 2.0), (1.0, 2), (1.0, 2.0, False), (1.0, 2.0, True), (1.0, 2.0, False, None),
                 (1.0, 2.0, True, True)):
        ours, torchs = params(3.0, -0.5), params(3.0, -0.5)
        norm, want = sg.clip_grad_norm_(ours, *args), torch.nn.utils.clip_grad_norm_(torchs, *args)
        assert abs(float(norm) - float(want)) <= 1e-6 * float(want)
        assert all(((a.grad - b.grad).abs() <= 1e-6 * b.grad.abs()).all() for a, b in zip(ours, torchs))
    bad = params(3.0, float("nan"))
    assert sg.clip_grad_norm_(bad, 1.0, 2.0).isnan()  # no error: none is asked for
    bad = params(3.0, float("nan"))
    with pytest.raises(RuntimeError, match="not clipped"):
        sg.clip_grad_norm_(bad, 1.0, 2.0, True)
    assert bool((bad[0].grad == 3).all())
    for kind in (1.0, float("inf"), 0.0, 3, "inf"):
        p = params(3.0)
        for call in (lambda: sg.clip_grad_norm_(p, 1.0, kind), lambda: sg.clip_grad_norm_(p, 1.0, norm_type=kind)):
            with pytest.raises(ValueError, match="2-norm"):
                call()
        assert bool((p[0].grad == 3).all())
