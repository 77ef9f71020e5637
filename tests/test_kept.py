"""Activations kept in 8 bits: codes and values from their definition, the activation function, linear layers and the feed-forward block that keep
their inputs so."""
import math

import pytest
import torch

from nmtgminor_b200 import ops
from nmtgminor_b200.ops import kept, reference as ref

DEV = "cuda"
HALF = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11, torch.float32: 2 ** -24}


def _matrix(rows, width, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + rows * 7 + width)
    x = torch.randn(rows, width, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    if rows > 2 and width > 2:
        x[0] = 0.0
        x[1, ::3] = 0.0
        x[2, 1] = 448.0 * 2 ** -3
        x[2, 0] = 1e4
    if dtype == torch.float16:
        x = x.clamp(-6e4, 6e4)
    return x.to(dtype)


def _defined(x):
    """Codes' values from the definition, in 64 bits."""
    rows, width = x.shape
    out = torch.zeros(rows, width, dtype=torch.float64)
    xd = x.double()
    for b in range(0, width, 32):
        part = xd[:, b:b + 32]
        most = part.abs().amax(1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(most / 448.0)).clamp(min=-127))
        v = part / unit
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, b:b + 32] = torch.round(v / step) * step * unit
    return out


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 31), (4, 32), (7, 33), (9, 200)])
def test_values_by_definition_on_the_cpu(dtype, rows, width):
    x = _matrix(rows, width, dtype)
    k = kept.quantise(x)
    v = kept.restore(k, torch.float32).double()
    assert k.shape == (rows, width) and k.nbytes() == rows * (-(-width // 32)) * 33
    assert torch.equal(v, _defined(x))
    unit = torch.exp2(k.scales.double() - 127).repeat_interleave(32, 1)[:, :width]
    assert ((v - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * unit)).all()


def test_extremes_on_the_cpu():
    x = torch.tensor([[math.inf, 1.0, -3.0, math.nan, 0.0, -math.inf], [65504.0, -65504.0, 1e-7, 0.0, 6e-8, 1.0]]).half()
    v = kept.restore(kept.quantise(x))
    assert torch.isnan(v[0, [0, 3, 5]]).all() and v[0, 1] == 1.0 and v[0, 2] == -3.0
    assert v[1, 0] == 65504.0 and v[1, 1] == -65504.0                # 65536 would be the nearest: brought into the type
    low = torch.full((1, 40), torch.finfo(torch.bfloat16).min).bfloat16()
    assert torch.equal(kept.restore(kept.quantise(low)), low)
    tiny = torch.full((1, 3), 2.0 ** -130, dtype=torch.float32)
    assert torch.equal(kept.restore(kept.quantise(tiny)), tiny)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_activation_on_the_cpu(act):
    z = _matrix(6, 70, torch.float32, spread=0.3).requires_grad_(True)
    y = kept.activation(z, act)
    fn = {"none": lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[act]
    assert torch.equal(y, fn(z))
    dy = torch.randn(6, 70, generator=torch.Generator().manual_seed(1))
    h = kept.restore(kept.quantise(z)).requires_grad_(True)
    want = torch.autograd.grad(fn(h), h, dy)[0]
    assert torch.allclose(torch.autograd.grad(y, z, dy)[0], want, atol=1e-7, rtol=1e-6)


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_linear_and_mlp_on_the_cpu(act):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(10, 40, generator=g).requires_grad_(True)
    w = (torch.randn(24, 40, generator=g) * 0.2).requires_grad_(True)
    b = torch.randn(24, generator=g).requires_grad_(True)
    dy = torch.randn(10, 24, generator=g)
    y, plain = ops.linear(x, w, b, act, keep8=True), ops.linear(x, w, b, act)
    assert torch.equal(y, plain)
    z = torch.nn.functional.linear(x, w, b)
    slope = dy if act == "none" else torch.autograd.grad(ref._act(h := kept.straight_through(z.detach()).requires_grad_(True), ops.ACT_IDS[act]), h, dy)[0]
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.allclose(gw, slope.t() @ kept.restore(kept.quantise(x)), atol=1e-5, rtol=1e-5)
    assert torch.allclose(gx, slope @ w, atol=1e-5, rtol=1e-5) and torch.allclose(gb, slope.sum(0), atol=1e-5, rtol=1e-5)
    if act == "none":
        return
    w2 = (torch.randn(40, 24, generator=g) * 0.2).requires_grad_(True)
    out, plain = ops.mlp(x, w, b, w2, None, act, keep8=True), ops.mlp(x, w, b, w2, None, act)
    assert torch.equal(out, plain)
    d2 = torch.randn(10, 40, generator=g)
    gx, gw, gw2 = torch.autograd.grad(out, (x, w, w2), d2)
    hidden = torch.relu(z) if act == "relu" else z
    held = kept.restore(kept.quantise(hidden.detach()))
    assert torch.allclose(gw2, d2.t() @ ref._act(held, ops.ACT_IDS[act]), atol=1e-5, rtol=1e-5)
    at = z.detach() if act == "relu" else held                        # ReLU keeps its signs
    at.requires_grad_(True)
    dz = torch.autograd.grad(ref._act(at, ops.ACT_IDS[act]), at, d2 @ w2)[0]
    assert torch.allclose(gw, dz.t() @ kept.restore(kept.quantise(x)), atol=1e-5, rtol=1e-5)
    assert torch.allclose(gx, dz @ w, atol=1e-5, rtol=1e-5)


def _refusals(device):
    x = torch.zeros(4, 8, device=device)
    for f in (lambda: kept.quantise(x[0]), lambda: kept.quantise(x.double()), lambda: kept.quantise(x.long()),
              lambda: kept.activation(x, "tanh"), lambda: kept.activation(x, dropout_p=1.0), lambda: kept.activation(x[None]),
              lambda: kept.restore(kept.quantise(x), torch.float64),
              lambda: ops.linear(x, torch.zeros(6, 8, device=device), act="gelu", dropout_p=0.1, keep8=True)):
        with pytest.raises((ValueError, TypeError)):
            f()


def test_refusals_on_the_cpu():
    _refusals("cpu")


# ---------------------------------------------------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (3, 7), (5, 31), (4, 32), (1, 4096), (7, 33), (300, 40), (9, 200), (64, 1000), (1000, 1024), (2, 70001), (70000, 8)]


def _laid_out(x, layout):
    """dense, rows of a wider matrix, or off every alignment but the element's"""
    if layout == "dense":
        return x.to(DEV)
    pad, skip = (8, 0) if layout == "wide" else (3, 1)
    flat = torch.full((x.shape[0] * (x.shape[1] + pad) + skip,), 9.0, dtype=x.dtype, device=DEV)
    v = flat[skip:].view(x.shape[0], -1)[:, :x.shape[1]]
    v.copy_(x)
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("layout", ["dense", "wide", "odd"])
def test_codes_are_those_of_the_restatement(dtype, layout):
    for rows, width in SHAPES:
        x = _matrix(rows, width, dtype)
        want = kept.quantise_reference(x)
        got = kept.quantise(_laid_out(x, layout))
        assert torch.equal(got.scales.cpu(), want.scales)
        assert torch.equal(got.codes.cpu()[:, :width], want.codes[:, :width])
        for out in HALF:
            if out != torch.float16 or dtype == torch.float16:
                assert torch.equal(kept.restore(got, out).cpu(), kept.restore_reference(want, out))


@pytest.mark.gpu
def test_extremes_on_the_gpu():
    for dtype in HALF:
        most, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        rows = [[math.inf, 1.0, -3.0, math.nan, 0.0, -math.inf], [most, -most, small, 0.0, -small / 2, 1.0], [small, small / 2, 0, 0, 0, -small],
                [-most] * 6, [448, 449, 447, 464, 480, 1], [0.0, -0.0, 0.0, 0.0, 0.0, 0.0]]
        x = torch.tensor(rows).to(dtype)
        want, got = kept.quantise_reference(x), kept.quantise(x.to(DEV))
        assert torch.equal(got.codes.cpu()[:, :6] & 127, want.codes[:, :6] & 127) and torch.equal(got.scales.cpu(), want.scales)
        assert torch.equal(kept.restore(got).cpu().nan_to_num(7.0), kept.restore_reference(want).nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_activation_and_its_slope(dtype, act):
    """16-bit types: the function is off by 2^-18 of its terms (the fit of the tail 1.1e-6, exp2 and the division 2^-22), then rounded once; fp32: by
    a few roundings of the terms.  In the tail the exponent's own roundings count: -log2(e) z^2 / 2 with three of 2^-24 makes
    3 ln 2 log2(e) / 2 z^2 2^-24 = 1.5 z^2 2^-24 of the tail, and erfcf's argument, rounded twice, 2 z^2 2^-24; beyond z^2 = 200 the tail
    is below every normal number.  The slope's terms are area, at most 1, and z times the bell, at most 0.25."""
    fn = {"none": lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[act]
    part = 2 ** -18 if dtype != torch.float32 else 2 ** -20
    for rows, width in SHAPES:
        for layout in ("dense", "odd"):
            x = _matrix(rows, width, dtype, spread=1.0)
            z = _laid_out(x, layout).requires_grad_(True)
            y = kept.activation(z, act)
            want = fn(z.detach().double())
            if act == "gelu":       # by erfc: 1 + erf leaves 2^-53 of 1 in the tail, at z = -8 an eighth of a percent
                want = 0.5 * z.detach().double() * torch.erfc(z.detach().double() * -math.sqrt(0.5))
            # below 2^-14 a 16-bit float's step is 2^-24; the tail of GELU falls to where exp2 is a denormal
            low = 2 ** -25 if dtype == torch.float16 else 2 ** -126
            if act == "silu":       # a gate below 2^-126 (z < -87.3) counts as 0: |z| gate is then below 89 * 2^-126
                low = max(low, 2 ** -119)
            tail = 2 ** -22 * z.detach().double().square().clamp(max=200.0)
            assert ((y.detach().double() - want).abs() <= (HALF[dtype] + part + tail) * want.abs() + low).all()
            dy = torch.randn(rows, width, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
            got = torch.autograd.grad(y, z, dy)[0]
            held = kept.restore_reference(kept.quantise_reference(x), torch.float32).to(DEV).double().requires_grad_(True)
            slope = torch.autograd.grad(fn(held).sum(), held)[0]
            terms = torch.ones_like(slope) if act != "relu" else slope
            assert ((got.double() - dy.double() * slope).abs() <= dy.double().abs() * (HALF[dtype] * slope.abs() + part * terms) + low).all()
            with torch.no_grad():
                assert torch.equal(kept.activation(z, act), y)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [256, 30, 33])
def test_dropout_mask_is_that_of_dropout_add(width):
    ops.manual_seed(77)
    z = torch.randn(200, width, device=DEV).bfloat16().requires_grad_(True)
    y = kept.activation(z, "none", 0.3)
    dy = torch.ones_like(y)
    dz = torch.autograd.grad(y, z, dy)[0]
    scale = 256.0 / (256 - int(0.3 * 256 + 0.5))
    kept_rows = dz != 0
    assert torch.allclose(dz[kept_rows].float(), torch.full((), scale, device=DEV).bfloat16().float())
    assert torch.equal(y != 0, kept_rows & (z != 0)) and 0.6 < kept_rows.float().mean().item() < 0.8
    if z.numel() % 16 == 0:
        ops.manual_seed(77)
        same = ops.dropout_add(z.detach(), None, 0.3)
        assert torch.equal(same, y.detach())


class _Store:
    """what the flat store attaches to a parameter"""

    @staticmethod
    def param(shape, scale, seed):
        g = torch.Generator().manual_seed(seed)
        work = (torch.randn(*shape, generator=g) * scale).bfloat16().to(DEV)
        p = torch.nn.Parameter(work.float())
        p.work, p.main_grad = work, torch.zeros(shape, device=DEV)
        return p


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N,act", [(1, 64, 8, "none"), (7, 136, 40, "none"), (200, 512, 1000, "none"), (1000, 1024, 512, "gelu"),
                                          (129, 256, 264, "relu"), (33, 72, 100, "silu")])
def test_linear_keeps_its_input(rows, K, N, act):
    w, b = _Store.param((N, K), K ** -0.5, 1), _Store.param((N,), 0.3, 2)
    x = _matrix(rows, K, torch.bfloat16, spread=0.3).to(DEV).requires_grad_(True)
    y = ops.linear(x, w, b, act, keep8=True)
    assert torch.equal(y, ops.linear(x, w, b, act))
    dy = torch.randn(rows, N, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    dx = torch.autograd.grad(y, x, dy)[0]
    held = kept.restore(kept.quantise(x)).double()
    dz = dy.double()
    if act != "none":       # the slope from the kept pre-activation, whose codes come from its bf16 values; one more rounding
        z = torch.empty(rows, N, dtype=torch.bfloat16, device=DEV)
        ops.gemm(x.detach(), w.work, ops.empty_rows(rows, N, DEV), bias=b.work, preact=(zz := ops.empty_rows(rows, N, DEV)), act=ops.ACT_IDS[act])
        z.copy_(zz)
        dz = ops.ext().kept_backward(dy, *(lambda k: (k.codes, k.scales))(kept.quantise(z)), ops.ACT_IDS[act], 0.0, 0, 0).double()
    want_w, size_w = dz.t() @ held, dz.abs().t() @ held.abs()
    want_x = dz @ w.work.double()
    # sums in 32 bits of exact products: 2^-24 of their terms, per term at most
    assert ((w.main_grad.double() - want_w).abs() <= 2 ** -24 * (rows + 32) * size_w).all()
    assert ((b.main_grad.double() - dz.sum(0)).abs() <= 2 ** -24 * (rows + 32) * dz.abs().sum(0)).all()
    assert ((dx.double() - want_x).abs() <= 2 ** -8 * want_x.abs() + 2 ** -24 * (N + 32) * (dz.abs() @ w.work.double().abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_mlp_keeps_its_activations(act, p):
    rows, K, Fd = 300, 256, 1024
    params = lambda: (_Store.param((Fd, K), K ** -0.5, 1), _Store.param((Fd,), 0.3, 2), _Store.param((K, Fd), Fd ** -0.5, 3), _Store.param((K,), 0.1, 4))
    x = torch.randn(rows, K, generator=torch.Generator().manual_seed(9)).bfloat16().to(DEV).requires_grad_(True)
    dy = torch.randn(rows, K, generator=torch.Generator().manual_seed(8)).bfloat16().to(DEV)
    outs = []
    for keep in (False, True):
        ops.manual_seed(5)
        w1, b1, w2, b2 = params()
        y = ops.mlp(x, w1, b1, w2, b2, act, p, p, residual=x, keep8=keep)
        outs.append((y.detach(), torch.autograd.grad(y, x, dy)[0], w1.main_grad, b1.main_grad, w2.main_grad, b2.main_grad))
    base, held = outs
    assert torch.equal(base[0], held[0])
    # the same column sums, whose blocks meet in 32-bit atomic additions in any order: two orders differ by 2^-24 of the terms a row, each
    masked = dy.abs().double().sum(0) / (1 - p if p else 1.0) * 1.01
    assert ((base[5] - held[5]).abs().double() <= 2 * rows * 2 ** -24 * masked).all()
    if act == "relu":       # signs are kept: only the weights' gradients see the 8 bits
        assert torch.equal(base[1], held[1]) and torch.allclose(base[3], held[3], atol=1e-4, rtol=1e-4)
    # rounding to 3 mantissa bits: each of the summed products is off by at most 2^-4 of itself, with signs as good as random 2^-4 / sqrt 3 of the
    # norm; the slope moves with z by at most its curvature (below 0.8 for GELU, 0.5 for SiLU) times 2^-4 |z|
    for a, b in zip(base[1:], held[1:]):
        assert (a.double() - b.double()).norm() <= 2 ** -4 * a.double().norm()
    assert not torch.equal(base[4], held[4])


@pytest.mark.gpu
def test_what_waits_takes_half_the_memory():
    K, Fd, rows = 512, 2048, 4096
    x = torch.randn(rows, K, device=DEV).bfloat16().requires_grad_(True)
    w1, w2 = _Store.param((Fd, K), 0.04, 1), _Store.param((K, Fd), 0.02, 2)
    size = {}
    for keep in (False, True):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = ops.mlp(x, w1, None, w2, None, "gelu", keep8=keep)
        size[keep] = torch.cuda.memory_allocated() - before - y.numel() * 2
        y.backward(torch.ones_like(y))
        del y
    assert size[True] <= 33 * rows * (K + Fd) // 32 + (1 << 14) and size[True] < 0.3 * size[False] + rows * K * 2


@pytest.mark.gpu
def test_streams_graphs_and_empty_matrices():
    z = [torch.randn(500, 333, device=DEV).bfloat16().requires_grad_(True) for _ in range(2)]
    dy = torch.randn(500, 333, device=DEV).bfloat16()
    step = lambda t: (lambda y: (y.detach(), torch.autograd.grad(y, t, dy)[0]))(kept.activation(t, "gelu"))
    want = [step(t) for t in z]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for t in z:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(t))
        graphs.append(g)
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, o in zip(want, outs) for a, b in zip(w, o))
    for shape in ((0, 32), (5, 0)):
        e = torch.zeros(shape, device=DEV).requires_grad_(True)
        y = kept.activation(e, "silu")
        assert y.shape == shape and torch.autograd.grad(y.sum(), e)[0].shape == shape
        assert kept.restore(kept.quantise(e)).shape == shape


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    _refusals(DEV)
    x = torch.zeros(4, 64, device=DEV)
    k = kept.quantise(x)
    for f in (lambda: ops.ext().kept_backward(x, k.codes[:2], k.scales, 0, 0.0, 0, 0), lambda: ops.ext().kept_backward(x, k.codes, k.scales, 9, 0.0, 0, 0),
              lambda: ops.ext().kept_quantise(x[:1].expand(4, 64)), lambda: ops.ext().kept_backward(x, k.codes.cpu(), k.scales, 0, 0.0, 0, 0)):
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_infinities_and_nan_reach_the_gradient(dtype, act):
    """One infinity and one NaN among ordinary elements, in layouts of every path: their own gradients are NaN, and no others."""
    for rows, width in ((64, 512), (5, 40), (3, 33)):
        x = _matrix(rows, width, dtype, spread=1.0).clamp(-3, 3).to(DEV)
        x[1, 7], x[2, 30] = math.inf, math.nan
        z = x.requires_grad_(True)
        grad = torch.autograd.grad(kept.activation(z, act), z, torch.ones_like(z))[0]
        bad = torch.zeros(rows, width, dtype=torch.bool, device=DEV)
        if act != "none":                    # without a function the gradient does not look at the element
            bad[1, 7] = bad[2, 30] = True
        assert torch.equal(torch.isnan(grad), bad)
        back = kept.restore(kept.quantise(x.detach()))
        bad[1, 7] = bad[2, 30] = True
        assert torch.equal(torch.isnan(back), bad)


@pytest.mark.gpu
def test_no_second_derivative():
    z = torch.randn(4, 64, device=DEV, requires_grad=True)
    y = kept.activation(z, "gelu")
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), z, create_graph=True)


@pytest.mark.gpu
def test_more_than_2_31_elements():
    """Offsets beyond 32 bits: the last rows of 2.2e9 elements against the same rows by themselves."""
    for rows, width in ((540000, 4096), (540000, 4100)):
        x = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(3))
        few = x[-5:].clone().requires_grad_(True)
        z = x.requires_grad_(True)
        y = kept.activation(z, "gelu")
        want = kept.activation(few, "gelu")
        assert torch.equal(y.detach()[-5:], want.detach())
        dy = torch.ones_like(y)
        del x
        assert torch.equal(torch.autograd.grad(y, z, dy)[0][-5:], torch.autograd.grad(want, few, dy[-5:])[0])
        del dy, y
        assert torch.equal(kept.restore(kept.quantise(z.detach()))[-5:], kept.restore(kept.quantise(few.detach())))
        del z


@pytest.mark.gpu
def test_what_waits_is_freed_with_the_pass():
    """The codes are saved tensors: the backward pass frees them while the result lives, a second one is refused, and a kept graph serves two."""
    rows, K, N = 2048, 512, 1024
    x = torch.randn(rows, K, device=DEV).bfloat16().requires_grad_(True)
    w1, w2 = _Store.param((N, K), 0.04, 1), _Store.param((K, N), 0.02, 2)
    for f in (lambda: ops.linear(x, w1, None, "gelu", keep8=True), lambda: ops.mlp(x, w1, None, w2, None, "relu", keep8=True),
              lambda: ops.mlp(x, w1, None, w2, None, "gelu", keep8=True), lambda: kept.activation(x, "silu")):
        y = f()
        ones = torch.ones_like(y)
        first = torch.autograd.grad(y, x, ones, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(y, x, ones, retain_graph=True)[0], first)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y.backward(ones)
        x.grad = None
        assert torch.cuda.memory_allocated() <= before - 33 * rows * K // 32
        with pytest.raises(RuntimeError):
            y.backward(ones)
