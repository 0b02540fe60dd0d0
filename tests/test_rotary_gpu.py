"""Rotary positions and the fused query/key norm (specdec.drafter.rotary,
qk_norm_rotary) against the formulas in float64.

Tolerances, per element, from the roundings on the way (u = 2^-24):
- rotation, fp32: the reduced angle is rounded once (2^-25 half turns =
  9.4e-8 rad), sincospif is within 2 u, the scale and the two products and
  their sum are one u each: below 5e-7 of (|x| + |y|) scale of the pair.
- norm: the sum of squares is a chain of at most 16 and a tree of 5 additions
  of positive terms, half of that relative error in the root, rsqrtf 2 u, two
  products: below 2e-6, so 3e-6 of (|x| + |y|) scale r |w| with the rotation.
- its dx is a difference of two such terms: 6e-6 of the sum of their sizes.
- dw: chains of at most a few hundred products: 2e-5 of the sum of |terms|.
- bf16 results: half a step (2^-8 relative) on top.
"""
import math

import pytest
import torch

from specdec import drafter


def _half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0


def _pairs(x, R, interleaved):
    return (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])


def _join(a, b, rest, interleaved):
    t = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((t, rest), -1)


def _rot64(x, pos, f, interleaved, scale, sign=1.0):
    """(rotated x, size of the terms of each element), fp64."""
    x = x.double()
    R = 2 * f.numel()
    pos = pos if pos.dim() == 2 else pos[None]
    ang = (pos.double()[..., None] * f)[:, :, None]
    c, s = ang.cos() * scale, sign * ang.sin() * scale
    a, b = _pairs(x, R, interleaved)
    size = (a.abs() + b.abs()) * abs(scale)
    return (_join(a * c - b * s, b * c + a * s, x[..., R:], interleaved),
            _join(size, size, x[..., R:].abs(), interleaved))


def _freq(R):
    return drafter.rotary_frequencies(R, device="cuda")[0]


def _randn(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _layout(B, T, H, D, how, dtype, seed):
    """A [B, T, H, D] tensor in one of the layouts a caller may hold."""
    if how == "contiguous":
        return _randn(B, T, H, D, seed=seed, dtype=dtype)
    if how == "fused":  # heads 1..H of a wider projection
        return _randn(B, T, (H + 3) * D, seed=seed, dtype=dtype)[..., D:(H + 1) * D].unflatten(-1, (H, D))
    if how == "heads-first":
        return _randn(B, H, T, D, seed=seed, dtype=dtype).transpose(1, 2)
    if how == "offset":  # not on a 16-byte boundary
        return _randn(B * T * H * D + 1, seed=seed, dtype=dtype)[1:].view(B, T, H, D)
    if how == "elements-strided":
        return _randn(B, T, H, 2 * D, seed=seed, dtype=dtype)[..., ::2]
    raise AssertionError(how)


SHAPES = [  # B, T, H, D, R
    (1, 1, 1, 64, 64), (2, 16, 4, 64, 64), (3, 37, 5, 128, 64), (2, 129, 3, 128, 128), (1, 700, 8, 96, 96),
    (2, 5, 2, 80, 40), (1, 3, 7, 2, 2), (2, 9, 3, 6, 4), (1, 33, 2, 512, 512), (2, 11, 1, 256, 32), (1, 4, 40, 192, 128),
    (4, 1, 33, 128, 126),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,D,R", SHAPES)
def test_rotary_forward_backward(cuda, B, T, H, D, R, dtype, interleaved):
    x = _randn(B, T, H, D, seed=D + T, dtype=dtype).requires_grad_(True)
    dy = _randn(B, T, H, D, seed=D + T + 1, dtype=dtype)
    pos = 1000 * torch.arange(B, device="cuda")[:, None] + torch.arange(T, device="cuda")[None] - 2
    f = _freq(R)
    y = drafter.rotary(x, pos, f, interleaved=interleaved, scale=1.25)
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    y.backward(dy)
    for got, src, sign in ((y, x, 1.0), (x.grad, dy, -1.0)):
        want, size = _rot64(src.detach(), pos, f, interleaved, 1.25, sign)
        err = (got.detach().double() - want).abs()
        assert bool((err <= 5e-7 * size + _half(dtype) * want.abs()).all()), float(err.max())
        assert torch.equal(got.detach()[..., R:], src.detach()[..., R:])  # the rest is copied


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["contiguous", "fused", "heads-first", "offset", "elements-strided"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_layouts_and_positions(cuda, how, dtype):
    B, T, H, D = 2, 50, 3, 128
    x = _layout(B, T, H, D, how, dtype, 5)
    f = _freq(D)
    far = torch.arange(T, device="cuda") * 999983 + 12345678  # past a million: angles need fp64
    both = torch.stack((far, far.flip(0)))
    for pos in (far, far.int(), both, both.t().contiguous().t(), far.expand(B, T), both[:, ::1]):
        want, size = _rot64(x, pos, f, False, 1.0)
        got = drafter.rotary(x, pos, f)
        assert bool(((got.double() - want).abs() <= 5e-7 * size + _half(dtype) * want.abs()).all())
    # the input is as it was; no tokens, no sequences
    assert torch.equal(x, _layout(B, T, H, D, how, dtype, 5))
    assert drafter.rotary(x[:, :0], far[:0], f).shape == (B, 0, H, D)
    assert drafter.rotary(x[:0], far, f).shape == (0, T, H, D)


@pytest.mark.gpu
def test_rotary_leaves_nan_and_infinity_in_their_pairs(cuda):
    x = _randn(1, 4, 2, 64, seed=1)
    clean = drafter.rotary(x, torch.arange(4, device="cuda"), _freq(64))
    x[0, 2, 1, 5] = math.nan
    x[0, 3, 0, 40] = math.inf
    got = drafter.rotary(x, torch.arange(4, device="cuda"), _freq(64))
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 2, 1, [5, 37]] = True
    hit[0, 3, 0, [8, 40]] = True
    assert torch.equal(got[~hit], clean[~hit]) and not bool(torch.isfinite(got[hit]).any())


def _norm64(x, w, dy, pos, f, eps, interleaved, scale):
    """Outputs, gradients and the sizes of their terms, fp64."""
    x, w, dy = x.double(), w.double(), dy.double()
    D = x.shape[-1]
    r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    y, ysize = _rot64(x * r * w, pos, f, interleaved, scale)
    dn, dnsize = _rot64(dy, pos, f, interleaved, scale, -1.0)
    g = dn * w
    dx = r * g - x * r ** 3 * (g * x).sum(-1, keepdim=True) / D
    dxsize = r * dnsize * w.abs() + x.abs() * r ** 3 * (dnsize * w.abs() * x.abs()).sum(-1, keepdim=True) / D
    t = dn * x * r
    tsize = dnsize * x.abs() * r
    return y, ysize, dx, dxsize, t.sum((0, 1, 2)), tsize.sum((0, 1, 2))


NORM_SHAPES = [  # B, T, Hq, Hk, D, R
    (1, 1, 1, 1, 64, 64), (2, 33, 4, 4, 64, 64), (3, 70, 6, 2, 128, 128), (1, 257, 32, 8, 128, 64), (2, 9, 3, 1, 96, 96),
    (2, 5, 5, 3, 80, 40), (1, 7, 2, 1, 512, 256), (1, 65, 1, 7, 256, 256), (1, 3, 2, 2, 6, 2), (40, 1, 8, 2, 128, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hq,Hk,D,R", NORM_SHAPES)
def test_qk_norm_rotary_forward_backward(cuda, B, T, Hq, Hk, D, R, dtype, interleaved):
    s = 31 * D + T
    q, k = _layout(B, T, Hq, D, "fused", dtype, s), _layout(B, T, Hk, D, "fused", dtype, s + 1)
    wq, wk = 1 + 0.3 * _randn(D, seed=s + 2), 1 + 0.3 * _randn(D, seed=s + 3)
    dq, dk = _randn(B, T, Hq, D, seed=s + 4, dtype=dtype), _layout(B, T, Hk, D, "heads-first", dtype, s + 5)
    for t in (q, k, wq, wk):
        t.requires_grad_(True)
    pos = torch.arange(T, device="cuda") + 4000
    f = _freq(R)
    yq, yk = drafter.qk_norm_rotary(q, k, wq, wk, pos, f, eps=1e-6, interleaved=interleaved, scale=0.9)
    grads = torch.autograd.grad((yq, yk), (q, k, wq, wk), (dq, dk))
    half = _half(dtype)
    for y, x, w, dy, dx, dw in ((yq, q, wq, dq, grads[0], grads[2]), (yk, k, wk, dk, grads[1], grads[3])):
        want, size, wdx, sdx, wdw, sdw = _norm64(x.detach(), w.detach(), dy, pos, f, 1e-6, interleaved, 0.9)
        assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == torch.float32 and dx.shape == x.shape
        assert bool(((y.detach().double() - want).abs() <= 3e-6 * size + half * want.abs()).all())
        assert bool(((dx.double() - wdx).abs() <= 6e-6 * sdx + half * wdx.abs()).all())
        assert bool(((dw.double() - wdw).abs() <= 2e-5 * sdw).all())
    yq, yk = drafter.qk_norm_rotary(q, k, wq, wk, pos, f, eps=1e-6, interleaved=interleaved, scale=0.9)
    again = torch.autograd.grad((yq, yk), (q, k, wq, wk), (dq, dk))
    for a, b in zip(grads, again):  # fixed summation order
        assert torch.equal(a, b)
    with torch.no_grad():  # the path without autograd gives the same bits
        zq, zk = drafter.qk_norm_rotary(q, k, wq, wk, pos, f, eps=1e-6, interleaved=interleaved, scale=0.9)
    assert torch.equal(zq, yq) and torch.equal(zk, yk)


@pytest.mark.gpu
def test_qk_norm_rotary_gradient_against_differences(cuda):
    """d/de of sum(out * dout) along a random direction, by central differences
    of the fp32 kernel: rounding 3e-7 / 1e-2 of the sizes, curvature (1e-2)^2."""
    B, T, Hq, Hk, D = 2, 20, 3, 1, 64
    q, k = _randn(B, T, Hq, D, seed=1), _randn(B, T, Hk, D, seed=2)
    wq, wk = 1 + 0.2 * _randn(D, seed=3), 1 + 0.2 * _randn(D, seed=4)
    dq, dk = _randn(B, T, Hq, D, seed=5), _randn(B, T, Hk, D, seed=6)
    pos, f = torch.arange(T, device="cuda"), _freq(D)
    x = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    out = drafter.qk_norm_rotary(*x, pos, f, eps=1e-6)
    grads = torch.autograd.grad(out, x, (dq, dk))
    for i, t in enumerate(x):
        v = _randn(*t.shape, seed=10 + i)
        def loss(e):
            moved = [a.detach() + e * v if a is t else a.detach() for a in x]
            yq, yk = drafter.qk_norm_rotary(*moved, pos, f, eps=1e-6)
            return float((yq.double() * dq).sum() + (yk.double() * dk).sum())
        got = float((grads[i].double() * v).sum())
        want = (loss(1e-2) - loss(-1e-2)) / 2e-2
        size = float(grads[i].double().norm() * v.double().norm())
        assert abs(got - want) <= 2e-3 * size, (i, got, want)


@pytest.mark.gpu
def test_qk_norm_rotary_weights_of_bf16_and_one_sided_gradients(cuda):
    q, k = _randn(2, 8, 4, 64, seed=1, dtype=torch.bfloat16), _randn(2, 8, 2, 64, seed=2, dtype=torch.bfloat16)
    wq = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    wk = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q.requires_grad_(True)
    pos, f = torch.arange(8, device="cuda"), _freq(64)
    yq, _ = drafter.qk_norm_rotary(q, k, wq, wk, pos, f)
    yq.float().sum().backward()  # an expanded gradient for q, none for k
    assert q.grad.dtype == torch.bfloat16 and wq.grad.dtype == torch.bfloat16
    assert bool((wk.grad == 0).all()) and bool(torch.isfinite(q.grad.float()).all())
    # an all-zero head normalises to zero and its gradient stays finite
    z = torch.zeros(1, 1, 1, 64, device="cuda", requires_grad=True)
    yz, _ = drafter.qk_norm_rotary(z, z.detach(), wq.float(), wk.float(), pos[:1], f, eps=1e-6)
    yz.sum().backward()
    assert bool((yz == 0).all()) and bool(torch.isfinite(z.grad).all())


def test_rotary_frequencies():
    f, s = drafter.rotary_frequencies(64, 10000.0)
    i = torch.arange(32, dtype=torch.float64)
    assert f.dtype == torch.float64 and s == 1.0
    assert torch.allclose(f, torch.exp(-math.log(10000.0) * 2 * i / 64), rtol=1e-14)
    lin, _ = drafter.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.allclose(lin, f / 4, rtol=1e-15)
    ntk, _ = drafter.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert abs(float(ntk[0]) - 1.0) < 1e-15 and abs(float(ntk[-1] / f[-1]) - 0.25) < 1e-12
    for kind, low, high in (("ramp", 1.0, 4.0), ("yarn", 1.0, 32.0)):
        g, s = drafter.rotary_frequencies(128, scaling=kind, factor=8.0, original_length=8192)
        f = drafter.rotary_frequencies(128)[0]
        turns = 8192 * f / (2 * math.pi)
        assert torch.equal(g[turns >= high], f[turns >= high])
        assert torch.allclose(g[turns <= low], f[turns <= low] / 8, rtol=1e-15)
        mid = (turns > low) & (turns < high)
        assert bool(mid.any()) and bool(((g < f) & (g > f / 8))[mid].all()) and bool((g[1:] < g[:-1]).all())
        assert s == (0.1 * math.log(8.0) + 1.0 if kind == "yarn" else 1.0)
    for bad in (dict(dim=63), dict(dim=0), dict(dim=64, base=0.0), dict(dim=64, factor=-1.0), dict(dim=64, scaling="x"),
                dict(dim=64, scaling="yarn", factor=2.0), dict(dim=2, scaling="ntk", factor=2.0),
                dict(dim=64, scaling="ramp", original_length=8, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            drafter.rotary_frequencies(**bad)


def test_rotary_refuses_cpu_tensors():
    x, f = torch.zeros(1, 2, 1, 64), torch.ones(32, dtype=torch.float64)
    with pytest.raises(AssertionError):
        drafter.rotary(x, torch.arange(2), f)
    with pytest.raises(AssertionError):
        drafter.qk_norm_rotary(x, x, torch.ones(64), torch.ones(64), torch.arange(2), f)


def test_rotary_c_argument_checks():
    import ctypes

    from specdec import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced: the checks fail first

    def rot(B=1, T=4, H=2, D=64, R=64, scale=1.0, dtype=0):
        return lib.specdec_rotary(p, None, p, p, 0, p, B, T, H, D, R, 0, scale, 0, dtype, None)

    for bad in (dict(B=-1), dict(T=-1), dict(H=0), dict(D=63), dict(D=0), dict(D=514), dict(R=66), dict(R=0), dict(R=31),
                dict(dtype=7), dict(B=65536, T=65536)):
        assert rot(**bad) == _lib.ERR_ARGUMENT, bad
    assert rot(scale=float("nan")) == _lib.ERR_VALUE
    assert rot(B=0) == _lib.OK and rot(T=0) == _lib.OK

    def norm(Hk=1, eps=1e-6, fn="forward"):
        if fn == "forward":
            return lib.specdec_qk_norm_rotary_forward(p, None, p, None, p, p, p, p, p, 0, p, 1, 4, 2, Hk, 64, 64, 0, 1.0,
                                                      eps, 0, None)
        return lib.specdec_qk_norm_rotary_backward(p, None, p, None, p, p, p, None, p, None, p, p, p, p, p, 0, p, 1, 4, 2,
                                                   Hk, 64, 64, 0, 1.0, eps, 0, p, 1 << 20, None)

    for fn in ("forward", "backward"):
        assert norm(Hk=0, fn=fn) == _lib.ERR_ARGUMENT
        assert norm(eps=-1.0, fn=fn) == _lib.ERR_VALUE
        assert norm(eps=float("nan"), fn=fn) == _lib.ERR_VALUE


@pytest.mark.gpu
def test_rotary_refusals(cuda):
    x, f = torch.zeros(2, 4, 2, 64, device="cuda"), _freq(64)
    w, pos = torch.ones(64, device="cuda"), torch.arange(4, device="cuda")
    for args in ((x[0], pos, f), (x.half(), pos, f), (x, pos.float(), f), (x, pos[:3], f), (x, pos.cpu(), f),
                 (x, pos, f.float()), (x, pos, f.cpu()), (x, pos, _freq(66)), (x, pos, f[:0]), (x, pos[:, None], f)):
        with pytest.raises(AssertionError):
            drafter.rotary(*args)
    with pytest.raises(AssertionError):
        drafter.qk_norm_rotary(x, x.bfloat16(), w, w, pos, f)
    with pytest.raises(AssertionError):
        drafter.qk_norm_rotary(x, x[:, :3], w, w, pos, f)
    with pytest.raises(AssertionError):
        drafter.qk_norm_rotary(x, x, w[:32], w, pos, f)
    with pytest.raises(ValueError):
        drafter.qk_norm_rotary(x, x, w, w, pos, f, eps=-1.0)
    y = drafter.rotary(x.requires_grad_(True), pos, f)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        g.sum().backward()


@pytest.mark.gpu
def test_rotary_past_32_bit_offsets(cuda):
    """2.2e9 elements: the last tokens lie past 2^31."""
    T, H, D = 262_200, 64, 128
    x = torch.zeros(1, T, H, D, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    x[0, -9:] = _randn(9, H, D, seed=3, dtype=torch.bfloat16)
    pos = torch.arange(T, device="cuda")
    y = drafter.rotary(x, pos, _freq(D))
    want, size = _rot64(x[:, -9:], pos[-9:], _freq(D), False, 1.0)
    assert bool(((y[:, -9:].double() - want).abs() <= 5e-7 * size + _half(x.dtype) * want.abs()).all())
    assert not bool(y[:, :-9].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_default_eps_is_torchs(cuda, dtype):
    """Small inputs, where eps counts: 2^-7 (bf16's own) would halve the constant
    0.05. Against the formula as above (3e-6, and half a step), and against
    torch's own with weights rounded to the type: three roundings at most."""
    D = 64
    pos = torch.zeros(3, device="cuda", dtype=torch.int64)  # no rotation: cos 1, sin 0
    f, _ = drafter.rotary_frequencies(D, device="cuda")
    w = torch.linspace(0.5, 2.0, D, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    for size in (0.05, 3e-4):
        x = (size * torch.randn(2, 3, 4, D, device="cuda", generator=g)).to(dtype)
        y, z = drafter.qk_norm_rotary(x, x[:, :, :2], w, w, pos, f)
        want = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 2.0 ** -23) * w.double()
        assert bool(((y.double() - want).abs() <= (3e-6 + _half(dtype)) * want.abs()).all())
        assert torch.equal(z, y[:, :, :2])
        torchs = torch.nn.functional.rms_norm(x, (D,), w.to(dtype), None).double()
        assert float((y.double() - torchs).norm() / torchs.norm()) <= 3 * _half(dtype) + 1e-5
