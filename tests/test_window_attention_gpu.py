"""Sliding-window attention with sinks (specdec.drafter.window_attention and
window_attention_cached) against the definition in float64, from the same bf16
inputs.

Tolerances, per element (h = 2^-8, half a step of bf16):
- o: each weight is rounded once (h), the sums are fp32, the result is rounded
  once (h): |error| <= h sum_j P_j |v_j| + h |o| + 1e-5.
- dv = P^T do: likewise with sum P |do|.
- dS = P (dP - delta) scale: P itself is exact to fp32 here, dP to fp32; delta
  uses the forward's sums (o and the residual of its rounding), which are
  h sum P |v| off. dS is rounded once. So each dS element is off by
  E = h |dS| + scale P h sum_d |do_d| sum_j P_j |v_jd|, and
  dq is off by sum_j E |k_j| + h |dq|, dk by sum_i E |q_i| + h |dk|.
fp32 accumulation of a few thousand terms and exp2's 2^-22 are covered by a
factor of 1.02 and 1e-5.
"""
import math

import pytest
import torch

from specdec import drafter

H = 2.0 ** -8


def _tokens(T, n_ctx, c):
    """Token of every row of a training batch's sequence, -1 for padding."""
    r = torch.arange(T)
    t = torch.where(r < n_ctx, torch.where(r < c, r, -1), c + r - n_ctx)
    return t


def _visible(pq, pk, c, W, S):
    """[queries, keys] from tokens (-1: padding)."""
    p, j = pq[:, None], pk[None]
    ctx = (j <= p) & ((p - j < W) | (j < S))
    blk = (j >= c) | (c - j <= W) | (j < S)
    return torch.where(p < c, ctx, blk) & (p >= 0) & (j >= 0)


def _oracle(q, k, v, vis, do=None, scale=None):
    """One sequence, fp64 on the CPU: q [Tq, Hq, D], k, v [Tk, Hk, D], vis
    [Tq, Tk]. Returns {name: (value, bound)}; rows and keys that are in no
    visible pair are left out of the arithmetic."""
    Hq, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    used = vis.any(0)
    rows = vis.any(1)
    z = lambda t, m: torch.where(m[:, None, None], t.double().cpu(), 0.0)  # noqa: E731
    q, k, v = z(q, rows), z(k, used), z(v, used)
    qg = q.view(-1, Hk, G, D)
    s = torch.einsum("thgd,jhd->hgtj", qg, k) * scale
    s = s.masked_fill(~vis, -math.inf)
    p = torch.exp(s - torch.logsumexp(s, -1, keepdim=True)).masked_fill(~vis, 0.0)
    o = torch.einsum("hgtj,jhd->thgd", p, v)
    oe = torch.einsum("hgtj,jhd->thgd", p, v.abs())
    out = {"o": (o.reshape(-1, Hq, D), (H * oe + H * o.abs()).reshape(-1, Hq, D))}
    if do is None:
        return out
    do = z(do, rows).view(-1, Hk, G, D)
    dv = torch.einsum("hgtj,thgd->jhd", p, do)
    dve = H * torch.einsum("hgtj,thgd->jhd", p, do.abs()) + H * dv.abs()
    dp = torch.einsum("thgd,jhd->hgtj", do, v)
    delta = (do * o).sum(-1).permute(1, 2, 0)[..., None]
    ds = p * (dp - delta) * scale
    off = H * (do.abs() * oe).sum(-1).permute(1, 2, 0)[..., None]
    e = H * ds.abs() + scale * p * off
    dq = torch.einsum("hgtj,jhd->thgd", ds, k)
    dqe = torch.einsum("hgtj,jhd->thgd", e, k.abs()) + H * dq.abs()
    dk = torch.einsum("hgtj,thgd->jhd", ds, qg)
    dke = torch.einsum("hgtj,thgd->jhd", e, qg.abs()) + H * dk.abs()
    return {**out, "dq": (dq.reshape(-1, Hq, D), dqe.reshape(-1, Hq, D)), "dk": (dk, dke), "dv": (dv, dve)}


def _near(name, got, want):
    value, bound = want
    err = (got.double().cpu() - value).abs()
    assert bool(torch.isfinite(got.float()).all()), name
    worst = (err - 1.02 * bound - 1e-5).max() if err.numel() else torch.tensor(0.0)
    assert float(worst) <= 0.0, (name, float(err.max()), float(worst))


def _rand(*shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(torch.bfloat16)


CASES = [  # B, n_ctx, n_block, Hq, Hk, D, W, S, lens
    (1, 1, 0, 1, 1, 64, 1, 0, None), (1, 0, 1, 1, 1, 128, 1, 0, None), (2, 0, 16, 4, 2, 64, 5, 3, None),
    (2, 100, 0, 2, 2, 64, 30, 0, None), (2, 300, 16, 4, 4, 64, 64, 4, None), (1, 513, 7, 2, 1, 128, 100, 1, None),
    (1, 700, 16, 6, 2, 128, 129, 70, None), (2, 257, 3, 3, 1, 64, 1, 1, None), (1, 640, 16, 5, 1, 64, 1000, 0, None),
    (4, 200, 9, 4, 2, 64, 40, 2, (0, 1, 200, 130)), (3, 333, 0, 2, 1, 128, 64, 5, (0, 333, 65)),
    (2, 128, 128, 2, 2, 128, 128, 64, (64, 128)), (1, 1500, 16, 1, 1, 64, 700, 200, None),
    (1, 400, 16, 130, 1, 64, 50, 4, None), (2, 90, 5, 7, 7, 64, None, 0, (17, 90)), (1, 1100, 33, 8, 2, 128, 256, 4, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,n_ctx,nb,Hq,Hk,D,W,S,lens", CASES)
def test_window_attention_forward_backward(cuda, B, n_ctx, nb, Hq, Hk, D, W, S, lens):
    T = n_ctx + nb
    seed = n_ctx + 10 * Hq + D
    q, do = _rand(B, T, Hq, D, seed=seed), _rand(B, T, Hq, D, seed=seed + 1)
    k, v = _rand(B, T, Hk, D, seed=seed + 2), _rand(B, T, Hk, D, seed=seed + 3)
    ctx_lens = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32)
    cs = [n_ctx] * B if lens is None else lens
    pads = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    for b, c in enumerate(cs):
        pads[b, c:n_ctx] = True
    for t in (q, k, v, do):  # padding may hold anything
        t[pads] = float("nan")
    for t in (q, k, v):
        t.requires_grad_(True)
    o = drafter.window_attention(q, k, v, n_ctx, window=W, sinks=S, ctx_lens=ctx_lens)
    grads = torch.autograd.grad(o, (q, k, v), do)
    got = dict(o=o.detach(), dq=grads[0], dk=grads[1], dv=grads[2])
    for b, c in enumerate(cs):
        tok = _tokens(T, n_ctx, c)
        vis = _visible(tok, tok, c, W or 10 ** 9, S)
        want = _oracle(q[b].detach(), k[b].detach(), v[b].detach(), vis, do[b])
        for n, t in got.items():
            _near(n, t[b], want[n])
            assert bool((t[b][pads[b]] == 0).all()), n  # padding: zero outputs and gradients
    with torch.no_grad():
        assert torch.equal(drafter.window_attention(q, k, v, n_ctx, window=W, sinks=S, ctx_lens=ctx_lens), o)
    o2 = drafter.window_attention(q, k, v, n_ctx, window=W, sinks=S, ctx_lens=ctx_lens)
    for a, c in zip(grads, torch.autograd.grad(o2, (q, k, v), do)):  # fixed summation order
        assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("B,n_ctx,nb,Hq,Hk,D,W,S,lens", [
    (2, 1584, 16, 16, 16, 64, 1540, 4, None),
    (2, 1584, 16, 16, 16, 128, 1540, 4, None),
    (1, 2000, 7, 40, 20, 128, 1700, 130, None),       # shared heads, two sink tiles
    (3, 1700, 0, 18, 6, 64, None, 0, (1700, 3, 900)),  # groups of three, padded tiles
    (3, 1650, 20, 16, 16, 128, 1600, 1, (0, 1650, 1500)),
])
def test_window_attention_of_long_windows(cuda, B, n_ctx, nb, Hq, Hk, D, W, S, lens):
    """More tiles than the device holds at once, windows of many key tiles; a few
    heads of each sequence are compared."""
    T, G = n_ctx + nb, Hq // Hk
    q, do = _rand(B, T, Hq, D, seed=1), _rand(B, T, Hq, D, seed=2)
    k, v = _rand(B, T, Hk, D, seed=3), _rand(B, T, Hk, D, seed=4)
    cs = [n_ctx] * B if lens is None else lens
    ctx_lens = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32)
    for b, c in enumerate(cs):
        for t in (q, k, v, do):
            t[b, c:n_ctx] = float("nan")
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = drafter.window_attention(*x, n_ctx, window=W, sinks=S, ctx_lens=ctx_lens)
    got = [o.detach(), *torch.autograd.grad(o, x, do)]
    with torch.no_grad():
        assert torch.equal(drafter.window_attention(*x, n_ctx, window=W, sinks=S, ctx_lens=ctx_lens), o)
    for b, c in enumerate(cs):
        for t in got:
            assert bool((t[b, c:n_ctx] == 0).all()) and bool(torch.isfinite(t[b].float()).all())
        tok = _tokens(T, n_ctx, c)
        vis = _visible(tok, tok, c, W or 10 ** 9, S)
        for h in {0, Hk - 1}:
            qs, ks = slice(h * G, (h + 1) * G), slice(h, h + 1)
            want = _oracle(q[b, :, qs].detach(), k[b, :, ks].detach(), v[b, :, ks].detach(), vis, do[b, :, qs])
            for n, t, s in zip(("o", "dq", "dk", "dv"), got, (qs, qs, ks, ks)):
                _near(n, t[b, :, s], want[n])


@pytest.mark.gpu
def test_without_window_it_is_the_dflash_attention(cuda):
    """window None, no sinks: the mask of dflash_attention; the two kernels
    round the same quantities, in tiles of their own."""
    q, k, v = (_rand(2, 528, 4, 64, seed=i) for i in range(3))
    a = drafter.window_attention(q, k, v, 512)
    b = drafter.dflash_attention(q, k, v, 512)
    assert float((a.float() - b.float()).abs().max()) <= 1e-2


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_layouts(cuda, D):
    """Views of one fused projection, heads-first tensors, rows off 16-byte
    boundaries and an expanded output gradient give the contiguous results."""
    B, T, Hq, Hk, n_ctx = 2, 150, 4, 2, 140
    qkv = _rand(B, T, (Hq + 2 * Hk) * D, seed=3)
    views = [t.unflatten(-1, (-1, D)) for t in qkv.split([Hq * D, Hk * D, Hk * D], -1)]
    first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in views]
    odd = []
    for t in views:
        u = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view(t.shape)
        odd.append(u.copy_(t))
    want = None
    for how in (views, [t.contiguous() for t in views], first, odd, [t.unsqueeze(-1).expand(*t.shape, 2)[..., 0] for t in views]):
        x = [t.detach().requires_grad_(True) for t in how]
        o = drafter.window_attention(*x, n_ctx, window=33, sinks=2)
        got = [o.detach(), *torch.autograd.grad(o.float().sum(), x)]
        want = got if want is None else want
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_rescale_path(cuda, D):
    """Scores that grow along the keys: a row's reference maximum is raised
    many times and O rescaled in tensor memory."""
    T, n_ctx = 400, 390
    q, do = _rand(1, T, 2, D, seed=1), _rand(1, T, 2, D, seed=2)
    k, v = _rand(1, T, 1, D, seed=3), _rand(1, T, 1, D, seed=4)
    k = (k.float() * (1 + torch.arange(T, device="cuda") / 8.0)[None, :, None, None]).to(torch.bfloat16)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = drafter.window_attention(*x, n_ctx, window=300, sinks=8)
    grads = torch.autograd.grad(o, x, do)
    tok = _tokens(T, n_ctx, n_ctx)
    want = _oracle(q[0].detach(), k[0].detach(), v[0].detach(), _visible(tok, tok, n_ctx, 300, 8), do[0])
    # scores reach a few hundred: the fp32 exponent s log2 e is off by up to 2^-24 |s| log2 e
    # ~ 5e-5 relative in p, below the 1e-4 added here to every relative rounding h
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        value, bound = want[n]
        _near(n, t[0].detach(), (value, bound * (1 + 1e-4 / H)))


@pytest.mark.gpu
def test_window_attention_gradient_against_differences(cuda):
    """Central differences of the fp64 definition along random directions."""
    T, n_ctx, D = 60, 50, 64
    q, do = _rand(1, T, 4, D, seed=1), _rand(1, T, 4, D, seed=2)
    k, v = _rand(1, T, 2, D, seed=3), _rand(1, T, 2, D, seed=4)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(drafter.window_attention(*x, n_ctx, window=20, sinks=3), x, do)
    tok = _tokens(T, n_ctx, n_ctx)
    vis = _visible(tok, tok, n_ctx, 20, 3)
    x64 = [t.detach()[0].double().cpu() for t in x]
    for i in range(3):
        d = torch.randn(x64[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        def loss(e):
            y = [t + e * d if n == i else t for n, t in enumerate(x64)]
            return float((_oracle(*y, vis)["o"][0] * do[0].double().cpu()).sum())
        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        got = float((grads[i][0].double().cpu() * d).sum())
        size = float(grads[i].double().norm()) * float(d.norm())
        assert abs(got - want) <= 2 * H * size, (i, got, want)


CACHED = [  # B, Tq, nb, Hq, Hk, D, size, W, S, lens
    (1, 1, 0, 1, 1, 64, 1, 1, 0, (1,)), (3, 1, 0, 4, 4, 64, 200, 50, 4, (1, 200, 77)), (2, 1, 0, 8, 2, 128, 900, 300, 4, (900, 0)),
    (2, 16, 16, 4, 4, 64, 600, 100, 4, (584, 30)), (2, 20, 16, 8, 2, 128, 700, 256, 1, (300, 2)),
    (1, 5, 4, 32, 1, 64, 3000, 2500, 4, (2996,)), (2, 300, 16, 2, 1, 128, 700, 90, 3, (600, 100)),
    (4, 3, 0, 3, 1, 64, 130, None, 0, (0, 1, 2, 130)), (1, 1, 1, 16, 1, 128, 5000, 5000, 0, (4999,)),
    (2, 2, 5, 6, 3, 64, 300, 64, 70, (295, 0)), (40, 1, 0, 8, 8, 128, 300, 200, 4, None), (1, 33, 0, 4, 4, 64, 64, 7, 2, (64,)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Tq,nb,Hq,Hk,D,size,W,S,lens", CACHED)
def test_window_attention_cached(cuda, B, Tq, nb, Hq, Hk, D, size, W, S, lens):
    if lens is None:
        lens = [(37 * b) % (size - nb + 1) for b in range(B)]
    q = _rand(B, Tq, Hq, D, seed=size + Tq)
    k, v = _rand(B, size, Hk, D, seed=size + 1), _rand(B, size, Hk, D, seed=size + 2)
    for b, c in enumerate(lens):  # rows behind the last token may hold anything
        k[b, c + nb:] = float("nan")
        v[b, c + nb:] = float("inf")
    kept = k.clone(), v.clone()
    ctx = torch.tensor(lens, device="cuda", dtype=torch.int32)
    o = drafter.window_attention_cached(q, k, v, ctx, n_block=nb, window=W, sinks=S)
    for b, c in enumerate(lens):
        pq = c + nb - Tq + torch.arange(Tq)
        pk = torch.arange(size)
        pk = torch.where(pk < c + nb, pk, -1)
        vis = _visible(pq, pk, c, W or 10 ** 9, S)
        _near("o", o[b], _oracle(q[b], k[b], v[b], vis)["o"])
    assert torch.equal(o, drafter.window_attention_cached(q, k, v, ctx.long(), n_block=nb, window=W, sinks=S))
    for a, b in zip(kept, (k, v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    # the cache as a slice of a larger one, heads first
    big = [torch.full((B, Hk, size + 3, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for t, src in zip(big, (k, v)):
        t[:, :, 2:size + 2] = src.transpose(1, 2)
    views = [t[:, :, 2:size + 2].transpose(1, 2) for t in big]
    assert torch.equal(o, drafter.window_attention_cached(q, *views, ctx, n_block=nb, window=W, sinks=S))


@pytest.mark.gpu
def test_cached_lengths_out_of_range_are_clamped(cuda):
    q, k, v = _rand(3, 2, 2, 64, seed=1), _rand(3, 50, 2, 64, seed=2), _rand(3, 50, 2, 64, seed=3)
    bad = torch.tensor([-5, 1000, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    good = torch.tensor([0, 46, 46], device="cuda", dtype=torch.int32)
    a = drafter.window_attention_cached(q, k, v, bad, n_block=4, window=16)
    assert torch.equal(a, drafter.window_attention_cached(q, k, v, good, n_block=4, window=16))
    x = _rand(3, 20, 2, 64, seed=4)
    lens = torch.tensor([-1, 99, 7], device="cuda", dtype=torch.int32)
    a = drafter.window_attention(x, x, x, 16, window=4, ctx_lens=lens)
    assert torch.equal(a, drafter.window_attention(x, x, x, 16, window=4, ctx_lens=lens.clamp(0, 16)))


def test_window_refuses_cpu_tensors():
    x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        drafter.window_attention(x, x, x, 4)
    with pytest.raises(AssertionError):
        drafter.window_attention_cached(x, x, x, torch.zeros(1, dtype=torch.int32))


def test_window_c_argument_checks():
    import ctypes

    from specdec import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced: the checks fail first

    def fwd(q=p, B=1, T=8, Hq=2, Hk=1, D=64, n_ctx=4, W=4, S=0, scale=0.125):
        return lib.specdec_window_attention_forward(q, None, p, None, p, None, p, p, p, None, B, T, Hq, Hk, D, n_ctx, W, S,
                                                    scale, None, None)

    def bwd(B=1, T=8, Hq=2, Hk=1, D=64, n_ctx=4, W=4, S=0, scale=0.125, ws=1 << 20):
        return lib.specdec_window_attention_backward(p, None, p, None, p, None, p, p, p, p, p, p, p, None, B, T, Hq, Hk, D,
                                                     n_ctx, W, S, scale, None, p, ws, None)

    def cached(B=1, T=1, size=8, Hq=2, Hk=1, D=64, nb=0, W=4, S=0, scale=0.125, lens=p):
        return lib.specdec_window_attention_cached(p, None, p, None, p, None, p, lens, B, T, size, Hq, Hk, D, nb, W, S,
                                                   scale, None, p, 1 << 30, None)

    for fn in (fwd, bwd, cached):
        for bad in (dict(D=32), dict(D=96), dict(Hq=3, Hk=2), dict(Hk=0), dict(Hq=0), dict(B=-1), dict(T=-1), dict(W=0),
                    dict(W=-3), dict(S=-1)):
            assert fn(**bad) == _lib.ERR_ARGUMENT, (fn, bad)
        for bad in (0.0, -1.0, float("nan"), float("inf")):
            assert fn(scale=bad) == _lib.ERR_VALUE
        assert fn(B=0) == _lib.OK
    for fn in (fwd, bwd):
        assert fn(n_ctx=9) == _lib.ERR_ARGUMENT and fn(n_ctx=-1) == _lib.ERR_ARGUMENT
        assert fn(T=2 ** 29, Hq=8, Hk=1, n_ctx=0) == _lib.ERR_ARGUMENT
    assert bwd(ws=16) == _lib.ERR_WORKSPACE
    assert fwd(q=ctypes.c_void_p(258)) == _lib.ERR_ARGUMENT  # not on a 16-byte boundary
    assert cached(nb=9) == _lib.ERR_ARGUMENT and cached(nb=-1) == _lib.ERR_ARGUMENT
    assert cached(lens=None) == _lib.ERR_ARGUMENT


@pytest.mark.gpu
def test_window_refusals(cuda):
    x = torch.zeros(2, 8, 4, 64, device="cuda", dtype=torch.bfloat16)
    lens = torch.zeros(2, device="cuda", dtype=torch.int32)
    for kw in (dict(window=0), dict(sinks=-1), dict(ctx_lens=lens[:1]), dict(ctx_lens=lens.cpu()), dict(ctx_lens=lens.float())):
        with pytest.raises(AssertionError):
            drafter.window_attention(x, x, x, 4, **kw)
    for args in ((x.float(), x.float(), x.float(), 4), (x, x[:, :, :3], x[:, :, :3], 4), (x, x, x, 9), (x, x, x, -1),
                 (x, x, x[:, :7], 4), (x, x[:, :7], x[:, :7], 4), (x[..., :32], x[..., :32], x[..., :32], 4), (x[0], x[0], x[0], 4)):
        with pytest.raises(AssertionError):
            drafter.window_attention(*args)
    with pytest.raises(ValueError):
        drafter.window_attention(x, x, x, 4, scale=0.0)
    with pytest.raises(AssertionError):
        drafter.window_attention_cached(x, x, x, lens, n_block=9)
    with pytest.raises(AssertionError):
        drafter.window_attention_cached(x, x[..., ::1].transpose(2, 3).contiguous().transpose(2, 3), x, lens)
    odd = torch.zeros(2 * 8 * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 8, 4, 64)
    with pytest.raises(AssertionError):  # a cache off 16-byte boundaries is refused, never copied
        drafter.window_attention_cached(x, odd, odd, lens)
    with pytest.raises(AssertionError):
        drafter.window_attention_cached(x.clone().requires_grad_(True), x, x, lens)
    e = drafter.window_attention(x[:, :0], x[:, :0], x[:, :0], 0)
    assert e.shape == (2, 0, 4, 64)


def _withheld(fn):
    """fn() with the next launch's first CTA left without its first products."""
    from specdec import _lib

    try:
        _lib.check(_lib.load().specdec_test_withhold_stage(1), "specdec_test_withhold_stage")
        out = fn()
    finally:
        _lib.load().specdec_test_withhold_stage(0)
    torch.cuda.synchronize()
    return out


def _reported():
    from specdec import ops

    with pytest.raises(RuntimeError, match="attention"):
        ops.check_backward()
    ops.check_backward()  # cleared


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hk,D,W,first", [
    (2, 300, 2, 1, 64, 40, 256),  # packed rows 512 .. 599 are tokens 256 .. 299
    (2, 2048, 16, 16, 128, None, 1920),
])
def test_an_expired_wait_of_the_forward_gives_nan_rows_and_a_report(cuda, B, T, Hq, Hk, D, W, first):
    q, k, v = _rand(B, T, Hq, D, seed=1), _rand(B, T, Hk, D, seed=2), _rand(B, T, Hk, D, seed=3)
    want = drafter.window_attention(q, k, v, T, window=W, sinks=2)
    got = _withheld(lambda: drafter.window_attention(q, k, v, T, window=W, sinks=2))
    _reported()
    lost = torch.zeros(B, T, Hq, dtype=torch.bool, device="cuda")
    lost[0, first:, :Hq // Hk] = True
    assert bool(torch.isnan(got[lost]).all()) and torch.equal(got[~lost], want[~lost])
    assert torch.equal(drafter.window_attention(q, k, v, T, window=W, sinks=2), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n_ctx,D,W,S", [(300, 300, 64, 40, 0), (2300, 2300, 128, 64, 4), (300, 290, 128, 40, 2)])
def test_an_expired_wait_of_the_backward_gives_nan_rows_and_a_report(cuda, T, n_ctx, D, W, S):
    x = [_rand(1, T, 2, D, seed=i).requires_grad_(True) for i in range(3)]
    do = _rand(1, T, 2, D, seed=5)
    o = drafter.window_attention(*x, n_ctx, window=W, sinks=S)
    want = torch.autograd.grad(o, x, do, retain_graph=True)
    got = _withheld(lambda: torch.autograd.grad(o, x, do, retain_graph=True))
    _reported()
    last = (T - 1) // 128 * 128
    for g, w, rows in zip(got, want, (slice(last, T), slice(0, 128), slice(0, 128))):
        lost = torch.zeros(1, T, 2, dtype=torch.bool, device="cuda")
        lost[0, rows, 0] = True
        assert bool(torch.isnan(g[lost]).all()) and torch.equal(g[~lost], w[~lost])
    for g, w in zip(torch.autograd.grad(o, x, do), want):
        assert torch.equal(g, w)


@pytest.mark.gpu
@pytest.mark.parametrize("size,c,W", [(900, 880, 700), (9500, 9400, 9300)])  # joined in a cluster, in the workspace
def test_an_expired_wait_of_the_cached_form_reaches_the_joined_rows(cuda, size, c, W):
    q, k, v = _rand(2, 5, 4, 64, seed=1), _rand(2, size, 2, 64, seed=2), _rand(2, size, 2, 64, seed=3)
    lens = torch.tensor([c, 500], device="cuda", dtype=torch.int32)
    run = lambda: drafter.window_attention_cached(q, k, v, lens, n_block=4, window=W, sinks=2)  # noqa: E731
    want = run()
    got = _withheld(run)
    _reported()
    lost = torch.zeros(2, 5, 4, dtype=torch.bool, device="cuda")
    lost[0, :, :2] = True
    assert bool(torch.isnan(got[lost]).all()) and torch.equal(got[~lost], want[~lost])


@pytest.mark.gpu
def test_a_cache_past_32_bit_offsets(cuda):
    """Keys and values of 2.4e9 elements each; the last sequence's last tokens
    lie past 2^31 elements."""
    B, size, Hk, D = 2, 150_000, 64, 128
    k, v = (torch.zeros(B, size, Hk, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert k.numel() > 2 ** 31
    c = size - 3
    for i, t in enumerate((k, v)):
        t[1, c - 70:] = _rand(73, Hk, D, seed=i)
    q = _rand(B, 4, Hk, D, seed=9)
    lens = torch.tensor([0, c], device="cuda", dtype=torch.int32)
    o = drafter.window_attention_cached(q, k, v, lens, n_block=3, window=60)
    tail = slice(c - 70, size)
    pk = torch.arange(c - 70, size)
    vis = _visible(c + 3 - 4 + torch.arange(4), pk, c, 60, 0)
    _near("o", o[1], _oracle(q[1], k[1, tail], v[1, tail], vis)["o"])


@pytest.mark.gpu
@pytest.mark.parametrize("B,n_ctx,nb,H,D,W,S,lens", [
    (2, 300, 7, 4, 64, 60, 3, (300, 101)), (2, 300, 7, 4, 128, 60, 70, None), (1, 90, 0, 3, 64, None, 0, None),
    (2, 1584, 16, 16, 64, 1540, 4, (1584, 1500)),
    (2, 1584, 16, 16, 128, None, 0, None),
])
def test_expanded_inputs_equal_their_copies(cuda, B, n_ctx, nb, H, D, W, S, lens):
    """Strides of zero (a head, a batch or a token broadcast) are read without
    tensor maps; the arithmetic is the same."""
    T = n_ctx + nb
    q, k, v, do = (_rand(B, T, H, D, seed=i) for i in range(4))
    ctx_lens = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32)
    for x in ((q, k[:, :, :1].expand_as(k), v[:, :, :1].expand_as(v)), (q[:1].expand_as(q), k[:1].expand_as(k), v),
              (q[:, :1].expand_as(q), k, v[:, :1].expand_as(v)), (k, k, k)):
        got = []
        for y in (x, [t.contiguous().clone() for t in x]):
            y = [t.detach().requires_grad_(True) for t in y]
            o = drafter.window_attention(*y, n_ctx, window=W, sinks=S, ctx_lens=ctx_lens)
            got.append([o.detach(), *torch.autograd.grad(o, y, do)])
        for a, b in zip(*got):
            assert bool(torch.isfinite(a.float()).all()) and torch.equal(a, b)


UNSEEN = [  # B, Tq, nb, Hq, Hk, D, size, W, S, lens; splits of the keys
    (2, 1, 0, 4, 2, 64, 900, 300, 4, (900, 640)),        # in a cluster
    (1, 3, 3, 8, 1, 128, 9500, 9000, 70, (9490,)),       # in the workspace
    (2, 1, 0, 4, 2, 64, 9000, None, 0, (9000, 100)),     # the same, most of the second's splits empty
    (40, 2, 0, 16, 16, 64, 500, 100, 33, None),          # none
    (1, 40, 3, 4, 2, 64, 2000, None, 0, (20,)),          # more queries than tokens, empty splits
    (1, 40, 3, 4, 2, 64, 9000, None, 0, (20,)),
    (3, 9, 5, 6, 2, 128, 600, 50, 130, (590, 300, 20)),  # groups of three: no map for the queries
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Tq,nb,Hq,Hk,D,size,W,S,lens", UNSEEN)
def test_cache_rows_that_no_query_sees_may_hold_anything(cuda, B, Tq, nb, Hq, Hk, D, size, W, S, lens):
    if lens is None:
        lens = [(size - 13 * b) % (size - nb + 1) for b in range(B)]
    q, k, v = _rand(B, Tq, Hq, D, seed=1), _rand(B, size, Hk, D, seed=2), _rand(B, size, Hk, D, seed=3)
    ctx = torch.tensor(lens, device="cuda", dtype=torch.int32)
    sees = []
    for b, c in enumerate(lens):
        pk = torch.arange(size)
        sees.append(_visible(c + nb - Tq + torch.arange(Tq), torch.where(pk < c + nb, pk, -1), c, W or 10 ** 9, S))
        k[b, ~sees[b].any(0)] = float("nan")
        v[b, ~sees[b].any(0)] = float("inf")
    o = drafter.window_attention_cached(q, k, v, ctx, n_block=nb, window=W, sinks=S)
    for b in range(B):
        _near("o", o[b], _oracle(q[b], k[b], v[b], sees[b])["o"])
    # one key head broadcast to all: no map for the keys
    k1, v1 = k[:, :, :1].expand_as(k), v[:, :, :1].expand_as(v)
    a, b = (drafter.window_attention_cached(q, x, y, ctx, n_block=nb, window=W, sinks=S)
            for x, y in ((k1, v1), (k1.contiguous(), v1.contiguous())))
    assert bool(torch.isfinite(a.float()).all()) and torch.equal(a, b)


@pytest.mark.gpu
def test_cached_calls_on_several_streams(cuda):
    """More CTAs of clusters at once than the device holds."""
    calls = []
    for i, (B, Hq, Hk, D, size) in enumerate([(8, 4, 4, 64, 700), (4, 8, 8, 64, 1500), (4, 16, 8, 128, 900), (2, 4, 4, 64, 600)]):
        q, k, v = _rand(B, 1, Hq, D, seed=i), _rand(B, size, Hk, D, seed=i + 10), _rand(B, size, Hk, D, seed=i + 20)
        lens = torch.full((B,), size, device="cuda", dtype=torch.int32)
        calls.append(lambda q=q, k=k, v=v, lens=lens: drafter.window_attention_cached(q, k, v, lens, window=600, sinks=4))
    want = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(30):
        for i, (f, st) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(st):
                got[i].append(f())
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.gpu
def test_a_training_batch_past_32_bit_offsets(cuda):
    """Queries of 2.16e9 elements; the last tokens of the last sequence lie past
    2^31 of them and see only one another (window 64)."""
    B, T, Hq, Hk, D, W, n = 2, 66_000, 128, 2, 128, 64, 200
    q = torch.zeros(B, T, Hq, D, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.zeros(B, T, Hk, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert q.numel() > 2 ** 31
    do = torch.zeros_like(q)
    m = n + W
    for i, t in enumerate((q, k, v, do)):
        t[1, T - m:] = _rand(m, t.shape[2], D, seed=i)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = drafter.window_attention(*x, T, window=W)
    grads = torch.autograd.grad(o, x, do)
    p = torch.arange(m) + 1000  # the first W rows see tokens in front of these: not compared
    qs, ks = slice(Hq // 2, Hq), slice(1, 2)
    want = _oracle(q[1, T - m:, qs].detach(), k[1, T - m:, ks].detach(), v[1, T - m:, ks].detach(),
                   _visible(p, p, 10 ** 6, W, 0), do[1, T - m:, qs])
    for name, t, h in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), (qs, qs, ks, ks)):
        _near(name, t[1, T - n:, h], tuple(w[m - n:] for w in want[name]))
    assert float(o[0].abs().max()) == 0.0 and float(grads[0][0].abs().max()) == 0.0


# Aggregate errors: |got - exact| / |bf16(exact) - exact| in norm. Where no query
# sees more than 64 keys, P (for o and delta), dS and o (for delta) enter their
# products in two bf16 parts, 16 bits: what is left of their rounding, 2^-17
# relative to each term, is 2^-7.7 of one rounding of the result (2^-9.3 in the
# mean), times at most 8 for terms that cancel: 1 + 0.0007. So 1.05 there; one missing
# second product makes it sqrt(2) and more (below). Elsewhere dS's rounding and the
# result's are sqrt(2) together, P's adds its square over the number of keys: 1.6.
# dv = P^T dO has P rounded once everywhere: 1.6.
ACCURATE = [  # B, n_ctx, n_block, Hq, Hk, D, W, S
    (6, 3, 0, 4, 4, 64, None, 0), (6, 5, 0, 4, 2, 128, None, 0), (4, 64, 0, 4, 4, 64, None, 0), (4, 48, 16, 8, 2, 128, None, 0),
    (4, 64, 0, 8, 2, 64, 10, 3),                                        # two query tiles, the second with a tile of sinks
    (1, 1000, 0, 4, 4, 64, 2, 0), (1, 700, 0, 2, 2, 128, 3, 0), (2, 300, 16, 4, 2, 64, 16, 4), (1, 300, 16, 8, 2, 128, 44, 4),
    (1, 300, 0, 16, 1, 64, 60, 4),                                      # two score buffers in the backward
    (1, 900, 0, 8, 1, 128, 30, 1), (1, 900, 0, 6, 2, 64, 30, 34),       # parts of sink tiles, groups of three
]
ROUNDED = [(4, 65, 0, 4, 4, 64, None, 0), (2, 256, 0, 4, 4, 64, None, 0), (2, 257, 0, 4, 2, 128, None, 0),
           (1, 400, 16, 4, 2, 64, 45, 4), (1, 400, 0, 8, 2, 128, 200, 0)]


def _ratios(got, exact):
    return {n: float((got[n].double().cpu() - e).norm() / (e.to(torch.bfloat16).double() - e).norm()) for n, e in exact.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("B,n_ctx,nb,Hq,Hk,D,W,S", ACCURATE + ROUNDED)
def test_window_attention_aggregate_errors(cuda, B, n_ctx, nb, Hq, Hk, D, W, S):
    few = (B, n_ctx, nb, Hq, Hk, D, W, S) in ACCURATE
    T = n_ctx + nb
    q, do = _rand(B, T, Hq, D, seed=1), _rand(B, T, Hq, D, seed=2)
    k, v = _rand(B, T, Hk, D, seed=3), _rand(B, T, Hk, D, seed=4)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = drafter.window_attention(*x, n_ctx, window=W, sinks=S)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, x, do))))
    tok = _tokens(T, n_ctx, n_ctx)
    vis = _visible(tok, tok, n_ctx, W or 10 ** 9, S)
    each = [_oracle(q[b].detach(), k[b].detach(), v[b].detach(), vis, do[b]) for b in range(B)]
    exact = {n: torch.stack([e[n][0] for e in each]) for n in got}
    for n, r in _ratios(got, exact).items():
        assert r <= (1.05 if few and n != "dv" else 1.6), (n, r)


@pytest.mark.parametrize("T,W", [(3, None), (64, None), (300, 2), (300, 16), (300, 60)])
def test_the_aggregate_errors_notice_a_missing_second_product(T, W):
    """The same roundings made in fp64 on the CPU: with all the second parts
    the ratios are 1.00, without any one of them (or with it the wrong way round)
    some ratio is above 1.05."""
    D, B = 64, 8
    g = torch.Generator().manual_seed(T)
    q, k, v, do = (torch.randn(B, T, D, generator=g).to(torch.bfloat16).double() for _ in range(4))
    p, j = torch.arange(T)[:, None], torch.arange(T)[None]
    vis = (j <= p) & (p - j < (W or T))

    def two(t, part):  # t as bf16 and, times ``part``, the bf16 rest
        high = t.to(torch.bfloat16).double()
        return high + part * (t - high).to(torch.bfloat16).double()

    def run(pp, ds_part, o_part, rounded=True):
        s = (q @ k.mT / 8).masked_fill(~vis, -math.inf)
        P = torch.softmax(s, -1)
        o = (two(P, pp) if rounded else P) @ v
        delta = (do * (two(o, o_part) if rounded else o)).sum(-1, keepdim=True)
        dS = P * (do @ v.mT - delta) / 8
        dS = two(dS, ds_part) if rounded else dS
        out = dict(o=o, dq=dS @ k, dk=dS.mT @ q)
        return {n: t.to(torch.bfloat16) for n, t in out.items()} if rounded else out

    exact = run(1, 1, 1, rounded=False)
    assert max(_ratios(run(1, 1, 1), exact).values()) <= 1.01
    for wrong in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (-1, 1, 1), (1, -1, 1), (1, 1, -1)):
        assert max(_ratios(run(*wrong), exact).values()) > 1.05, wrong
