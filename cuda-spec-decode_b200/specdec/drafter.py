"""The DFlash drafter's own layers on this library's kernels.

- ``rms_norm(x, weight, eps)``: RMSNorm over the last dimension (fp32 or bf16
  input, fp32 weight), forward and backward kernels of libspecdec.so; the
  weight gradient is reduced in a fixed order (bitwise repeatable).
- ``dflash_attention(q, k, v, n_ctx, scale)``: multi-head attention under the
  DFlash mask (query t < n_ctx sees keys j <= t, later queries see every key)
  for bf16 q, k, v of shape [B, T, H, 64] -- the projections' own layout.
  Forward and backward run on the tensor cores (tcgen05: products in tensor
  memory); the backward recomputes the probabilities from the forward's
  log-sum-exp and accumulates dq, dk, dv in a fixed order.
- ``rotary(x, positions, inv_freq)``: rotary positions (half or interleaved
  pairs, all or part of the head); ``rotary_frequencies`` gives the
  frequencies, also scaled for long contexts.
- ``qk_norm_rotary(q, k, q_weight, k_weight, positions, inv_freq)``: RMSNorm
  of every query and key head and the rotation in one pass.
- ``window_attention(q, k, v, n_ctx, window=, sinks=)``: attention under the
  DFlash mask with a sliding window over the context and a few first tokens
  that stay visible; shared key heads, heads of 64 or 128, padded contexts;
  forward and backward on the tensor cores. ``window_attention_cached`` is its
  serving form: the last few tokens' queries against a cache.

Reference: models/dflash/model.py:25-53 (DFlashAttention), :56-73 (the
pre-norm layer, torch.nn.RMSNorm), :123-131 (the mask).
``ENABLED`` switches the drafter modules between these kernels and plain
torch (for comparison); the kernels run only on CUDA tensors of the shapes and
dtypes above.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ENABLED = True


def set_enabled(enabled: bool) -> None:
    global ENABLED
    ENABLED = bool(enabled)


_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _stream(t: torch.Tensor) -> int:
    return _lib.stream_handle(t.device)


def _status(dev: torch.device) -> int:
    """The stream's sticky drafter status word: the attention kernels set it
    when a bounded wait expires (their failed rows are then NaN); the next
    synchronising check (specdec.ops.check_backward, a validating D-PACE
    forward, GraphedStep.check) raises RuntimeError and clears it."""
    return _lib.status_words(dev).data_ptr() + 4 * _lib.STATUS_DRAFTER


def _once(fn):
    """once_differentiable, but only where a graph of the backward is being
    built: its wrapper costs 20 us per call."""
    slow = once_differentiable(fn)

    def backward(ctx, *grads):
        return slow(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return backward


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        lib = _lib.load()
        D = x.shape[-1]
        x2 = x.contiguous().view(-1, D)
        w = weight.detach().float().contiguous()
        y = torch.empty_like(x2)
        rstd = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
        with _lib.on_device(x.device):
            _lib.check(lib.specdec_rmsnorm_forward(x2.data_ptr(), w.data_ptr(), y.data_ptr(), rstd.data_ptr(),
                                                   x2.shape[0], D, float(eps), _DTYPES[x.dtype], _stream(x)),
                       "specdec_rmsnorm_forward")
        ctx.save_for_backward(x2, w, rstd)
        ctx.wdtype = weight.dtype
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        lib = _lib.load()
        x2, w, rstd = ctx.saved_tensors
        D = x2.shape[-1]
        dy2 = dy.to(x2.dtype).contiguous().view(-1, D)
        dx = torch.empty_like(x2)
        dw = torch.empty(D, dtype=torch.float32, device=x2.device)
        with _lib.on_device(x2.device):
            ws_bytes = lib.specdec_rmsnorm_workspace_bytes(x2.shape[0], D, x2.device.index)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x2.device)
            _lib.check(lib.specdec_rmsnorm_backward(x2.data_ptr(), w.data_ptr(), rstd.data_ptr(), dy2.data_ptr(),
                                                    dx.data_ptr(), dw.data_ptr(), x2.shape[0], D, _DTYPES[x2.dtype],
                                                    ws.data_ptr(), ws_bytes, _stream(x2)),
                       "specdec_rmsnorm_backward")
        return dx.view(dy.shape), dw.to(ctx.wdtype), None


def rms_norm_supported(x: torch.Tensor, weight: torch.Tensor | None) -> bool:
    return (ENABLED and x.is_cuda and x.dtype in _DTYPES and weight is not None
            and weight.dtype == torch.float32 and x.shape[-1] == weight.numel() and x.numel() > 0)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float | None = None) -> torch.Tensor:
    """RMSNorm of the last dimension; eps None = finfo(x.dtype).eps (torch's default)."""
    e = torch.finfo(x.dtype).eps if eps is None else float(eps)
    return _RMSNorm.apply(x, weight, e)


class _DFlashAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, n_ctx, scale):
        lib = _lib.load()
        B, T, H, Dh = q.shape
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        o = torch.empty_like(q)
        lse = torch.empty(B, H, T, dtype=torch.float32, device=q.device)
        with _lib.on_device(q.device):
            _lib.check(lib.specdec_dflash_attention_forward(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), B, T, H, Dh,
                int(n_ctx), float(scale), _status(q.device), _stream(q)), "specdec_dflash_attention_forward")
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.n_ctx, ctx.scale = int(n_ctx), float(scale)
        return o

    @staticmethod
    def backward(ctx, do):
        lib = _lib.load()
        q, k, v, o, lse = ctx.saved_tensors
        B, T, H, Dh = q.shape
        do = do.to(q.dtype).contiguous()
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        with _lib.on_device(q.device):
            ws_bytes = lib.specdec_dflash_attention_workspace_bytes(B, T, H)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
            _lib.check(lib.specdec_dflash_attention_backward(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), do.data_ptr(),
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, T, H, Dh, ctx.n_ctx, ctx.scale, _status(q.device),
                ws.data_ptr(), ws_bytes, _stream(q)), "specdec_dflash_attention_backward")
        return dq, dk, dv, None, None


def attention_supported(q: torch.Tensor) -> bool:
    return (ENABLED and q.is_cuda and q.dtype == torch.bfloat16 and q.dim() == 4 and q.shape[-1] == 64
            and q.shape[1] <= 65535 * 128)


def dflash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n_ctx: int,
                     scale: float | None = None) -> torch.Tensor:
    """Attention under the DFlash mask; q, k, v bf16 [B, T, H, 64] -> o [B, T, H, 64]."""
    s = q.shape[-1] ** -0.5 if scale is None else float(scale)
    return _DFlashAttention.apply(q, k, v, n_ctx, s)


# ---- rotary positions, norms of queries and keys --------------------------------

def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str | None = None, *, factor: float = 1.0,
                       original_length: int | None = None, low: float | None = None, high: float | None = None,
                       device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq, scale) for ``rotary`` over ``dim`` elements of a head:
    inv_freq[i] = base^(-2i / dim), fp64 [dim / 2] on ``device``, and the factor
    on the rotated elements. ``scaling`` stretches them to contexts ``factor``
    times as long as the ``original_length`` they were trained for:

    - "linear": every frequency divided by factor (positions interpolated);
    - "ntk": base * factor^(dim / (dim - 2)): the slowest pair is divided by
      factor, the fastest stays;
    - "ramp": pairs that turn more than ``high`` times within original_length
      stay, those that turn less than ``low`` times are divided by factor, a
      linear ramp in the number of turns between them (defaults 1 and 4);
    - "yarn": the ramp from 1 to 32 turns, and scale 0.1 ln(factor) + 1
      (Peng et al., 2023, arXiv:2309.00071, equations 17, 18 and 22).
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and >= 2, got {dim}")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be > 0")
    exponent = -torch.arange(0, dim, 2, dtype=torch.float64) / dim
    freq = float(base) ** exponent
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs dim >= 4")
        freq = (float(base) * factor ** (dim / (dim - 2))) ** exponent
    elif scaling in ("ramp", "yarn"):
        if original_length is None or original_length < 1:
            raise ValueError(f"{scaling} scaling needs original_length >= 1")
        lo, hi = (1.0, 4.0) if scaling == "ramp" else (1.0, 32.0)
        lo, hi = lo if low is None else float(low), hi if high is None else float(high)
        if not hi > lo:
            raise ValueError("high must be > low")
        keep = ((original_length * freq / (2.0 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        freq = keep * freq + (1.0 - keep) * freq / factor
        if scaling == "yarn":
            scale = 0.1 * math.log(max(factor, 1.0)) + 1.0
    elif scaling is not None:
        raise ValueError(f"unknown scaling {scaling!r}, expected linear, ntk, ramp or yarn")
    return freq.to(device=device), scale


def _strided(t: torch.Tensor) -> torch.Tensor:
    """A head's elements contiguous; the other dimensions as they are."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _new(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor shaped as t (empty_like costs the
    host half of torch.empty)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """The C ABI's three element strides (None: contiguous)."""
    return None if t.is_contiguous() else (ctypes.c_int64 * 3)(*t.stride()[:3])


def _check_heads(name: str, x: torch.Tensor, like: torch.Tensor | None = None) -> None:
    assert x.is_cuda and x.dim() == 4 and x.dtype in _DTYPES, f"{name} must be cuda float32 or bfloat16 [B, T, heads, D]"
    if like is not None:
        assert x.device == like.device and x.dtype == like.dtype and x.shape[:2] == like.shape[:2] \
            and x.shape[3] == like.shape[3], f"{name} must match q's device, dtype, batch, length and head size"


def _check_rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    assert positions.device == x.device and positions.dtype in (torch.int64, torch.int32) \
        and (positions.shape == x.shape[:2] or positions.shape == x.shape[1:2]), \
        "positions must be int64 (or int32) [T] or [B, T] on the heads' device"
    assert inv_freq.device == x.device and inv_freq.dtype == torch.float64 and inv_freq.dim() == 1, \
        "inv_freq must be float64 [rotary_dim / 2] on the heads' device"
    assert 0 < 2 * inv_freq.numel() <= x.shape[3], "inv_freq must turn at least one pair and at most the head"
    positions = positions.long()
    if positions.stride(-1) != 1 and positions.shape[-1] > 1:
        positions = positions.contiguous()
    return positions, inv_freq.contiguous()


def _position_stride(positions: torch.Tensor) -> int:
    return positions.stride(0) if positions.dim() == 2 else 0


def _rotary(x, positions, inv_freq, interleaved, scale, inverse):
    lib = _lib.load()
    B, T, H, D = x.shape
    x = _strided(x)
    y = _new(x)
    with _lib.on_device(x.device):
        _lib.check(lib.specdec_rotary(
            x.data_ptr(), _strides(x), y.data_ptr(), positions.data_ptr(), _position_stride(positions),
            inv_freq.data_ptr(), B, T, H, D, 2 * inv_freq.numel(), interleaved, scale, inverse, _DTYPES[x.dtype],
            _stream(x)), "specdec_rotary")
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, interleaved, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = interleaved, scale
        return _rotary(x, positions, inv_freq, interleaved, scale, 0)

    @staticmethod
    @_once
    def backward(ctx, dy):
        positions, inv_freq = ctx.saved_tensors
        return _rotary(dy, positions, inv_freq, *ctx.how, 1), None, None, None, None


def rotary_supported(x: torch.Tensor) -> bool:
    return (ENABLED and x.is_cuda and x.dtype in _DTYPES and x.dim() == 4 and x.shape[3] % 2 == 0
            and 0 < x.shape[3] <= 512)


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           scale: float = 1.0) -> torch.Tensor:
    """Rotary positions of every head of x [B, T, heads, D] (fp32 or bf16, any
    strides; D even, <= 512): of the first R = 2 len(inv_freq) elements, pair i
    -- (i, i + R/2), or (2i, 2i + 1) with ``interleaved`` -- turns by the angle
    position * inv_freq[i] and is multiplied by ``scale``; the rest is copied.
    positions: int64 [T] or [B, T]; inv_freq: fp64 (``rotary_frequencies``).
    Angles are formed in fp64. Differentiable in x."""
    _check_heads("x", x)
    positions, inv_freq = _check_rotary(x, positions, inv_freq)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotary.apply(x, positions, inv_freq, int(bool(interleaved)), float(scale))
    return _rotary(x, positions, inv_freq, int(bool(interleaved)), float(scale), 0)


def _qk_norm_rotary(q, k, wq, wk, positions, inv_freq, eps, interleaved, scale):
    lib = _lib.load()
    B, T, Hq, D = q.shape
    yq, yk = _new(q), _new(k)
    with _lib.on_device(q.device):
        _lib.check(lib.specdec_qk_norm_rotary_forward(
            q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), wq.data_ptr(), wk.data_ptr(), yq.data_ptr(),
            yk.data_ptr(), positions.data_ptr(), _position_stride(positions), inv_freq.data_ptr(), B, T, Hq, k.shape[2],
            D, 2 * inv_freq.numel(), interleaved, scale, eps, _DTYPES[q.dtype], _stream(q)),
            "specdec_qk_norm_rotary_forward")
    return yq, yk


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved, scale):
        q, k = _strided(q), _strided(k)
        wq, wk = q_weight.float().contiguous(), k_weight.float().contiguous()
        ctx.save_for_backward(q, k, wq, wk, positions, inv_freq)
        ctx.how = eps, interleaved, scale
        ctx.wdtypes = q_weight.dtype, k_weight.dtype
        return _qk_norm_rotary(q, k, wq, wk, positions, inv_freq, eps, interleaved, scale)

    @staticmethod
    @_once
    def backward(ctx, dyq, dyk):
        lib = _lib.load()
        q, k, wq, wk, positions, inv_freq = ctx.saved_tensors
        eps, interleaved, scale = ctx.how
        B, T, Hq, D = q.shape
        Hk = k.shape[2]
        dyq, dyk = _strided(dyq), _strided(dyk)
        dq, dk, dwq, dwk = _new(q), _new(k), _new(wq), _new(wk)
        with _lib.on_device(q.device):
            ws_bytes = lib.specdec_qk_norm_rotary_workspace_bytes(B, T, D, q.device.index)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
            _lib.check(lib.specdec_qk_norm_rotary_backward(
                q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), wq.data_ptr(), wk.data_ptr(), dyq.data_ptr(),
                _strides(dyq), dyk.data_ptr(), _strides(dyk), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(),
                dwk.data_ptr(), positions.data_ptr(), _position_stride(positions), inv_freq.data_ptr(), B, T, Hq, Hk,
                D, 2 * inv_freq.numel(), interleaved, scale, eps, _DTYPES[q.dtype], ws.data_ptr(), ws_bytes,
                _stream(q)), "specdec_qk_norm_rotary_backward")
        return dq, dk, dwq.to(ctx.wdtypes[0]), dwk.to(ctx.wdtypes[1]), None, None, None, None, None


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                   positions: torch.Tensor, inv_freq: torch.Tensor, *, eps: float | None = None,
                   interleaved: bool = False, scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm over the elements of every head of q [B, T, Hq, D] and k
    [B, T, Hk, D] (weights [D]; eps None = finfo(dtype).eps), then ``rotary`` of
    both, in one pass: x / sqrt(mean(x^2) + eps) * weight, rotated. fp32 or bf16,
    any strides (views of one fused projection); fp32 arithmetic, one rounding.
    Differentiable in q, k and the weights (their gradients are summed in a
    fixed order)."""
    _check_heads("q", q)
    _check_heads("k", k, q)
    D = q.shape[3]
    assert q_weight.shape == (D,) and k_weight.shape == (D,) and q_weight.device == q.device \
        and k_weight.device == q.device, "weights must be [D] on q's device"
    positions, inv_freq = _check_rotary(q, positions, inv_freq)
    e = torch.finfo(q.dtype).eps if eps is None else float(eps)
    how = e, int(bool(interleaved)), float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad
                                    or k_weight.requires_grad):
        return _QKNormRotary.apply(q, k, q_weight, k_weight, positions, inv_freq, *how)
    return _qk_norm_rotary(_strided(q), _strided(k), q_weight.float().contiguous(), k_weight.float().contiguous(),
                           positions, inv_freq, *how)


# ---- sliding-window attention with sinks ------------------------------------------

_NO_WINDOW = 2 ** 31 - 1


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t itself if every row of a head starts on a 16-byte boundary, else a copy."""
    if t.data_ptr() % 16 == 0 and (t.is_contiguous() or t.stride(3) == 1 and all(
            t.stride(d) % 8 == 0 or t.shape[d] <= 1 for d in range(3))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_window(q, k, v, window, sinks, scale) -> tuple[int, int, float]:
    assert q.is_cuda and q.dtype == torch.bfloat16 and q.dim() == 4, "q must be cuda bfloat16 [B, T, heads, D]"
    assert q.shape[3] in (64, 128), f"heads must have 64 or 128 elements, got {q.shape[3]}"
    assert k.dim() == 4 and k.shape == v.shape and k.shape[0] == q.shape[0] and k.shape[3] == q.shape[3], \
        "k and v must be [B, T, k_heads, D] with q's batch and head size"
    assert k.dtype == q.dtype and v.dtype == q.dtype and k.device == q.device and v.device == q.device, \
        "k and v must have q's dtype and device"
    assert k.shape[2] > 0 and q.shape[2] > 0 and q.shape[2] % k.shape[2] == 0, \
        f"query heads must be a multiple of key heads ({q.shape[2]}, {k.shape[2]})"
    assert window is None or window >= 1, f"window must be >= 1 or None, got {window}"
    assert sinks >= 0, f"sinks must be >= 0, got {sinks}"
    return (_NO_WINDOW if window is None else min(int(window), _NO_WINDOW), min(int(sinks), _NO_WINDOW),
            q.shape[3] ** -0.5 if scale is None else float(scale))


def _check_lens(ctx_lens: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    assert ctx_lens.shape == (q.shape[0],) and ctx_lens.dtype in (torch.int32, torch.int64) \
        and ctx_lens.device == q.device, "ctx_lens must be int32 (or int64) [B] on q's device"
    return ctx_lens.to(torch.int32).contiguous()


def _window_forward(q, k, v, ctx_lens, n_ctx, window, sinks, scale, train):
    lib = _lib.load()
    B, T, Hq, D = q.shape
    Hk = k.shape[2]
    o = _new(q)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device) if train else None
    res = _new(q) if train else None  # what o's rounding took away: the backward's delta needs it
    with _lib.on_device(q.device):
        _lib.check(lib.specdec_window_attention_forward(
            q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), o.data_ptr(),
            _lib.ptr(res), _lib.ptr(lse), _lib.ptr(ctx_lens), B, T, Hq, Hk, D, n_ctx, window, sinks, scale, _status(q.device),
            _stream(q)), "specdec_window_attention_forward")
    return o, res, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, ctx_lens, n_ctx, window, sinks, scale):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        o, res, lse = _window_forward(q, k, v, ctx_lens, n_ctx, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, o, res, lse, ctx_lens)
        ctx.how = n_ctx, window, sinks, scale
        return o

    @staticmethod
    @_once
    def backward(ctx, do):
        lib = _lib.load()
        q, k, v, o, res, lse, ctx_lens = ctx.saved_tensors
        B, T, Hq, D = q.shape
        Hk = k.shape[2]
        do = do.contiguous()
        if do.data_ptr() % 16:
            do = do.clone()
        dq, dk, dv = _new(q), _new(k), _new(v)
        with _lib.on_device(q.device):
            ws_bytes = lib.specdec_window_attention_workspace_bytes(B, T, Hq, Hk, D, *ctx.how[:3], q.device.index)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
            _lib.check(lib.specdec_window_attention_backward(
                q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), o.data_ptr(),
                res.data_ptr(), lse.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(ctx_lens), B, T,
                Hq, Hk, D, *ctx.how, _status(q.device), ws.data_ptr(), ws_bytes, _stream(q)),
                "specdec_window_attention_backward")
        return dq, dk, dv, None, None, None, None, None


def window_attention_supported(q: torch.Tensor) -> bool:
    return ENABLED and q.is_cuda and q.dtype == torch.bfloat16 and q.dim() == 4 and q.shape[-1] in (64, 128)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n_ctx: int, *, window: int | None = None,
                     sinks: int = 0, scale: float | None = None, ctx_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention under the DFlash mask with a sliding window; q bf16
    [B, T, Hq, D], k and v [B, T, Hk, D] (Hk divides Hq: head h reads key head
    h // (Hq // Hk); D 64 or 128; any strides) -> o [B, T, Hq, D].

    The first n_ctx rows are context, the others block slots (n_ctx = T: an
    ordinary causal attention). A context query sees, of the keys up to itself,
    the last ``window`` (itself included; None: all) and the first ``sinks``;
    a block query sees every block token, the last ``window`` context tokens and
    the sinks. ctx_lens int32 [B] (None: all n_ctx): sequence b has only
    ctx_lens[b] context tokens, in rows 0 .. ctx_lens[b]-1; the rows behind
    them up to n_ctx are padding, never read, with zero outputs and gradients.
    Differentiable in q, k, v; scale None = D^-0.5."""
    window, sinks, scale = _check_window(q, k, v, window, sinks, scale)
    assert k.shape[1] == q.shape[1], "k and v must have q's length"
    assert 0 <= n_ctx <= q.shape[1], f"n_ctx must be in [0, T], got {n_ctx}"
    if ctx_lens is not None:
        ctx_lens = _check_lens(ctx_lens, q)
    how = int(n_ctx), window, sinks, scale
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(q, k, v, ctx_lens, *how)
    return _window_forward(_rows16(q), _rows16(k), _rows16(v), ctx_lens, *how, False)[0]


def window_attention_cached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, ctx_lens: torch.Tensor, *,
                            n_block: int = 0, window: int | None = None, sinks: int = 0,
                            scale: float | None = None) -> torch.Tensor:
    """``window_attention`` of the last tokens of each sequence against a cache,
    forward only. k_cache, v_cache bf16 [B, size, Hk, D] hold sequence b's
    ctx_lens[b] context tokens (int32 [B], at most size - n_block) in rows
    0, 1, ... and its n_block block tokens right behind them; later rows are
    never read. q [B, Tq, Hq, D] are the sequence's last Tq tokens, context and
    block together (Tq = 1, n_block = 0: the next token); a query in front of
    the first token gives zeros. The cache is read in place: its rows must start
    on 16-byte boundaries."""
    window, sinks, scale = _check_window(q, k_cache, v_cache, window, sinks, scale)
    assert not (torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad)), \
        "window_attention_cached has no backward: call it under torch.no_grad()"
    ctx_lens = _check_lens(ctx_lens, q)
    lib = _lib.load()
    B, Tq, Hq, D = q.shape
    size, Hk = k_cache.shape[1], k_cache.shape[2]
    assert k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the cache's heads must be contiguous"
    assert 0 <= n_block <= size, f"n_block must be in [0, size of the cache], got {n_block}"
    q = _rows16(q)
    o = _new(q)
    with _lib.on_device(q.device):
        ws_bytes = lib.specdec_window_attention_cached_workspace_bytes(B, Tq, size, Hq, Hk, D, n_block, window, sinks,
                                                                       q.device.index)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        _lib.check(lib.specdec_window_attention_cached(
            q.data_ptr(), _strides(q), k_cache.data_ptr(), _strides(k_cache), v_cache.data_ptr(), _strides(v_cache),
            o.data_ptr(), ctx_lens.data_ptr(), B, Tq, size, Hq, Hk, D, int(n_block), window, sinks, scale,
            _status(q.device), _lib.ptr(ws), ws_bytes, _stream(q)), "specdec_window_attention_cached")
    return o
