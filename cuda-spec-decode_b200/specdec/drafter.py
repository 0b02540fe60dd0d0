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

import math

import torch

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
    """RMSNorm of the last dimension; eps None = finfo(x.dtype).eps. (torch's own
    rms_norm takes fp32's eps for bf16 inputs: the drafter's modules pass that.)"""
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


def _ops():
    """The torch binding of these operators (csrc/drafter_bind.cpp): checks,
    outputs, streams and autograd in C++ over the same C ABI."""
    global _torch_ops
    if _torch_ops is None:
        _lib.load()  # raises if the library is not built
        try:
            from . import _torch_ops as module
        except ImportError as e:
            raise ImportError("_torch_ops.so is not built; build it with `make -C cuda-spec-decode_b200/csrc` or "
                              "__graft_entry__.build()") from e
        _torch_ops = module
    return _torch_ops


_torch_ops = None


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
    return _ops().rotary(x, positions, inv_freq, interleaved, scale)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                   positions: torch.Tensor, inv_freq: torch.Tensor, *, eps: float | None = None,
                   interleaved: bool = False, scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm over the elements of every head of q [B, T, Hq, D] and k
    [B, T, Hk, D] (weights [D]; eps None: fp32's 2^-23 for both types, as torch's
    rms_norm takes it), then ``rotary`` of both, in one pass: x / sqrt(mean(x^2) + eps) * weight, rotated. fp32 or bf16,
    any strides (views of one fused projection); fp32 arithmetic, one rounding.
    Differentiable in q, k and the weights (their gradients are summed in a
    fixed order)."""
    return _ops().qk_norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved, scale)


# ---- sliding-window attention with sinks ------------------------------------------

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
    them up to n_ctx are padding: they may hold anything, their outputs and
    gradients are zero.
    Differentiable in q, k, v; scale None = D^-0.5. Products take bf16 operands
    and sum in fp32; where no query can see more than 64 keys (min(T, window +
    sinks + block)) the probabilities of the forward and the scores' gradients
    enter in two bf16 parts."""
    return _ops().window_attention(q, k, v, n_ctx, window, sinks, scale, ctx_lens)


def window_attention_cached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, ctx_lens: torch.Tensor, *,
                            n_block: int = 0, window: int | None = None, sinks: int = 0,
                            scale: float | None = None) -> torch.Tensor:
    """``window_attention`` of the last tokens of each sequence against a cache,
    forward only. k_cache, v_cache bf16 [B, size, Hk, D] hold sequence b's
    ctx_lens[b] context tokens (int32 [B], at most size - n_block) in rows
    0, 1, ... and its n_block block tokens right behind them; later rows, and
    rows that no query sees (between the sinks and the first query's window),
    may hold anything. q [B, Tq, Hq, D] are the sequence's last Tq tokens,
    context and block together (Tq = 1, n_block = 0: the next token); a query in
    front of the first token gives zeros. The cache is read in place: its rows
    must start on 16-byte boundaries."""
    return _ops().window_attention_cached(q, k_cache, v_cache, ctx_lens, n_block, window, sinks, scale)
