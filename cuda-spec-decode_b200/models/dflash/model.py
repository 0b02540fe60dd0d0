"""DFlash block drafter with the swappable-objective hook.

Interface-compatible with harvestingmoon/cuda-spec-decode
models/dflash/model.py: same class names, constructor arguments, parameter
names (so state dicts load either way), attention mask rule and the
``compute_loss(target_features, ground_truth_block_tokens, loss_fn=None)``
hook (model.py:152-170) that lets the fused losses of this library replace
plain cross entropy.

Architecture (model.py:76-150): target features -> proj_in -> append
``block_size`` trainable slot queries -> pre-RMSNorm transformer layers under
a mask where context tokens are causal and block tokens see every token ->
RMSNorm -> proj_out -> optional RMSNorm -> frozen verifier lm_head ->
[batch, block_size, V] logits. The mask is applied by its structure (the
context causal, the block queries over every token), never as a [T, T]
tensor. Layers on this library's kernels (specdec.drafter): the RMSNorms
(fp32 or bf16 activations) and, for bf16 q/k/v with 64-dim heads (e.g.
under bf16 autocast), the attention forward on the tensor cores; otherwise
attention runs through F.scaled_dot_product_attention (a causal attention
over the context plus an unmasked one for the block queries). GEMMs are
cuBLAS (nn.Linear).

Beyond the reference, for long contexts (``attention=dict(...)`` of
DFlashSpeculator; all off by default): rotary positions (the context's tokens
at 0, 1, ..., the block behind them), norms of queries and keys, key heads
shared by groups of query heads, a sliding window over the context with a few
first tokens that stay visible, contexts of different lengths in one batch
(``ctx_lens``), and drafting from a cache of keys and values
(``new_cache`` / ``draft(..., cache=)``). On bf16 CUDA activations they run on
specdec.drafter's kernels, elsewhere on plain torch operations.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from specdec import drafter as _kernels


class RMSNorm(nn.RMSNorm):
    """torch.nn.RMSNorm (same parameters and state-dict keys) whose forward
    runs the library's RMSNorm kernels on CUDA tensors. eps None: fp32's, which
    torch takes for bf16 inputs too."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if len(self.normalized_shape) == 1 and _kernels.rms_norm_supported(x, self.weight):
            return _kernels.rms_norm(x, self.weight, torch.finfo(torch.float32).eps if self.eps is None else self.eps)
        return super().forward(x)


def _rotate_plain(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool,
                  scale: float) -> torch.Tensor:
    """specdec.drafter.rotary in torch operations (angles in fp64)."""
    R = 2 * inv_freq.numel()
    ang = positions.double()[..., None] * inv_freq
    if ang.dim() == 2:
        ang = ang[None]
    cos, sin = ((t * scale).to(x.dtype)[:, :, None] for t in (ang.cos(), ang.sin()))
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _window_plain(q, k, v, tokens_q, tokens_k, ctx_lens, window, sinks) -> torch.Tensor:
    """The windowed DFlash attention in torch operations. tokens_q [B, Tq],
    tokens_k [B, Tk]: each row's place in its sequence, -1 for padding (zero
    output, seen by nobody); ctx_lens [B]."""
    p, j, c = tokens_q[:, :, None], tokens_k[:, None, :], ctx_lens.view(-1, 1, 1)
    W = 2 ** 31 if window is None else window
    seen = torch.where(p < c, (j <= p) & ((p - j < W) | (j < sinks)), (j >= c) | (c - j <= W) | (j < sinks))
    seen = seen & (p >= 0) & (j >= 0)
    some = seen.any(-1, keepdim=True)
    G = q.shape[2] // k.shape[2]
    live = (tokens_k >= 0)[:, :, None, None]
    k, v = (torch.where(live, t, 0).transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    y = F.scaled_dot_product_attention(q.transpose(1, 2), k, v, attn_mask=(seen | ~some)[:, None])
    return torch.where(some[:, None], y, 0).transpose(1, 2)


class DFlashAttention(nn.Module):
    """Multi-head attention taking an additive mask (reference model.py:25-53).

    Options beyond the reference, off by default:
    num_kv_heads  key / value heads, each shared by num_heads / num_kv_heads
                  query heads (None: num_heads)
    qk_norm       RMSNorm of every query and key head (weights q_norm, k_norm)
    rotary        rotary positions: a dict of specdec.drafter.rotary_frequencies'
                  arguments (dim: the rotated elements of the head, default all)
                  and ``interleaved``; None: no positions
    window, sinks context tokens a query sees: the last ``window`` (None: all)
                  and the first ``sinks``
    """

    def __init__(self, d_model: int, num_heads: int, qkv_bias: bool = False, *, num_kv_heads: int | None = None,
                 qk_norm: bool = False, rotary: dict | None = None, window: int | None = None, sinks: int = 0):
        super().__init__()
        if d_model % num_heads:
            raise AssertionError("d_model must be divisible by num_heads")
        self.d_model = d_model
        self.num_heads = num_heads
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if self.num_kv_heads < 1 or num_heads % self.num_kv_heads:
            raise AssertionError("num_heads must be a multiple of num_kv_heads")
        if (window is not None and window < 1) or sinks < 0:
            raise AssertionError("window must be >= 1 or None, sinks >= 0")
        self.head_dim = d_model // num_heads
        kv = self.num_kv_heads * self.head_dim
        self.q_proj = nn.Linear(d_model, d_model, bias=qkv_bias)
        self.k_proj = nn.Linear(d_model, kv, bias=qkv_bias)
        self.v_proj = nn.Linear(d_model, kv, bias=qkv_bias)
        self.out_proj = nn.Linear(d_model, d_model, bias=qkv_bias)
        self.q_norm = RMSNorm(self.head_dim, eps=1e-6) if qk_norm else None
        self.k_norm = RMSNorm(self.head_dim, eps=1e-6) if qk_norm else None
        self.window, self.sinks = window, sinks
        self.rotary = None
        if rotary is not None:
            opts = dict(rotary)
            self.interleaved = bool(opts.pop("interleaved", False))
            self.rotary = (opts.pop("dim", self.head_dim), opts)
            if not 2 <= self.rotary[0] <= self.head_dim:
                raise AssertionError("rotary dim must be in [2, head_dim]")
            # fp64, kept apart from the module's buffers: .to(dtype) must not round it
            with torch.inference_mode(False), torch.device("cpu"):
                self._freq = {torch.device("cpu"): _kernels.rotary_frequencies(self.rotary[0], **opts)}
            self._frequencies(self.q_proj.weight.device)
        self.extended = (qk_norm or rotary is not None or window is not None or sinks > 0
                         or self.num_kv_heads != num_heads)

    def _heads(self, t: torch.Tensor) -> torch.Tensor:
        b, s, _ = t.shape
        return t.view(b, s, self.num_heads, self.head_dim).transpose(1, 2)

    def _frequencies(self, device: torch.device):
        """(inv_freq, scale) on ``device``: a copy kept for the module's life, so
        never an inference tensor (a later training step saves it for its
        backward). Made when the module moves there: a first use inside a graph
        capture could not copy from the host."""
        got = self._freq.get(device)
        if got is None:
            freq, scale = self._freq[torch.device("cpu")]
            with torch.inference_mode(False):
                got = self._freq[device] = (freq.to(device), scale)
        return got

    def _apply(self, fn, *args, **kwargs):  # .to(), .cuda(), ...
        super()._apply(fn, *args, **kwargs)
        first = next(self.parameters(), None)
        if self.rotary is not None and first is not None:
            self._frequencies(first.device)
        return self

    def _project(self, x: torch.Tensor, positions: torch.Tensor):
        """Queries, keys and values [B, T, heads, D], normalised and rotated."""
        b, s, _ = x.shape
        q = self.q_proj(x).view(b, s, self.num_heads, self.head_dim)
        k = self.k_proj(x).view(b, s, self.num_kv_heads, self.head_dim)
        v = self.v_proj(x).view(b, s, self.num_kv_heads, self.head_dim)
        if self.rotary is None:
            if self.q_norm is not None:
                q, k = self.q_norm(q), self.k_norm(k)
            return q, k, v
        freq, scale = self._frequencies(x.device)
        if _kernels.rotary_supported(q):
            if self.q_norm is not None:
                q, k = _kernels.qk_norm_rotary(q, k, self.q_norm.weight, self.k_norm.weight, positions, freq,
                                               eps=self.q_norm.eps, interleaved=self.interleaved, scale=scale)
            else:
                q, k = (_kernels.rotary(t, positions, freq, interleaved=self.interleaved, scale=scale) for t in (q, k))
            return q, k, v
        if self.q_norm is not None:
            q, k = self.q_norm(q), self.k_norm(k)
        return *(_rotate_plain(t, positions, freq, self.interleaved, scale) for t in (q, k)), v

    def forward(self, x: torch.Tensor, attn_mask: torch.Tensor | None = None,
                n_ctx: int | None = None, ctx_lens: torch.Tensor | None = None) -> torch.Tensor:
        """attn_mask: additive [.., T, T] mask (the reference's form). n_ctx
        instead states the DFlash mask by its structure -- the first n_ctx
        tokens causal among themselves and blind to the rest, the others
        seeing every token -- and runs it as two mask-free attentions (causal
        over the context; the block queries over all keys), which the fused
        SDPA kernels handle without reading a [T, T] mask. With n_ctx, ctx_lens
        int [B] gives each sequence's own context length (the rows behind it up
        to n_ctx are padding: no other row sees them, but the projections' weight
        gradients multiply them by zero, so they have to be finite), and the
        options above apply."""
        b, s, _ = x.shape
        if self.extended or ctx_lens is not None:
            if attn_mask is not None or n_ctx is None:
                raise AssertionError("the options and ctx_lens need n_ctx instead of an explicit mask")
            return self._forward_window(x, n_ctx, ctx_lens)
        if n_ctx is not None and attn_mask is None:
            qs = self.q_proj(x).view(b, s, self.num_heads, self.head_dim)
            if _kernels.attention_supported(qs):  # [b, s, heads, dim]: the kernels' layout
                ks = self.k_proj(x).view(b, s, self.num_heads, self.head_dim)
                vs = self.v_proj(x).view(b, s, self.num_heads, self.head_dim)
                y = _kernels.dflash_attention(qs, ks.to(qs.dtype), vs.to(qs.dtype), n_ctx)
                return self.out_proj(y.reshape(b, s, self.d_model))
        q, k, v = self._heads(self.q_proj(x)), self._heads(self.k_proj(x)), self._heads(self.v_proj(x))
        if n_ctx is not None and attn_mask is None:
            y_ctx = F.scaled_dot_product_attention(q[:, :, :n_ctx], k[:, :, :n_ctx], v[:, :, :n_ctx],
                                                   is_causal=True)
            y_blk = F.scaled_dot_product_attention(q[:, :, n_ctx:], k, v)
            y = torch.cat([y_ctx, y_blk], dim=2)
        else:
            mask = None if attn_mask is None else attn_mask.to(q.dtype)
            y = F.scaled_dot_product_attention(q, k, v, attn_mask=mask)
        return self.out_proj(y.transpose(1, 2).reshape(b, s, self.d_model))

    def _forward_window(self, x: torch.Tensor, n_ctx: int, ctx_lens: torch.Tensor | None) -> torch.Tensor:
        b, s, _ = x.shape
        row = torch.arange(s, device=x.device)
        if ctx_lens is None:
            positions = row
        else:  # the block's tokens follow their own sequence's context
            ctx_lens = ctx_lens.to(device=x.device)
            positions = torch.where(row < n_ctx, row, row - n_ctx + ctx_lens.clamp(0, n_ctx)[:, None])
        q, k, v = self._project(x, positions)
        if _kernels.window_attention_supported(q):
            y = _kernels.window_attention(q, k.to(q.dtype), v.to(q.dtype), n_ctx, window=self.window, sinks=self.sinks,
                                          ctx_lens=ctx_lens)
        else:
            lens = torch.full((b,), n_ctx, device=x.device) if ctx_lens is None else ctx_lens.clamp(0, n_ctx)
            tokens = torch.where((row < n_ctx) & (row >= lens[:, None]), -1, positions.expand(b, s))
            y = _window_plain(q, k, v, tokens, tokens, lens, self.window, self.sinks)
        return self.out_proj(y.reshape(b, s, self.d_model))

    def forward_cached(self, x: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, positions: torch.Tensor,
                       rows: torch.Tensor, ctx_lens: torch.Tensor, n_block: int) -> torch.Tensor:
        """The last x.shape[1] tokens of every sequence against its cache (see
        DraftCache): writes their keys and values to ``rows`` [B, Tq] of the
        cache, then attends. positions [B, Tq]: their places in the sequence;
        ctx_lens [B]: context tokens including the new ones."""
        b, s, _ = x.shape
        q, k, v = self._project(x, positions)
        at = torch.arange(b, device=x.device)[:, None]
        k_cache[at, rows] = k.to(k_cache.dtype)
        v_cache[at, rows] = v.to(v_cache.dtype)
        size = k_cache.shape[1] - 1  # the last row takes what belongs to no token
        kc, vc = k_cache[:, :size], v_cache[:, :size]
        if _kernels.window_attention_supported(q) and kc.dtype == q.dtype:
            y = _kernels.window_attention_cached(q, kc, vc, ctx_lens, n_block=n_block, window=self.window,
                                                 sinks=self.sinks)
        else:
            place = torch.arange(size, device=x.device)[None]
            tokens = torch.where(place < ctx_lens[:, None] + n_block, place, -1)
            y = _window_plain(q, kc.to(q.dtype), vc.to(q.dtype), positions, tokens, ctx_lens, self.window, self.sinks)
        return self.out_proj(y.reshape(b, s, self.d_model))


def _lens(ctx_lens: torch.Tensor | None) -> dict:
    """ctx_lens as a keyword, where given: a subclass or a replaced layer without
    it still takes whole contexts."""
    return {} if ctx_lens is None else {"ctx_lens": ctx_lens}


class DFlashTransformerLayer(nn.Module):
    """Pre-norm block: x + attn(norm(x)), then x + mlp(norm(x)) (reference
    model.py:56-73). ``attention``: DFlashAttention's options."""

    def __init__(self, d_model: int, num_heads: int, d_ffn: int, attention: dict | None = None):
        super().__init__()
        self.norm1 = RMSNorm(d_model)
        self.attn = DFlashAttention(d_model=d_model, num_heads=num_heads, **(attention or {}))
        self.norm2 = RMSNorm(d_model)
        self.mlp = nn.Sequential(nn.Linear(d_model, d_ffn, bias=False), nn.SiLU(),
                                 nn.Linear(d_ffn, d_model, bias=False))

    def forward(self, x: torch.Tensor, attn_mask: torch.Tensor | None = None,
                n_ctx: int | None = None, ctx_lens: torch.Tensor | None = None) -> torch.Tensor:
        x = x + self.attn(self.norm1(x), attn_mask=attn_mask, n_ctx=n_ctx, **_lens(ctx_lens))
        return x + self.mlp(self.norm2(x))

    def forward_cached(self, x: torch.Tensor, *cached) -> torch.Tensor:
        x = x + self.attn.forward_cached(self.norm1(x), *cached)
        return x + self.mlp(self.norm2(x))


def _capturing(t: torch.Tensor) -> bool:
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class DraftCache:
    """Keys and values of the context tokens drafted from so far, per layer
    [B, size + 1, kv_heads, head_dim]: sequence b's ``lens[b]`` tokens in rows 0,
    1, ..., the current block's right behind them, overwritten by the next
    tokens; the last row takes what belongs to no token."""

    def __init__(self, layers: int, batch: int, size: int, kv_heads: int, head_dim: int, device, dtype):
        shape = (batch, size + 1, kv_heads, head_dim)
        self.k = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(layers)]
        self.v = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(layers)]
        self.size = size
        self.lens = torch.zeros(batch, device=device, dtype=torch.int32)
        self.longest = 0  # on the host: no sequence is longer, unless
        self.captured = False  # a draft was captured: its replays add tokens without the host

    def reserve(self, tokens: int, block: int, new: torch.Tensor | None = None) -> None:
        """Room for ``tokens`` more per sequence (``new`` [B]: for so many of them)
        and a block, or ValueError (synchronises only when the host's bound does
        not already show it, or no longer holds). A capture is let through: it adds
        nothing by itself, its replays look after themselves."""
        if _capturing(self.lens):
            self.captured = True
            return
        longest = self.longest + tokens
        if self.captured or longest + block > self.size:
            lens = self.lens + (tokens if new is None else new)
            longest = int(lens.max()) if lens.numel() else 0
            if longest + block > self.size:
                raise ValueError(f"the cache holds {self.size} tokens: a sequence of {longest} with the new ones and a "
                                 f"block of {block} do not fit")
        self.longest = longest


class DFlashSpeculator(nn.Module):
    """Block-parallel drafter emitting ``block_size`` draft logits per sequence."""

    def __init__(self, d_target: int, d_model: int, target_vocab_size: int, block_size: int = 4,
                 num_layers: int = 3, num_heads: int = 4,
                 target_lm_head: nn.Linear | None = None, norm_before_head: bool = True,
                 attention: dict | None = None):
        super().__init__()
        self.d_target = d_target
        self.d_model = d_model
        self.block_size = block_size
        self.target_vocab_size = target_vocab_size
        self.proj_in = nn.Linear(d_target, d_model, bias=False)
        self.slot_queries = nn.Parameter(0.02 * torch.randn(1, block_size, d_model))
        self.layers = nn.ModuleList(
            DFlashTransformerLayer(d_model, num_heads, 4 * d_model, attention) for _ in range(num_layers))
        self.norm_out = RMSNorm(d_model)
        self.proj_out = nn.Linear(d_model, d_target, bias=False)
        self.final_norm = RMSNorm(d_target) if norm_before_head else None
        if target_lm_head is not None:
            self.lm_head = target_lm_head
            self.lm_head.weight.requires_grad = False  # the verifier head stays frozen
        else:
            self.lm_head = nn.Linear(d_target, target_vocab_size, bias=False)

    def _build_dflash_mask(self, S_ctx: int, S_block: int, device) -> torch.Tensor:
        """Additive [1, 1, T, T] mask: context rows causal over the context and
        blind to the block; block rows see every token."""
        T = S_ctx + S_block
        row = torch.arange(T, device=device).view(T, 1)
        col = torch.arange(T, device=device).view(1, T)
        visible = (row >= S_ctx) | ((col <= row) & (col < S_ctx))
        mask = torch.zeros(T, T, device=device)
        mask.masked_fill_(~visible, float("-inf"))
        return mask.view(1, 1, T, T)

    @staticmethod
    def _check_lens(ctx_lens: torch.Tensor, target_features: torch.Tensor) -> None:
        if ctx_lens.shape != target_features.shape[:1] or ctx_lens.dtype.is_floating_point or ctx_lens.dtype == torch.bool:
            raise AssertionError(f"ctx_lens must be int [batch], got {ctx_lens.dtype} {list(ctx_lens.shape)} for a batch of "
                                 f"{target_features.shape[0]}")

    def _embed(self, target_features: torch.Tensor) -> torch.Tensor:
        return torch.cat([self.proj_in(target_features),
                          self.slot_queries.expand(target_features.shape[0], -1, -1).to(target_features.dtype)], dim=1)

    def _block_logits(self, h: torch.Tensor) -> torch.Tensor:
        feat = self.proj_out(self.norm_out(h)[:, h.shape[1] - self.block_size:, :])
        if self.final_norm is not None:
            feat = self.final_norm(feat)
        return self.lm_head(feat)

    def forward(self, target_features: torch.Tensor, ctx_lens: torch.Tensor | None = None) -> torch.Tensor:
        """target_features [batch, S_ctx, d_target] -> draft logits [batch, block_size, V].
        ctx_lens int [batch]: sequence b's context is its first ctx_lens[b] features; the
        others may hold anything (they enter as zeros: a weight's gradient is a product
        with them too)."""
        s_ctx = target_features.shape[1]
        if ctx_lens is not None:
            self._check_lens(ctx_lens, target_features)
            live = torch.arange(s_ctx, device=target_features.device) < ctx_lens.to(target_features.device)[:, None]
            target_features = torch.where(live[:, :, None], target_features, 0)
        h = self._embed(target_features)
        # the _build_dflash_mask rule, applied by structure (no [T, T] mask tensor)
        for layer in self.layers:
            h = layer(h, n_ctx=s_ctx, **_lens(ctx_lens))
        return self._block_logits(h)

    def compute_loss(self, target_features: torch.Tensor, ground_truth_block_tokens: torch.Tensor,
                     loss_fn=None, ctx_lens: torch.Tensor | None = None) -> torch.Tensor:
        """Training loss over the block slots. ``loss_fn(logits, targets) -> scalar``
        swaps the objective (dpace_loss, dflash_objective(...)); None = plain CE."""
        logits = self.forward(target_features, **_lens(ctx_lens))
        if loss_fn is not None:
            return loss_fn(logits, ground_truth_block_tokens)
        return F.cross_entropy(logits.reshape(-1, self.target_vocab_size),
                               ground_truth_block_tokens.reshape(-1))

    def new_cache(self, batch: int, size: int, device=None, dtype=torch.bfloat16) -> DraftCache:
        """An empty cache for ``draft``: ``size`` tokens per sequence, the block
        among them; dtype: that of the layers' activations (bf16 under autocast)."""
        attn = self.layers[0].attn
        device = self.slot_queries.device if device is None else device
        return DraftCache(len(self.layers), batch, size, attn.num_kv_heads, attn.head_dim, device, dtype)

    @torch.no_grad()
    def draft(self, target_features: torch.Tensor, ctx_lens: torch.Tensor | None = None,
              cache: DraftCache | None = None):
        """Single-pass drafting: (draft_tokens [batch, block], draft_logits).

        With a cache (``new_cache``), target_features are only the features that
        follow those already in it -- the tokens accepted since the last draft --
        and ctx_lens int [batch] says how many of them each sequence has: its
        last ctx_lens[b] rows (None: all). Their keys and values join the cache.
        Without room for them ValueError; in a replayed graph, where the host does
        not look, the sequence keeps what it has and its logits are NaN."""
        if cache is None:
            logits = self.forward(target_features, **_lens(ctx_lens))
            return logits.argmax(dim=-1), logits
        if ctx_lens is not None:
            self._check_lens(ctx_lens, target_features)
        b, n_new, _ = target_features.shape
        if b != cache.lens.shape[0]:
            raise ValueError(f"the cache is for {cache.lens.shape[0]} sequences, got {b}")
        new = torch.full((b,), n_new, device=cache.lens.device, dtype=torch.int32) if ctx_lens is None else \
            ctx_lens.to(device=cache.lens.device).clamp(0, n_new).to(torch.int32)
        cache.reserve(n_new, self.block_size, None if ctx_lens is None else new)
        lens = cache.lens + new
        i = torch.arange(n_new + self.block_size, device=cache.lens.device)
        positions = lens.long()[:, None] + i - n_new
        # a captured draft is replayed without the host's check: what has no room goes to the last row
        fits = lens + self.block_size <= cache.size
        rows = torch.where((i >= n_new - new[:, None]) & fits[:, None], positions, cache.size)
        h = self._embed(target_features)
        for layer, k, v in zip(self.layers, cache.k, cache.v):
            h = layer.forward_cached(h, k, v, positions, rows, lens, self.block_size)
        cache.lens.copy_(torch.where(fits, lens, cache.lens))
        logits = self._block_logits(torch.where(fits[:, None, None], h, float("nan")))
        return logits.argmax(dim=-1), logits
