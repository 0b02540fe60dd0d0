"""The drafter's long-context attention layer as a user runs it: rotary
positions, norms of queries and keys, shared key heads, a sliding window with
sinks, padded batches and drafting from a cache -- in plain torch on the CPU,
and on the GPU with the kernels.

CPU (fp32): two ways to the same numbers differ by the order of their sums,
below 1e-5 of logits of size about 1 through two layers. GPU (bf16 activations):
every activation is rounded to 8 bits, 2^-8 of its size, in a few dozen places
on the way to the logits; as in the other drafter tests, logits agree to 5e-2 of
the largest and gradients to 5e-2 in norm.
"""
import pytest
import torch
import torch.nn as nn

from models.dflash import DFlashAttention, DFlashSpeculator, DraftCache
from models.dflash.model import _rotate_plain, _window_plain

OPTIONS = [
    dict(rotary={}),
    dict(window=5, sinks=2),
    dict(num_kv_heads=2, qk_norm=True, rotary=dict(interleaved=True, scaling="yarn", factor=4.0, original_length=16), window=7),
    dict(num_kv_heads=1, rotary=dict(dim=8, base=500.0), sinks=1, window=3),
]


def _model(options, seed=0, d_model=64, heads=4, d_target=48, V=50, block=4, layers=2):
    torch.manual_seed(seed)
    m = DFlashSpeculator(d_target=d_target, d_model=d_model, target_vocab_size=V, block_size=block, num_layers=layers,
                         num_heads=heads, attention=options)
    for p in m.parameters():  # norms' weights away from one
        if p.dim() == 1:
            p.data += 0.2 * torch.randn_like(p)
    for n in m.modules():  # the default eps is the activations' type's, which plain torch and the kernels take differently
        if isinstance(n, nn.RMSNorm):
            n.eps = 1e-6
    return m


def test_options_are_off_by_default():
    a, b = _model(None), _model({})
    assert list(a.state_dict()) == list(b.state_dict()) and not a.layers[0].attn.extended
    x = torch.randn(2, 9, 48)
    assert torch.equal(a(x), b(x))
    m = _model(dict(num_kv_heads=2, qk_norm=True))
    names = set(m.state_dict())
    assert names - set(a.state_dict()) == {f"layers.{i}.attn.{n}_norm.weight" for i in range(2) for n in "qk"}
    assert m.layers[0].attn.k_proj.weight.shape == (32, 64)


@pytest.mark.parametrize("options", OPTIONS)
def test_plain_layer_follows_the_definition(options):
    """One layer against loops over queries, heads and keys."""
    torch.manual_seed(1)
    at = DFlashAttention(64, 4, **options)
    b, n, nb = 2, 11, 3
    lens = torch.tensor([11, 6])
    x = torch.randn(b, n + nb, 64)
    got = at(x, n_ctx=n, ctx_lens=lens)
    want = torch.zeros(b, n + nb, 64)
    W, S = options.get("window") or 10 ** 9, options.get("sinks", 0)
    for i in range(b):
        c = int(lens[i])
        rows = list(range(c)) + list(range(n, n + nb))  # the sequence's tokens in order
        q, k, v = at._project(x[i:i + 1, rows], torch.arange(c + nb))
        for p in range(c + nb):
            seen = [j for j in range(c + nb) if (j <= p and (p - j < W or j < S) if p < c else j >= c or c - j <= W or j < S)]
            for h in range(4):
                kh = h // (4 // at.num_kv_heads)
                w = torch.softmax(torch.stack([q[0, p, h] @ k[0, j, kh] for j in seen]) * at.head_dim ** -0.5, 0)
                y = sum(w[a] * v[0, j, kh] for a, j in enumerate(seen))
                want[i, rows[p], h * 16:(h + 1) * 16] = y
    want = at.out_proj(want)
    live = torch.arange(n + nb) >= n
    for i in range(b):
        rows = live | (torch.arange(n + nb) < lens[i])
        assert float((got[i, rows] - want[i, rows]).abs().max()) < 1e-5


@pytest.mark.parametrize("options", OPTIONS)
def test_a_padded_batch_equals_its_sequences_alone(options):
    m = _model(options)
    x = torch.randn(3, 20, 48)
    lens = torch.tensor([20, 7, 1])
    padded = x.clone()
    for i, c in enumerate(lens.tolist()):
        padded[i, c:] = float("nan")
    got = m(padded, ctx_lens=lens)
    for i, c in enumerate(lens.tolist()):
        assert float((got[i] - m(x[i:i + 1, :c])[0]).abs().max()) < 1e-5
    empty = m(torch.full((1, 5, 48), float("nan")), ctx_lens=torch.tensor([0]))
    assert bool(torch.isfinite(empty).all())
    loss = m.compute_loss(padded, torch.randint(0, 50, (3, 4)), ctx_lens=lens)
    assert bool(torch.isfinite(loss))


def _draft_in_steps(m, x, steps, cache):
    """Feeds x's features in ragged steps (steps: list of per-sequence counts),
    right-aligned with NaN in front; returns the last (tokens, logits)."""
    done = torch.zeros(x.shape[0], dtype=torch.int64)
    for counts in steps:
        width = max(counts)
        feats = torch.full((x.shape[0], width, x.shape[2]), float("nan"), device=x.device)
        for i, c in enumerate(counts):
            if c:
                feats[i, width - c:] = x[i, done[i]:done[i] + c]
        done += torch.tensor(counts)
        out = m.draft(feats, ctx_lens=torch.tensor(counts), cache=cache)
    return out, done


@pytest.mark.parametrize("options", OPTIONS + [None])
def test_drafting_from_a_cache_equals_the_whole_context(options):
    m = _model(options)
    x = torch.randn(3, 30, 48)
    cache = m.new_cache(3, 40, dtype=torch.float32)
    steps = [(5, 0, 3), (1, 4, 2), (3, 2, 0), (9, 1, 4)]
    (tok, logits), done = _draft_in_steps(m, x, steps, cache)
    assert cache.lens.tolist() == done.tolist()
    for i, c in enumerate(done.tolist()):
        t, want = m.draft(x[i:i + 1, :c])
        assert float((logits[i] - want[0]).abs().max()) < 1e-5 and torch.equal(tok[i], t[0])
    # no new token: the same block again
    again = m.draft(x[:, :0], cache=cache)[1]
    assert float((again - logits).abs().max()) < 1e-5


def test_cache_is_refused_when_full_or_for_another_batch():
    m = _model(dict(rotary={}))
    cache = m.new_cache(2, 10, dtype=torch.float32)
    x = torch.randn(2, 6, 48)
    with pytest.raises(ValueError):
        m.draft(x[:1], cache=cache)
    m.draft(x, ctx_lens=torch.tensor([1, 2]), cache=cache)  # two tokens at most are there, not six
    m.draft(x[:, :4], cache=cache)
    assert cache.longest == 6
    with pytest.raises(ValueError):
        m.draft(x[:, :1], cache=cache)
    assert isinstance(cache, DraftCache) and cache.lens.tolist() == [5, 6]


def test_a_draft_that_does_not_fit_gives_nan_and_leaves_the_cache():
    """Replays of a captured draft pass by the host's check: a sequence without
    room keeps its tokens and gets NaN, the others go on."""
    m = _model(dict(rotary={}, window=6, sinks=1))
    cache = m.new_cache(2, 12, dtype=torch.float32)
    x = torch.randn(2, 20, 48)
    m.draft(x[:, :7], ctx_lens=torch.tensor([2, 7]), cache=cache)
    kept = [t[1, :7].clone() for t in cache.k + cache.v]
    cache.longest = 0  # as if the host had not seen the steps before
    new = torch.stack([x[0, 2:5], x[1, 7:10]])
    tok, logits = m.draft(new, cache=cache)
    assert cache.lens.tolist() == [5, 7] and bool(torch.isnan(logits[1]).all())
    want = m.draft(torch.cat([x[:1, 5:7], x[:1, 2:5]], 1))[1]  # the last two rows, then three more
    assert float((logits[0] - want[0]).abs().max()) < 1e-5
    for a, t in zip(kept, cache.k + cache.v):
        assert torch.equal(a, t[1, :7])
    again = m.draft(x[:, :0], cache=cache)[1]
    assert float((again[1] - m.draft(x[1:, :7])[1][0]).abs().max()) < 1e-5


def test_option_refusals():
    for bad in (dict(num_kv_heads=3), dict(num_kv_heads=0), dict(window=0), dict(sinks=-1), dict(rotary=dict(dim=18))):
        with pytest.raises(AssertionError):
            DFlashAttention(64, 4, **bad)
    for bad in (dict(rotary=dict(dim=7)), dict(rotary=dict(scaling="none"))):
        with pytest.raises(ValueError):
            DFlashAttention(64, 4, **bad)
    at = DFlashAttention(64, 4, window=3)
    with pytest.raises(AssertionError):
        at(torch.randn(1, 4, 64), attn_mask=torch.zeros(1, 1, 4, 4))


def test_frequencies_survive_a_change_of_dtype():
    m = _model(dict(rotary={})).bfloat16().float()
    f, _ = m.layers[0].attn._frequencies(torch.device("cpu"))
    assert f.dtype == torch.float64 and float(f[1]) == 10000.0 ** (-2.0 / 16)


@pytest.mark.parametrize("options", OPTIONS + [None])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 3.0])
def test_gradients_do_not_depend_on_the_padding(options, fill):
    """Weights' and features' gradients of a padded batch: finite whatever the
    padding holds, those of zero padding, and zero for the padding itself."""
    m = _model(options)
    x = torch.randn(3, 20, 48)
    lens = torch.tensor([20, 7, 0])
    pad = torch.arange(20)[None] >= lens[:, None]
    tokens = torch.randint(0, 50, (3, 4))
    got = []
    for value in (fill, 0.0):
        feats = x.clone()
        feats[pad] = value
        feats.requires_grad_(True)
        m.zero_grad(set_to_none=True)
        loss = m.compute_loss(feats, tokens, ctx_lens=lens)
        loss.backward()
        got.append([loss.detach(), feats.grad] + [p.grad for p in m.parameters() if p.grad is not None])
    assert bool((got[0][1][pad] == 0).all()) and len(got[0]) > 2 + len(m.layers)
    for a, b in zip(*got):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


def test_frequencies_are_never_inference_tensors():
    """A copy that is made while drafting in inference mode is kept: the next
    training step has to be able to save it."""
    m = _model(dict(rotary={}))
    at = m.layers[0].attn
    with torch.inference_mode():
        assert not at._frequencies(torch.device("meta"))[0].is_inference()
        m.draft(torch.randn(1, 5, 48))
        born = DFlashAttention(64, 4, rotary={})
    assert not at._frequencies(torch.device("cpu"))[0].is_inference()
    assert not born._frequencies(torch.device("cpu"))[0].is_inference()


def test_frequencies_follow_the_module():
    """They are there before the first call: one inside a capture could not copy them."""
    at = DFlashAttention(64, 4, rotary={})
    want = at._frequencies(torch.device("cpu"))[0]
    at.to("meta")
    assert torch.device("meta") in at._freq
    with torch.device("meta"):
        born = DFlashAttention(64, 4, rotary={})
    assert torch.device("meta") in born._freq
    back = born.to_empty(device="cpu")._frequencies(torch.device("cpu"))[0]
    assert back.device.type == "cpu" and torch.equal(back, want)


def test_a_cache_counts_the_new_tokens_not_the_width():
    """Five tokens there, one more each in features five wide, a block of four:
    ten of twelve places."""
    m = _model(dict(rotary={}))
    cache = m.new_cache(2, 12, dtype=torch.float32)
    x = torch.randn(2, 9, 48)
    m.draft(x[:, :5], cache=cache)
    wide = torch.cat([torch.full((2, 4, 48), float("nan")), x[:, 5:6]], 1)
    _, logits = m.draft(wide, ctx_lens=torch.tensor([1, 1]), cache=cache)
    assert cache.lens.tolist() == [6, 6] and cache.longest == 6
    assert float((logits - m.draft(x[:, :6])[1]).abs().max()) < 1e-5
    m.draft(x[:, 6:8], ctx_lens=torch.tensor([2, 0]), cache=cache)  # eight and six: full
    with pytest.raises(ValueError):
        m.draft(x[:, :2], ctx_lens=torch.tensor([1, 2]), cache=cache)
    assert cache.lens.tolist() == [8, 6]
    m.draft(x[:, 6:9], ctx_lens=torch.tensor([0, 2], dtype=torch.int64), cache=cache)
    assert cache.lens.tolist() == [8, 8] and cache.longest == 8
    m.draft(x[:, :3], ctx_lens=torch.tensor([-1, -2 ** 33]), cache=cache)  # clamped: none
    assert cache.lens.tolist() == [8, 8]


def test_a_draft_after_replays_is_checked_against_the_real_lengths(monkeypatch):
    """A captured draft's replays add tokens behind the host's back: later eager
    drafts look at the lengths again."""
    from models.dflash import model

    m = _model(dict(rotary={}))
    cache = m.new_cache(2, 12, dtype=torch.float32)
    x = torch.randn(2, 12, 48)
    m.draft(x[:, :1], cache=cache)
    with monkeypatch.context() as patch:
        patch.setattr(model, "_capturing", lambda t: True)  # every call like a replay: it adds, the host does not look
        for i in range(1, 4):
            m.draft(x[:, 2 * i - 1:2 * i + 1], cache=cache)
    assert cache.lens.tolist() == [7, 7]
    with pytest.raises(ValueError):
        m.draft(x[:, :2], cache=cache)
    assert cache.lens.tolist() == [7, 7]
    _, logits = m.draft(x[:, 7:8], cache=cache)
    assert float((logits - m.draft(x[:, :8])[1]).abs().max()) < 1e-5
    with pytest.raises(ValueError):
        m.draft(x[:, 8:9], cache=cache)


def test_subclasses_without_ctx_lens_take_whole_contexts():
    """forward(target_features) and layers called with n_ctx alone, as they were
    before contexts had lengths of their own."""
    class Layer(nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x, attn_mask=None, n_ctx=None):
            return self.inner(x, attn_mask=attn_mask, n_ctx=n_ctx)

    class Attention(DFlashAttention):
        def forward(self, x, attn_mask=None, n_ctx=None):
            return super().forward(x, attn_mask, n_ctx)

    class Speculator(DFlashSpeculator):
        def forward(self, target_features):
            return super().forward(target_features)

    a, b = _model(None), _model(None)
    b.__class__ = Speculator
    for layer in b.layers:
        layer.attn.__class__ = Attention
    b.layers = nn.ModuleList(Layer(layer) for layer in b.layers)
    x, tokens = torch.randn(2, 9, 48), torch.randint(0, 50, (2, 4))
    assert torch.equal(a.compute_loss(x, tokens), b.compute_loss(x, tokens))
    assert torch.equal(a.draft(x)[1], b.draft(x)[1])


def test_ctx_lens_of_another_batch_are_refused():
    """They would be broadcast, one sequence to several."""
    m = _model(dict(rotary={}))
    x, tokens = torch.randn(1, 6, 48), torch.randint(0, 50, (1, 4))
    for bad in (torch.tensor([3, 4, 5]), torch.tensor(3), torch.tensor([[3]]), torch.tensor([3.0]), torch.tensor([True])):
        for call in (lambda: m(x, bad), lambda: m.compute_loss(x, tokens, ctx_lens=bad), lambda: m.draft(x, bad),
                     lambda: m.draft(x, bad, cache=m.new_cache(1, 20, dtype=torch.float32))):
            with pytest.raises(AssertionError):
                call()
    with pytest.raises(AssertionError):
        m(x.expand(3, -1, -1), torch.tensor([3]))


# ---- on the GPU ------------------------------------------------------------------

GPU_OPTIONS = [
    dict(d_model=256, heads=4, options=dict(rotary={}, window=64, sinks=4)),
    dict(d_model=512, heads=4, options=dict(num_kv_heads=2, qk_norm=True, window=48, sinks=1,
                                            rotary=dict(dim=64, interleaved=True, scaling="linear", factor=2.0))),
    dict(d_model=192, heads=3, options=dict(num_kv_heads=1, qk_norm=True)),
]


def _gpu_model(d_model, heads, options):
    return _model(options, d_model=d_model, heads=heads, d_target=256, V=500, block=16).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("case", GPU_OPTIONS)
def test_kernels_against_plain_torch(cuda, case):
    from specdec import drafter

    m = _gpu_model(**case)
    x = torch.randn(3, 150, 256, device="cuda")
    lens = torch.tensor([150, 40, 97], device="cuda")
    tokens = torch.randint(0, 500, (3, 16), device="cuda")

    def run(enabled, lens):
        drafter.set_enabled(enabled)
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits = m(x, lens)
            loss = nn.functional.cross_entropy(logits.float().reshape(-1, 500), tokens.reshape(-1))
        loss.backward()
        return logits.float().detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}

    for some in (None, lens):
        try:
            got, grads = run(True, some)
            want, ref = run(False, some)
        finally:
            drafter.set_enabled(True)
        assert float((got - want).abs().max()) <= 5e-2 * float(want.abs().max())
        assert set(grads) == set(ref)
        for n, g in ref.items():
            assert float((grads[n] - g).norm()) <= 5e-2 * float(g.norm()) + 1e-7, n


@pytest.mark.gpu
@pytest.mark.parametrize("case", GPU_OPTIONS)
def test_drafting_from_a_cache_on_the_gpu(cuda, case):
    m = _gpu_model(**case)
    x = torch.randn(4, 220, 256, device="cuda")
    cache = m.new_cache(4, 260)
    steps = [(150, 90, 1, 0), (3, 1, 4, 2), (1, 1, 1, 1), (16, 0, 5, 12)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        (_, logits), done = _draft_in_steps(m, x, steps, cache)
        for i, c in enumerate(done.tolist()):
            want = m.draft(x[i:i + 1, :c])[1][0].float()
            assert float((logits[i].float() - want).abs().max()) <= 5e-2 * float(want.abs().max())


@pytest.mark.gpu
def test_graphed_training_step(cuda):
    """The whole step with the options, captured and replayed on new inputs,
    against the same steps run eagerly."""
    from losses import dpace_loss
    from specdec.graphs import GraphedStep

    case = GPU_OPTIONS[1]

    def build():
        m = _gpu_model(**case)
        params = [p for p in m.parameters() if p.requires_grad]
        opt = torch.optim.AdamW(params, lr=1e-3, capturable=True)

        def fn(feats, tokens, lens):
            opt.zero_grad(set_to_none=True)
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                loss = m.compute_loss(feats, tokens, loss_fn=lambda a, t: dpace_loss(a.float(), t, 0.5), ctx_lens=lens)
            loss.backward()
            torch.nn.utils.clip_grad_norm_(params, 1.0)
            opt.step()
            return loss
        return m, opt, fn

    (ma, oa, fa), (mb, ob, fb) = build(), build()
    g = torch.Generator(device="cuda").manual_seed(3)
    batches = [(torch.randn(4, 100, 256, device="cuda", generator=g), torch.randint(0, 500, (4, 16), device="cuda", generator=g),
                torch.randint(0, 101, (4,), device="cuda", generator=g)) for _ in range(4)]
    for _ in range(3):
        fa(*batches[0])
    step = GraphedStep(fb, *batches[0], optimizers=(ob,))
    for batch in batches[1:]:
        la, lb = float(fa(*batch)), float(step(*batch))
        assert abs(la - lb) <= 1e-5 * abs(la), (la, lb)
    step.check()
    for (n, a), b in zip(ma.named_parameters(), mb.parameters()):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-6), n


def _layer_pass(seed, D=64, dtype=torch.bfloat16):
    """Inputs of one layer and a function of them: norm + rotation, windowed
    attention, gradients."""
    from specdec import drafter

    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, Hq, Hk = 2, 300, 4, 2
    q, k, v = (torch.randn(B, T, h, D, device="cuda", generator=g).to(dtype).requires_grad_(True) for h in (Hq, Hk, Hk))
    w = [(1 + 0.1 * torch.randn(D, device="cuda", generator=g)).requires_grad_(True) for _ in range(2)]
    do = torch.randn(B, T, Hq, D, device="cuda", generator=g).to(dtype)
    pos = torch.arange(T, device="cuda")
    f, _ = drafter.rotary_frequencies(D, device="cuda")

    def fn():
        qr, kr = drafter.qk_norm_rotary(q, k, *w, pos, f)
        o = drafter.window_attention(drafter.rotary(qr, pos, f), kr, v, 290, window=60, sinks=3)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v, *w), do)]
    return fn


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    fns = [_layer_pass(s) for s in (1, 2)]
    want = [fn() for fn in fns]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in fns]
    for _ in range(5):
        got = []
        for s, fn in zip(streams, fns):
            with torch.cuda.stream(s):
                got.append(fn())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_two_captured_passes_replayed_in_turn(cuda):
    fns = [_layer_pass(s) for s in (3, 4)]
    side = torch.cuda.Stream()
    graphs, outs, want = [], [], []
    with torch.cuda.stream(side):
        for fn in fns:
            want.append([t.clone() for t in fn()])
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(fn())
            graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for x, y in zip(o, w):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_draft_from_the_cache(cuda):
    """One draft step captured and replayed: the cache's lengths are on the
    device, so a replay sees the tokens that earlier replays added."""
    m = _gpu_model(**GPU_OPTIONS[0])
    x = torch.randn(2, 60, 256, device="cuda")
    new = torch.zeros(2, 3, 256, device="cuda")
    side = torch.cuda.Stream()
    with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
        with torch.cuda.stream(side):
            cache, ref = m.new_cache(2, 100), m.new_cache(2, 100)
            m.draft(x[:, :40], cache=cache)
            for _ in range(2):
                m.draft(x[:, :3], cache=m.new_cache(2, 100))  # warm up
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = m.draft(new, cache=cache)[1]
            m.draft(x[:, :40], cache=ref)
            for at in (40, 43, 46):
                new.copy_(x[:, at:at + 3])
                g.replay()
                want = m.draft(x[:, at:at + 3], cache=ref)[1]
                assert torch.equal(out, want)
    assert cache.lens.tolist() == ref.lens.tolist() == [49, 49]
    for _ in range(20):  # room for 11 more: the last replays give NaN and write nothing
        g.replay()
    assert cache.lens.tolist() == [82, 82] and bool(torch.isnan(out).all())


@pytest.mark.gpu
def test_forward_mode_raises(cuda):
    """None of the four has a forward-mode derivative: a tangent on any input, or
    on the gradient that comes back, is refused instead of lost."""
    import torch.autograd.forward_ad as fwAD

    from specdec import drafter

    x = torch.randn(2, 6, 4, 64, device="cuda").bfloat16()
    w, pos = torch.ones(64, device="cuda"), torch.arange(6, device="cuda")
    f, _ = drafter.rotary_frequencies(64, device="cuda")
    lens = torch.full((2,), 6, device="cuda", dtype=torch.int32)
    calls = [
        (lambda x: drafter.rotary(x, pos, f), (x,)),
        (lambda f: drafter.rotary(x, pos, f), (f,)),
        (lambda q, k, a, b: drafter.qk_norm_rotary(q, k, a, b, pos, f, eps=1e-6), (x, x.clone(), w, w.clone())),
        (lambda f: drafter.qk_norm_rotary(x, x, w, w, pos, f, eps=1e-6), (f,)),
        (lambda q, k, v: drafter.window_attention(q, k, v, 6), (x, x.clone(), x.clone())),
        (lambda q, k, v: drafter.window_attention_cached(q, k, v, lens), (x, x.clone(), x.clone())),
    ]
    for fn, args in calls:
        fn(*args)
        for i in range(len(args)):
            for grad in (True, False):
                with fwAD.dual_level(), torch.set_grad_enabled(grad):
                    dual = [fwAD.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
                    with pytest.raises(NotImplementedError):
                        fn(*dual)
    for fn, args in (calls[0], calls[2], calls[4]):
        leaves = [a.clone().requires_grad_(True) for a in args]
        y = fn(*leaves)
        y = y if torch.is_tensor(y) else y[0]
        with fwAD.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
            torch.autograd.grad(y, leaves[0], fwAD.make_dual(torch.ones_like(y), torch.ones_like(y)))
        y = fn(*leaves)
        y = y if torch.is_tensor(y) else y[0]
        assert bool(torch.isfinite(torch.autograd.grad(y, leaves[0], torch.ones_like(y))[0].float()).all())


@pytest.mark.gpu
def test_training_after_a_draft_in_inference_mode(cuda):
    """The frequencies' device copy is the module's, not the first call's; and a
    draft may be captured as the first call."""
    case = GPU_OPTIONS[1]
    m, again = _gpu_model(**case), _gpu_model(**case)
    x, tokens = torch.randn(2, 40, 256, device="cuda"), torch.randint(0, 500, (2, 16), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
        with torch.inference_mode():
            m.draft(x)
        losses = []
        for model in (m, again):
            loss = model.compute_loss(x, tokens)
            loss.backward()
            losses.append(loss.detach())
        assert torch.equal(*losses)
        device = m.layers[0].attn.q_proj.weight.device
        assert all(device in layer.attn._freq for layer in _gpu_model(**case).layers)


@pytest.mark.gpu
def test_an_eager_draft_after_replays(cuda):
    m = _gpu_model(**GPU_OPTIONS[0])
    x = torch.randn(2, 40, 256, device="cuda")
    side = torch.cuda.Stream()
    with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False), torch.cuda.stream(side):
        cache, ref = m.new_cache(2, 30), m.new_cache(2, 30)
        for c in (m.new_cache(2, 30), cache, ref):
            m.draft(x[:, :3], cache=c)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            m.draft(x[:, 3:6], cache=cache)
        assert cache.lens.tolist() == [3, 3] and cache.longest == 3
        for _ in range(3):
            g.replay()
            m.draft(x[:, 3:6], cache=ref)
        with pytest.raises(ValueError):
            m.draft(x[:, :3], cache=cache)
        assert torch.equal(m.draft(x[:, 6:8], cache=cache)[1], m.draft(x[:, 6:8], cache=ref)[1])
        assert cache.lens.tolist() == ref.lens.tolist() == [14, 14]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_modules_norm_has_torchs_default_eps(cuda, dtype):
    """The drafter's norms are made without an eps. Three roundings to the type at
    most lie between the two (torch's x / rms before the weight, both results)."""
    from models.dflash.model import RMSNorm

    g = torch.Generator(device="cuda").manual_seed(1)
    a, b = RMSNorm(256).cuda(), nn.RMSNorm(256).cuda()
    with torch.no_grad():
        b.weight.copy_(a.weight.copy_(1 + 0.2 * torch.randn(256, device="cuda", generator=g)))
    for size in (1.0, 0.05, 3e-4):
        x = (size * torch.randn(5, 7, 256, device="cuda", generator=g)).to(dtype)
        got, want = a(x).double(), b(x).double()
        assert float((got - want).norm() / want.norm()) <= 3 * torch.finfo(dtype).eps / 2 + 1e-5
