"""Measured cases of the drafter's long-context attention layer: rotary
positions, the norms of queries and keys with the rotation, and attention
with a sliding window and sinks, over a training batch and from a cache.

``run`` with ``own`` false computes each operator in elementary torch
operations in fp32 (angles in fp64), rounded once at the end; with ``own`` true
it makes the calls a user makes of specdec.drafter. ``exact`` computes the same
outputs from the definitions in fp64.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _drafter():
    loaded = sys.modules.get("specdec.drafter")
    if loaded is not None:
        return loaded
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-spec-decode_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from specdec import drafter

    return drafter


# ---- the cases ----------------------------------------------------------------

def listed():
    return [
        # the 16 slot queries of one draft, 4 heads of 64: the smallest call of the rotation
        _rotary("rotary slots", B=1, T=16, H=4, D=64, R=64, dtype="bf16"),
        # fp32 training activations, rotary on half of the head, neighbouring pairs, positions far along, odd length
        _rotary("rotary fp32 far", B=2, T=8191, H=16, D=128, R=64, dtype="fp32", interleaved=True, start=1000003, train=True),
        # one new token of each of 32 sequences, grouped heads
        _norm("norm token", B=32, T=1, Hq=32, Hk=8, D=128, R=128, dtype="bf16", start=4095),
        # the drafter's training batch: 512 context tokens and 16 slots, 4 heads of 64
        _norm("norm drafter", B=32, T=528, Hq=4, Hk=4, D=64, R=64, dtype="bf16", train=True),
        # a long context, q and k as views of one fused projection, positions interpolated by 4
        _norm("norm long", B=1, T=32768, Hq=32, Hk=8, D=128, R=128, dtype="bf16", fused=True, factor=4.0, train=True),
        # the drafter's training batch under a short window
        _window("window drafter", B=32, n_ctx=512, n_block=16, Hq=4, Hk=4, D=64, W=128, S=4, train=True),
        # an odd padded batch with shared heads; one of its sequences is empty
        _window("window ragged", B=5, n_ctx=1221, n_block=7, Hq=6, Hk=2, D=64, W=200, S=1, ragged=True, train=True),
        # long-context training with grouped heads of 128
        _window("window long", B=1, n_ctx=8192, n_block=16, Hq=32, Hk=8, D=128, W=2048, S=4, train=True),
        # a prompt, forward only
        _window("window prompt", B=2, n_ctx=4096, n_block=0, Hq=16, Hk=16, D=128, W=1024, S=16),
        # one token of a short cache: latency
        _cached("cached token", B=1, Tq=1, n_block=0, Hq=4, Hk=4, D=64, size=1024, W=1024, S=4),
        # one token of each of 16 sequences in a long cache, most of it visible
        _cached("cached long", B=16, Tq=1, n_block=0, Hq=32, Hk=8, D=128, size=32768, W=24576, S=4),
        # a draft step: 4 accepted tokens join the context, 16 slots see it
        _cached("cached draft", B=8, Tq=20, n_block=16, Hq=32, Hk=8, D=128, size=16384, W=4096, S=4),
    ]


def _rotary(name, B, T, H, D, R, dtype, interleaved=False, start=0, factor=1.0, scale=1.0, train=False):
    c = {"op": "rotary", "B": B, "T": T, "H": H, "D": D, "R": R, "dtype": dtype, "interleaved": interleaved, "start": start,
         "factor": factor, "scale": scale, "train": train}
    return {"name": name, **c} if name else c


def _norm(name, B, T, Hq, Hk, D, R, dtype, interleaved=False, start=0, factor=1.0, scale=1.0, fused=False, train=False):
    c = {"op": "norm", "B": B, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "R": R, "dtype": dtype, "interleaved": interleaved,
         "start": start, "factor": factor, "scale": scale, "fused": fused, "train": train}
    return {"name": name, **c} if name else c


def _window(name, B, n_ctx, n_block, Hq, Hk, D, W, S, ragged=False, train=False):
    c = {"op": "window", "B": B, "n_ctx": n_ctx, "n_block": n_block, "Hq": Hq, "Hk": Hk, "D": D, "W": W, "S": S,
         "ragged": ragged, "train": train}
    return {"name": name, **c} if name else c


def _cached(name, B, Tq, n_block, Hq, Hk, D, size, W, S):
    c = {"op": "cached", "B": B, "Tq": Tq, "n_block": n_block, "Hq": Hq, "Hk": Hk, "D": D, "size": size, "W": W, "S": S}
    return {"name": name, **c} if name else c


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "window", "cached"])
    D = rng.choice([64, 128])
    Hk = rng.choice([1, 2, 3, 4, 8])
    G = rng.choice([1, 1, 2, 3, 4])
    if op in ("rotary", "norm"):
        B = _spread(rng, 1, 32)
        T = _spread(rng, 1, max(1, 40_000_000 // (B * Hk * (G + 1) * D)))
        T = min(T, 32768)
        R = rng.choice([D, D, D // 2])
        more = {"dtype": rng.choice(["bf16", "bf16", "fp32"]), "interleaved": rng.random() < 0.4, "start": _spread(rng, 1, 1 << 20),
                "factor": rng.choice([1.0, 2.0, 8.0]), "scale": rng.choice([1.0, 1.1]), "train": rng.random() < 0.6}
        if op == "rotary":
            return _rotary(None, B, T, Hk * G, D, R, **more)
        return _norm(None, B, T, Hk * G, Hk, D, R, fused=rng.random() < 0.5, **more)
    if op == "window":
        n_ctx = _spread(rng, 1, 4096)
        n_block = rng.choice([0, 1, 4, 16])
        B = _spread(rng, 1, max(1, min(32, 300_000_000 // ((n_ctx + n_block) ** 2 * Hk * G))))
        return _window(None, B, n_ctx, n_block, Hk * G, Hk, D, _spread(rng, 16, 4096), rng.choice([0, 1, 4, 16]),
                       ragged=rng.random() < 0.4, train=rng.random() < 0.6)
    size = _spread(rng, 128, 32768)
    n_block = rng.choice([0, 0, 4, 16])
    Tq = n_block + rng.choice([1, 1, 4])
    B = _spread(rng, 1, max(1, min(32, 400_000_000 // (size * Hk * D))))
    return _cached(None, B, Tq, n_block, Hk * G, Hk, D, size, _spread(rng, 16, 32768), rng.choice([0, 1, 4, 16]))


# ---- inputs -------------------------------------------------------------------

def _frequencies(c):
    i = torch.arange(0, c["R"], 2, dtype=torch.float64, device="cuda")
    return 10000.0 ** (-i / c["R"]) / c["factor"]


def _positions(c):
    """Consecutive positions; each sequence begins at a place of its own."""
    t = torch.arange(c["T"], device="cuda", dtype=torch.int64)
    return c["start"] + 7 * torch.arange(c["B"], device="cuda", dtype=torch.int64)[:, None] + t[None]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)

    if c["op"] in ("rotary", "norm"):
        dt = _DTYPES[c["dtype"]]
        c["positions"], c["inv_freq"] = _positions(c), _frequencies(c)
        B, T, D = c["B"], c["T"], c["D"]
        if c["op"] == "rotary":
            c["x"] = rand(B, T, c["H"], D, dtype=dt)
            if c["train"]:
                c["x"].requires_grad_(True)
                c["dy"] = rand(B, T, c["H"], D, dtype=dt)
            return c
        Hq, Hk = c["Hq"], c["Hk"]
        if c["fused"]:  # q, k and v of one projection
            qkv = rand(B, T, (Hq + 2 * Hk) * D, dtype=dt)
            c["q"] = qkv[..., :Hq * D].unflatten(-1, (Hq, D))
            c["k"] = qkv[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
        else:
            c["q"], c["k"] = rand(B, T, Hq, D, dtype=dt), rand(B, T, Hk, D, dtype=dt)
        c["wq"], c["wk"] = (1.0 + 0.2 * rand(D, dtype=torch.float32) for _ in range(2))
        if c["train"]:
            for n in ("q", "k", "wq", "wk"):
                c[n].requires_grad_(True)
            c["dq"], c["dk"] = rand(B, T, Hq, D, dtype=dt), rand(B, T, Hk, D, dtype=dt)
        return c
    B, Hq, Hk, D = c["B"], c["Hq"], c["Hk"], c["D"]
    if c["op"] == "window":
        T = c["n_ctx"] + c["n_block"]
        c["q"], c["k"], c["v"] = rand(B, T, Hq, D), rand(B, T, Hk, D), rand(B, T, Hk, D)
        c["lens"] = None
        if c["ragged"]:
            c["lens"] = torch.randint(1, c["n_ctx"] + 1, (B,), device="cuda", dtype=torch.int32, generator=g)
            c["lens"][0] = 0
            c["lens"][-1] = c["n_ctx"]
        if c["train"]:
            for n in ("q", "k", "v"):
                c[n].requires_grad_(True)
            c["do"] = rand(B, T, Hq, D)
        return c
    size, n_block = c["size"], c["n_block"]
    c["q"] = rand(B, c["Tq"], Hq, D)
    c["k"], c["v"] = rand(B, size, Hk, D), rand(B, size, Hk, D)
    # lengths between half of the cache and all of it, the last sequence at its end
    c["lens"] = torch.randint(size // 2, size - n_block + 1, (B,), device="cuda", dtype=torch.int32, generator=g)
    c["lens"][-1] = size - n_block
    return c


# ---- one pass -----------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "window": _plain_window, "cached": _plain_cached}[s["op"]](s)


def _run_own(s):
    drafter = _drafter()
    if s["op"] == "rotary":
        y = drafter.rotary(s["x"], s["positions"], s["inv_freq"], interleaved=s["interleaved"], scale=s["scale"])
        if not s["train"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    if s["op"] == "norm":
        q, k = drafter.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["inv_freq"], eps=1e-6,
                                      interleaved=s["interleaved"], scale=s["scale"])
        if not s["train"]:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if s["op"] == "window":
        o = drafter.window_attention(s["q"], s["k"], s["v"], s["n_ctx"], window=s["W"], sinks=s["S"], ctx_lens=s["lens"])
        if not s["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    return {"o": drafter.window_attention_cached(s["q"], s["k"], s["v"], s["lens"], n_block=s["n_block"], window=s["W"],
                                                 sinks=s["S"])}


def _angles(s):
    a = s["positions"].double()[..., None] * s["inv_freq"]  # [B, T, R / 2]
    return a.cos().float()[:, :, None], a.sin().float()[:, :, None]


def _turn(x, cos, sin, s):
    """The first R elements of fp32 x turned by the angles, the rest as they are."""
    R = s["R"]
    a, b = (x[..., :R:2], x[..., 1:R:2]) if s["interleaved"] else (x[..., :R // 2], x[..., R // 2:R])
    u, v = (a * cos - b * sin) * s["scale"], (b * cos + a * sin) * s["scale"]
    turned = torch.stack((u, v), -1).flatten(-2) if s["interleaved"] else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _plain_rotary(s):
    with torch.no_grad():
        cos, sin = _angles(s)
        y = _turn(s["x"].float(), cos, sin, s).to(s["x"].dtype)
        if not s["train"]:
            return {"y": y}
        return {"y": y, "dx": _turn(s["dy"].float(), cos, -sin, s).to(s["x"].dtype)}


def _plain_norm(s):
    with torch.no_grad():
        cos, sin = _angles(s)
        out = {}
        for n, w in (("q", "wq"), ("k", "wk")):
            x = s[n].float()
            r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            out[n] = _turn(x * r * s[w], cos, sin, s).to(s[n].dtype)
            if s["train"]:
                dn = _turn(s["d" + n].float(), cos, -sin, s)
                g = dn * s[w]
                out["d" + n] = (r * g - x * r ** 3 * (g * x).mean(-1, keepdim=True)).to(s[n].dtype)
                out["d" + w] = (dn * x * r).double().sum((0, 1, 2)).float()
        return out


def _heads(t, G=1):
    """[B, T, H, D] -> fp32 [B, H G, T, D], each head G times."""
    t = t.float().transpose(1, 2)
    return t if G == 1 else t.repeat_interleave(G, 1)


def _visible_window(s):
    """[B, 1, T, T]: query row, key row."""
    n, W, S = s["n_ctx"], s["W"], s["S"]
    T = n + s["n_block"]
    c = s["lens"].long() if s["lens"] is not None else torch.full((s["B"],), n, device="cuda")
    c = c[:, None, None]
    row = torch.arange(T, device="cuda")[None, :, None]
    key = torch.arange(T, device="cuda")[None, None]
    context = (row < c) & (key <= row) & ((row - key < W) | (key < S))
    slot = (row >= n) & ((key >= n) | ((key < c) & ((c - key <= W) | (key < S))))
    return (context | slot)[:, None]


def _softmax(q, k, seen):
    """The weights over what is seen, zero where nothing is."""
    p = q @ k.transpose(-1, -2)
    p *= 1.0 / math.sqrt(q.shape[-1])
    p.masked_fill_(~seen, -math.inf)
    p -= p.amax(-1, keepdim=True).clamp_min(-1e30)
    p.exp_()
    p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
    return p


def _plain_window(s):
    with torch.no_grad():
        G, dt = s["Hq"] // s["Hk"], s["q"].dtype
        q, k, v = _heads(s["q"]), _heads(s["k"], G), _heads(s["v"], G)
        p = _softmax(q, k, _visible_window(s))
        o = p @ v
        out = {"o": o.transpose(1, 2).contiguous().to(dt)}
        if not s["train"]:
            return out
        do = _heads(s["do"])
        dv = p.transpose(-1, -2) @ do
        ds = do @ v.transpose(-1, -2)
        ds -= (do * o).sum(-1, keepdim=True)
        ds *= p
        ds *= 1.0 / math.sqrt(s["D"])
        dq = ds @ k
        dk = ds.transpose(-1, -2) @ q
        out["dq"] = dq.transpose(1, 2).contiguous().to(dt)
        for n, t in (("dk", dk), ("dv", dv)):
            out[n] = t.unflatten(1, (s["Hk"], G)).sum(2).transpose(1, 2).contiguous().to(dt)
        return out


def _plain_cached(s):
    with torch.no_grad():
        G, Tq, nb, W, S = s["Hq"] // s["Hk"], s["Tq"], s["n_block"], s["W"], s["S"]
        c = s["lens"].long()[:, None, None]
        p = c + nb - Tq + torch.arange(Tq, device="cuda")[None, :, None]
        key = torch.arange(s["size"], device="cuda")[None, None]
        context = (p < c) & (key <= p) & ((p - key < W) | (key < S))
        slot = (p >= c) & (key < c + nb) & ((key >= c) | (c - key <= W) | (key < S))
        # the queries of a group are rows of one product with its shared head
        q = s["q"].float().unflatten(2, (s["Hk"], G)).permute(0, 2, 3, 1, 4).flatten(2, 3)
        w = _softmax(q, _heads(s["k"]), (context | slot)[:, None].repeat(1, 1, G, 1))
        o = (w @ _heads(s["v"])).unflatten(2, (G, Tq))
        return {"o": o.permute(0, 3, 1, 2, 4).flatten(2, 3).contiguous().to(s["q"].dtype)}


# ---- the definition in fp64 ----------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return _exact_rotation(s) if s["op"] in ("rotary", "norm") else _exact_attention(s)


def _rotate64(x, s, way):
    """Each pair as a complex number times e^(i way angle) and the factor."""
    R = s["R"]
    x = x.double()
    z = x[..., :R].unflatten(-1, (R // 2, 2)) if s["interleaved"] else x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
    turn = torch.polar(torch.full((1,), float(s["scale"]), dtype=torch.float64, device="cuda"),
                       way * (s["positions"].double()[:, :, None, None] * s["inv_freq"]))
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., R:]), -1)


def _exact_rotation(s):
    if s["op"] == "rotary":
        out = {"y": _rotate64(s["x"], s, 1.0)}
        return {**out, "dx": _rotate64(s["dy"], s, -1.0)} if s["train"] else out
    out, grads, sums = {}, {}, {}
    for n in ("q", "k"):
        x, w = s[n].double(), s["w" + n].double()
        size = torch.sqrt((x * x).sum(-1, keepdim=True) / s["D"] + 1e-6)
        unit = x / size
        out[n] = _rotate64(unit * w, s, 1.0)
        if s["train"]:
            back = _rotate64(s["d" + n], s, -1.0)
            sums["dw" + n] = (back * unit).sum((0, 1, 2))
            back = back * w
            grads["d" + n] = (back - unit * (back * unit).sum(-1, keepdim=True) / s["D"]) / size
    return {**out, **grads, **sums}


def _exact_attention(s):
    """Sequence by sequence, its tokens alone in their order (the context, then
    the block), a stretch of queries at a time against the keys they can see."""
    B, Hk, D, W, S, nb = s["B"], s["Hk"], s["D"], s["W"], s["S"], s["n_block"]
    G, train = s["Hq"] // Hk, s.get("train", False)
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") if train else None for n in ("q", "k", "v"))
    lens = s["lens"].tolist() if s["lens"] is not None else [s["n_ctx"]] * B
    for b, c in enumerate(lens):
        total = c + nb
        if s["op"] == "window":
            rows = torch.cat((torch.arange(c), torch.arange(s["n_ctx"], s["n_ctx"] + nb))).cuda()  # token -> row
            q_rows, first = rows, 0
        else:
            rows = torch.arange(total).cuda()
            q_rows, first = torch.arange(s["Tq"]).cuda(), total - s["Tq"]
        step = max(1, 2 ** 27 // max(1, total * Hk * G))
        for at in range(0, len(q_rows), step):
            mine = q_rows[at:at + step]
            tok = first + at + torch.arange(len(mine)).cuda()
            low = 0 if S else max(0, min(first + at, c) - W)
            keys = torch.arange(low, total).cuda()
            t, j = tok[:, None], keys[None]
            hidden = torch.where(t < c, (j > t) | ((t - j >= W) & (j >= S)), (j < c) & (c - j > W) & (j >= S)) | (t < 0)
            q = s["q"][b, mine].double().view(len(mine), Hk, G, D).permute(1, 2, 0, 3)
            k = s["k"][b, rows[low:]].double().permute(1, 0, 2)[:, None]
            v = s["v"][b, rows[low:]].double().permute(1, 0, 2)[:, None]
            x = torch.matmul(q, k.mT) / math.sqrt(D)
            x = x.masked_fill(hidden, -math.inf)
            p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)).masked_fill(hidden, 0.0)
            y = torch.matmul(p, v)
            o[b, mine] = y.permute(2, 0, 1, 3).reshape(len(mine), Hk * G, D)
            if train:
                do = s["do"][b, mine].double().view(len(mine), Hk, G, D).permute(1, 2, 0, 3)
                dv[b, rows[low:]] += torch.matmul(p.mT, do).sum(1).permute(1, 0, 2)
                dx = p * (torch.matmul(do, v.mT) - (y * do).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[b, mine] = torch.matmul(dx, k).permute(2, 0, 1, 3).reshape(len(mine), Hk * G, D)
                dk[b, rows[low:]] += torch.matmul(dx.mT, q).sum(1).permute(1, 0, 2)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if train else {"o": o}


# ---- what a pass cannot do without ----------------------------------------------

def work(c):
    B, D = c["B"], c["D"]
    if c["op"] in ("rotary", "norm"):
        H = c["H"] if c["op"] == "rotary" else c["Hq"] + c["Hk"]
        n = B * c["T"] * H * D
        size = 4 if c["dtype"] == "fp32" else 2
        # x and y; in training dy and dx too, x stays in hand where the norm needs it again
        moved = (4 if c["train"] else 2) * n * size + 8 * B * c["T"]
        each = (3 if c["op"] == "rotary" else 7) * (3 if c["train"] else 1)
        return {"bytes": moved, "flops": each * n}
    Hq, Hk, W, S = c["Hq"], c["Hk"], c["W"], c["S"]
    if c["op"] == "window":
        n, nb = c["n_ctx"], c["n_block"]
        T = n + nb
        lens = [n] * B
        if c["ragged"] and B > 1:
            lens = [0] + [(n + 1) // 2] * (B - 2) + [n]  # the mean length
        pairs = sum(sum(min(t + 1, W + max(0, min(S, t + 1 - W))) for t in range(n_b)) + nb * (nb + min(n_b, W + max(0, min(S, n_b - W))))
                    for n_b in lens)
        tokens = sum(lens) + B * nb  # padding is never read; its outputs are zeros
        moved = 2 * D * (tokens * (Hq + 2 * Hk) + B * T * Hq)  # q, k, v; o
        if c["train"]:
            moved += 2 * D * (tokens * Hq + B * T * (Hq + 2 * Hk))  # do; dq, dk, dv
        return {"bytes": moved, "flops": pairs * Hq * D * (14 if c["train"] else 4)}
    size, nb, Tq = c["size"], c["n_block"], c["Tq"]
    mean = 0.75 * size
    seen = min(mean, W + S) + nb
    return {"bytes": 2 * B * D * (2 * Hq * Tq + 2 * Hk * seen), "flops": 4 * B * Hq * Tq * D * seen}
