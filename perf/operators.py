"""What the language-model operators are measured on.

``listed()`` names the cases and ``draw()`` gives more of the same ranges;
``prepare()`` makes a case's inputs on the GPU, ``run()`` makes one pass
through the operator and ``work()`` says what a pass cannot do without.  With
``own`` false ``run()`` computes the operator in elementary torch operations
in 32 bits; with ``own`` true it calls cail_b200.ops.  ``exact()`` computes
the same outputs in 64 bits from the operators' definitions.

Four kinds of case:

* ``attention``  window_attention on [B, T, H, D]; ``step`` adds its backward
* ``decode``     window_attention_decode: one token per sequence and a cache
* ``rotary``     rotary on q and k together; ``step`` adds its backward
* ``distill``    distill_loss and the gradient of the logits
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # GPT-2 medium's heads and context, micro-batch 8: a training step whose layers see a quarter of the context
        dict(name="attention step gpt2", op="attention", step=True, B=8, T=1024, H=16, Hkv=16, D=64, window=256, sinks=4,
             ragged=False, type="bf16"),
        # a long document with shared heads: a training step
        dict(name="attention step long", op="attention", step=True, B=1, T=8192, H=16, Hkv=4, D=128, window=1024, sinks=16,
             ragged=False, type="bf16"),
        # fp32 training, the data-parallel harness' type, on a padded batch of odd length
        dict(name="attention step fp32", op="attention", step=True, B=3, T=333, H=16, Hkv=16, D=64, window=100, sinks=3,
             ragged=True, type="fp32"),
        # prompts of unequal length on their way into a cache, window beyond the context, a head size between powers of two
        dict(name="attention prefill ragged", op="attention", step=False, B=4, T=2047, H=12, Hkv=4, D=80, window=4096, sinks=0,
             ragged=True, type="fp16"),
        # one user, one token: latency
        dict(name="decode one", op="decode", B=1, Tmax=1024, H=16, Hkv=16, D=64, window=256, sinks=4, ragged=False, type="bf16"),
        # a serving batch of unequal lengths over long caches with shared heads: bandwidth
        dict(name="decode batch", op="decode", B=64, Tmax=8192, H=32, Hkv=8, D=128, window=4096, sinks=16, ragged=True,
             type="bf16"),
        # the rotation of one decoded token for each of 8 users: latency
        dict(name="rotary token", op="rotary", step=False, B=8, T=1, H=16, Hkv=16, D=64, part=64, interleaved=False,
             scaling="none", first=777, type="bf16"),
        # the training step's rotation, GPT-2 medium's heads
        dict(name="rotary step gpt2", op="rotary", step=True, B=8, T=1024, H=16, Hkv=16, D=64, part=64, interleaved=False,
             scaling="none", first=0, type="bf16"),
        # a long prompt far from the start, interleaved pairs over half the head, frequencies scaled by parts, odd length
        dict(name="rotary long parts", op="rotary", step=False, B=1, T=32767, H=32, Hkv=8, D=128, part=64, interleaved=True,
             scaling="parts", first=100000, type="fp32"),
        # a few tokens at GPT-2's vocabulary in fp32
        dict(name="distill few", op="distill", N=37, V=50257, K=16, tau=2.0, hard=0.5, left_out=0.0, gone=0.0, seed_grad=1.0,
             type="fp32"),
        # micro-batch 8 x 1024 tokens at GPT-2's vocabulary
        dict(name="distill step gpt2", op="distill", N=8192, V=50257, K=64, tau=2.0, hard=0.5, left_out=0.0, gone=0.0,
             seed_grad=1.0, type="bf16"),
        # a padded batch in fp16 under loss scaling, teacher rows shorter than K, no hard labels in the loss
        dict(name="distill padded fp16", op="distill", N=1023, V=32001, K=20, tau=1.0, hard=0.0, left_out=0.3, gone=0.2,
             seed_grad=65536.0, type="fp16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "attention", "decode", "rotary", "distill"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "attention":
        Hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
        T = _spread(rng, 1, 2048 if kind == "fp32" else 6000)
        B = max(1, min(rng.randint(1, 8), (1 << 29) // (Hkv * group * T * T)))
        return dict(op=op, step=rng.random() < 0.7, B=B, T=T, H=Hkv * group, Hkv=Hkv, D=rng.choice([16, 33, 64, 64, 72, 128, 128]),
                    window=_spread(rng, 1, 2 * T), sinks=rng.choice([0, 1, 4, rng.randint(0, 300)]), ragged=rng.random() < 0.5,
                    type=kind)
    if op == "decode":
        Hkv, group, D = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 4, 8]), rng.choice([16, 64, 64, 80, 128, 128])
        Tmax = _spread(rng, 1, 40000)
        B = max(1, min(_spread(rng, 1, 96), (1 << 28) // (Tmax * Hkv * D)))
        return dict(op=op, B=B, Tmax=Tmax, H=Hkv * group, Hkv=Hkv, D=D, window=_spread(rng, 1, 2 * Tmax),
                    sinks=rng.choice([0, 1, 4, rng.randint(0, 300)]), ragged=rng.random() < 0.6, type=kind)
    if op == "rotary":
        D = rng.choice([16, 64, 64, 80, 128, 128])
        T, Hkv = _spread(rng, 1, 30000), rng.choice([1, 2, 8, 16])
        H = Hkv * rng.choice([1, 1, 2, 4])
        B = max(1, min(_spread(rng, 1, 16), (1 << 25) // (T * H * 128)))
        return dict(op=op, step=rng.random() < 0.5, B=B, T=T, H=H, Hkv=Hkv, D=D, part=rng.choice([D, D, D // 2, D // 4 * 2]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "parts"]),
                    first=rng.choice([0, 1, rng.randint(0, 500000)]), type=kind)
    V = _spread(rng, 200, 150000)
    N = max(1, min(_spread(rng, 1, 8192), (1 << 27) // V))
    return dict(op=op, N=N, V=V, K=_spread(rng, 1, min(128, V)), tau=rng.choice([1.0, 2.0, rng.uniform(0.5, 4.0)]),
                hard=rng.choice([0.0, 0.5, 1.0, rng.uniform(0.1, 0.9)]), left_out=rng.choice([0.0, 0.2]), gone=rng.choice([0.0, 0.3]),
                seed_grad=65536.0 if kind == "fp16" else 1.0, type=kind)


def _lengths(n, longest, ragged):
    """The lengths of a batch: all the longest, or falling evenly to a short one, the last of a batch of four or more empty."""
    if not ragged:
        return [longest] * n
    falling = [max(1, longest - (i * longest) // n) for i in range(n)]
    return falling[:-1] + [0] if n >= 4 else falling


def _pairs(length, window, sinks):
    """How many keys the rows of a sequence see in all."""
    w, s = min(window, length), min(sinks, length)
    inside = w * (w + 1) // 2 + (length - w) * w
    past = max(0, length - w)  # rows that the window has left something out of: row w + r - 1 has left out r keys, of which s stay
    return inside + (past * (past + 1) // 2 if past <= s else s * (s + 1) // 2 + (past - s) * s)


def _scaling(case):
    if case["scaling"] == "none":
        return {}
    more = dict(original=8192) if case["scaling"] == "parts" else {}
    return dict(scaling=case["scaling"], factor=16.0, **more)


def prepare(case, seed):
    c = dict(case)
    t = _TYPES[c["type"]]
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)

    def randn(*shape, dtype=t, by=1.0):
        x = torch.randn(*shape, dtype=dtype, device="cuda", generator=gen)
        return x.mul_(by) if by != 1.0 else x

    s = {"case": c}
    if c["op"] == "attention":
        B, T, H, Hkv, D = (c[k] for k in ("B", "T", "H", "Hkv", "D"))
        s["q"], s["k"], s["v"] = randn(B, T, H, D), randn(B, T, Hkv, D), randn(B, T, Hkv, D)
        s["lengths"] = torch.tensor(_lengths(B, T, True), dtype=torch.int32, device="cuda") if c["ragged"] else None
        if c["step"]:
            s["do"] = randn(B, T, H, D)
            for n in "qkv":
                s[n].requires_grad_()
    elif c["op"] == "decode":
        B, T, H, Hkv, D = (c[k] for k in ("B", "Tmax", "H", "Hkv", "D"))
        s["q"], s["k"], s["v"] = randn(B, H, D), randn(B, T, Hkv, D), randn(B, T, Hkv, D)
        s["lengths"] = torch.tensor(_lengths(B, T, c["ragged"]), dtype=torch.int32, device="cuda")
    elif c["op"] == "rotary":
        B, T, H, Hkv, D = (c[k] for k in ("B", "T", "H", "Hkv", "D"))
        s["q"], s["k"] = randn(B, T, H, D), randn(B, T, Hkv, D)
        s["positions"] = torch.arange(c["first"], c["first"] + T, dtype=torch.int64, device="cuda")
        s["freqs"], s["amplitude"] = _frequencies(c)
        if c["step"]:
            s["dq"], s["dk"] = randn(B, T, H, D), randn(B, T, Hkv, D)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        if own:
            from cail_b200.ops import Rotary
            s["plan"] = Rotary(c["part"], base=10000.0, interleaved=c["interleaved"], device="cuda", **_scaling(c))
    else:
        N, V, K = c["N"], c["V"], c["K"]
        s["z"] = randn(N, V, by=2.0).requires_grad_()
        # a teacher's top entries: distinct ids, one in each K-th part of the vocabulary from a start of the row's own
        cell = V // K
        ids = torch.arange(K, device="cuda") * cell + torch.randint(0, cell, (N, K), device="cuda", generator=gen)
        s["ids"] = (ids + torch.randint(0, V, (N, 1), device="cuda", generator=gen)) % V
        s["t"] = randn(N, K, dtype=torch.float32, by=1.5).add_(8.0).sort(dim=1, descending=True).values
        s["y"] = torch.randint(0, V, (N,), device="cuda", generator=gen)
        if c["gone"]:
            s["ids"] = torch.where(torch.rand(N, K, device="cuda", generator=gen) < c["gone"], -1, s["ids"])
        if c["left_out"]:
            s["y"] = torch.where(torch.rand(N, device="cuda", generator=gen) < c["left_out"], -100, s["y"])
        s["g"] = torch.full((), c["seed_grad"], dtype=torch.float32, device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms


def _seen(T, lengths, window, sinks, device):
    """[B or 1, 1, T, T]: whether row i sees key j."""
    i, j = torch.arange(T, device=device)[:, None], torch.arange(T, device=device)[None, :]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    if lengths is None:
        return seen[None, None]
    return seen[None, None] & (i < lengths.long()[:, None, None])[:, None]


def _plain_attention(s):
    c, q, k, v = s["case"], s["q"].detach(), s["k"].detach(), s["v"].detach()
    B, T, H, D = q.shape
    Hkv, t, scale = k.shape[2], q.dtype, D**-0.5
    # [B, Hkv, g, T, D]: the query heads of a key head side by side
    q32 = q.float().view(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4)
    k32, v32 = (x.float().permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
    seen = _seen(T, s["lengths"], c["window"], c["sinks"], q.device)[:, :, None]
    p = torch.matmul(q32 * scale, k32.transpose(-1, -2)).masked_fill_(~seen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    o = torch.matmul(p, v32)

    def back(x):
        return x.permute(0, 3, 1, 2, 4).reshape(B, T, -1, D).to(t)

    if not c["step"]:
        return back(o)
    do = s["do"].float().view(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    ds = torch.matmul(do, v32.transpose(-1, -2))
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)  # so a row that sees one key has exactly none
    del p
    return back(o), back(torch.matmul(ds, k32)), back(torch.matmul(ds.transpose(-1, -2), q32).sum(2, keepdim=True)), back(dv)


def _plain_decode(s):
    c, q, k, v, n = s["case"], s["q"], s["k"], s["v"], s["lengths"].long()
    B, H, D = q.shape
    Hkv = k.shape[2]
    q32 = q.float().view(B, Hkv, H // Hkv, D) * D**-0.5
    j = torch.arange(k.shape[1], device=q.device)
    seen = (j < n[:, None]) & ((n[:, None] - 1 - j < c["window"]) | (j < c["sinks"]))
    p = torch.matmul(q32, k.float().permute(0, 2, 3, 1)).masked_fill_(~seen[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    return torch.matmul(p, v.float().permute(0, 2, 1, 3)).reshape(B, H, D).to(q.dtype)


def _frequencies(c):
    """The angle by which a pair turns from one position to the next, in 64 bits, and the amplitude."""
    r, how = c["part"], c["scaling"]
    base = 10000.0 * (16.0 ** (r / (r - 2)) if how == "ntk" else 1.0)
    f = torch.tensor([base ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64)
    if how == "linear":
        f = f / 16.0
    if how == "parts":  # kept where a pair turns 32 times or more over the first context, divided where it turns less than once
        w = ((8192.0 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * w + f / 16.0 * (1 - w)
    return f.cuda(), 0.1 * math.log(16.0) + 1.0 if how == "parts" else 1.0


def _plain_turn(x, cos, sin, c):
    r, x32 = c["part"], x.detach().float()
    y = x32.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x32[..., a] * cos - x32[..., b] * sin
    y[..., b] = x32[..., b] * cos + x32[..., a] * sin
    return y.to(x.dtype)


def _plain_rotary(s):
    angle = (s["positions"].double()[:, None] * s["freqs"]).remainder_(2 * math.pi)[:, None, :]
    cos, sin = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()
    out = [_plain_turn(s[n], cos, sin, s["case"]) for n in ("q", "k")]
    if s["case"]["step"]:
        out += [_plain_turn(s[n], cos, -sin, s["case"]) for n in ("dq", "dk")]
    return out


def _plain_distill(s):
    c, z, ids, y = s["case"], s["z"].detach().float(), s["ids"], s["y"]
    tau, hard = c["tau"], c["hard"]
    valid = (ids >= 0) & (ids < c["V"])
    at = ids.clamp(0, c["V"] - 1)
    counts = (y >= 0) & (y < c["V"])
    y0 = y.clamp(0, c["V"] - 1)[:, None]
    t = (s["t"] / tau).masked_fill(~valid, -math.inf)
    log_p = t - t.amax(1, keepdim=True).clamp(min=-3e38)
    log_p = log_p - log_p.exp().sum(1, keepdim=True).clamp(min=1e-30).log()
    p = log_p.exp()
    top = z.amax(1, keepdim=True)
    e = ((z - top) / tau).exp()
    total = e.sum(1, keepdim=True)
    log_q = (z.gather(1, at) - top) / tau - total.log()
    kl = torch.where(valid, p * (log_p - log_q), 0.0).sum(1)
    e1 = (z - top).exp()
    total1 = e1.sum(1, keepdim=True)
    ce = (total1.log() + top - z.gather(1, y0))[:, 0]
    n = counts.sum().clamp(min=1)
    loss = torch.where(counts, (1 - hard) * tau * tau * kl + hard * ce, 0.0).sum() / n
    dz = e.div_(total).mul_(p.sum(1, keepdim=True)).scatter_add_(1, at, -p).mul_((1 - hard) * tau)
    dz.add_(e1.div_(total1).scatter_add_(1, y0, -torch.ones_like(y0, dtype=torch.float32)), alpha=hard)
    dz.mul_(torch.where(counts, s["g"] / n, 0.0)[:, None])
    return loss, dz.to(s["z"].dtype)


# ---------------------------------------------------------------- one pass


def run(s):
    c = s["case"]
    if not own:
        return {"attention": _plain_attention, "decode": _plain_decode, "rotary": _plain_rotary,
                "distill": _plain_distill}[c["op"]](s)
    from cail_b200 import ops

    if c["op"] == "attention":
        o = ops.window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"], lengths=s["lengths"])
        return (o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])) if c["step"] else o
    if c["op"] == "decode":
        return ops.window_attention_decode(s["q"], s["k"], s["v"], s["lengths"], c["window"], c["sinks"])
    if c["op"] == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["plan"], s["positions"])
        if not c["step"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    loss = ops.distill_loss(s["z"], s["ids"], s["t"], s["y"], temperature=c["tau"], hard_weight=c["hard"])
    return (loss.detach(), *torch.autograd.grad(loss, s["z"], s["g"]))


def work(case):
    c, size = case, _BYTES[case["type"]]
    if c["op"] == "attention":
        lengths = _lengths(c["B"], c["T"], c["ragged"])
        pairs = sum(_pairs(n, c["window"], c["sinks"]) for n in lengths) * c["H"]
        # only the rows within the lengths are read; every row of the outputs is written
        read = sum(lengths) * (2 * c["Hkv"] + c["H"] * (2 if c["step"] else 1))
        written = c["B"] * c["T"] * (c["H"] * (2 if c["step"] else 1) + (2 * c["Hkv"] if c["step"] else 0))
        return {"bytes": (read + written) * c["D"] * size, "flops": pairs * c["D"] * (14 if c["step"] else 4)}
    if c["op"] == "decode":
        keys = sum(min(n, c["window"]) + min(c["sinks"], max(0, n - c["window"])) for n in _lengths(c["B"], c["Tmax"], c["ragged"]))
        return {"bytes": (keys * c["Hkv"] * 2 + c["B"] * c["H"] * 2) * c["D"] * size, "flops": 4 * keys * c["H"] * c["D"]}
    if c["op"] == "rotary":
        tokens = c["B"] * c["T"] * (c["H"] + c["Hkv"]) * (2 if c["step"] else 1)
        return {"bytes": 2 * tokens * c["D"] * size + 8 * c["T"], "flops": 3 * tokens * c["part"]}
    n = c["N"] * c["V"]
    # the logits of a row that is left out are not read; its gradient is written
    return {"bytes": (2 - c["left_out"]) * n * size + c["N"] * (12 * c["K"] + 8), "flops": n * (6 if c["tau"] == 1.0 or c["hard"] in (0.0, 1.0) else 10)}


# ---------------------------------------------------------------- the definitions, in 64 bits


def _exact_head(q, k, v, seen):
    """Softmax attention of [T, D] queries against [J, D] keys; a row that sees nothing gives zeros."""
    scores = torch.where(seen, q @ k.T / math.sqrt(q.shape[-1]), torch.tensor(-1e300, dtype=torch.float64, device=q.device))
    return torch.where(seen, torch.softmax(scores, -1), torch.zeros_like(scores)) @ v


def _exact_attention(s):
    c = s["case"]
    q, k, v = (s[n].detach().double().requires_grad_(c["step"]) for n in "qkv")
    group = c["H"] // c["Hkv"]
    lengths = [c["T"]] * c["B"] if s["lengths"] is None else s["lengths"].tolist()
    at = torch.arange(c["T"], device=q.device)
    o = torch.zeros_like(q, requires_grad=False)
    for b in range(c["B"]):
        back = at[:, None] - at[None, :]
        seen = (back >= 0) & ((back < c["window"]) | (at < c["sinks"])[None, :]) & (at < lengths[b])[:, None]
        for h in range(c["H"]):
            one = _exact_head(q[b, :, h], k[b, :, h // group], v[b, :, h // group], seen)
            o[b, :, h] = one.detach()
            if c["step"]:
                one.backward(s["do"][b, :, h].double())
    return (o, q.grad, k.grad, v.grad) if c["step"] else o


def _exact_decode(s):
    c = s["case"]
    group = c["H"] // c["Hkv"]
    o = torch.zeros_like(s["q"], dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        keep = sorted(set(range(min(c["sinks"], n))) | set(range(max(0, n - c["window"]), n)))
        if keep:
            at = torch.tensor(keep, device=o.device)
            k, v = (s[x][b, at].double().repeat_interleave(group, 1) for x in ("k", "v"))
            p = torch.softmax(torch.einsum("hd,jhd->hj", s["q"][b].double(), k) / math.sqrt(c["D"]), -1)
            o[b] = torch.einsum("hj,jhd->hd", p, v)
    return o


def _exact_rotary(s):
    c, r = s["case"], s["case"]["part"]
    angle = s["positions"].double()[:, None] * s["freqs"]
    turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, None, :]

    def turned(x, by):
        x = x.detach().double()
        head, rest = x[..., :r], x[..., r:]
        pairs = head.unflatten(-1, (r // 2, 2)) if c["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat([y, rest], -1)

    out = [turned(s["q"], turn), turned(s["k"], turn)]
    return out + [turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())] if c["step"] else out


def _exact_distill(s):
    c = s["case"]
    counts = (s["y"] >= 0) & (s["y"] < c["V"])
    n, loss = max(1, int(counts.sum())), 0.0
    dz = torch.zeros_like(s["z"], dtype=torch.float64)
    for lo in range(0, c["N"], 1024):  # parts of the rows, for the memory
        part = slice(lo, lo + 1024)
        z = s["z"][part].detach().double().requires_grad_()
        ids, y, rows = s["ids"][part], s["y"][part], counts[part]
        valid = (ids >= 0) & (ids < c["V"])
        p = torch.softmax(torch.where(valid, s["t"][part].double() / c["tau"], -1e300), 1) * valid
        teacher = torch.zeros_like(z, requires_grad=False).scatter_add(1, ids.clamp(0, c["V"] - 1), p)
        soft = torch.special.xlogy(p, p).sum(1) - (teacher * torch.log_softmax(z / c["tau"], 1)).sum(1)
        plain = -torch.log_softmax(z, 1).gather(1, y.clamp(0, c["V"] - 1)[:, None])[:, 0]
        each = ((1 - c["hard"]) * c["tau"] ** 2 * soft + c["hard"] * plain) * rows / n
        dz[part] = torch.autograd.grad(each.sum(), z)[0] * float(s["g"])
        loss = loss + each.detach().sum()
    return loss, dz


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "decode": _exact_decode, "rotary": _exact_rotary,
            "distill": _exact_distill}[case["op"]](s)
