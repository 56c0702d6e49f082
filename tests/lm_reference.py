"""Plain 64-bit forms of the language-model operators, for the tests."""
import math

import torch


def seen_mask(T, n, window, sinks, device="cpu"):
    i, j = torch.arange(T, device=device)[:, None], torch.arange(T, device=device)[None, :]
    return (i < n) & (j <= i) & ((i - j < window) | (j < sinks))


def attention(q, k, v, window, sinks, lengths=None, scale=None):
    """[B, T, H, D] in float64, differentiable; rows that see nothing are zeros."""
    B, T, H, D = q.shape
    g = H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = []
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        on = seen_mask(T, n, window, sinks, q.device)
        heads = []
        for h in range(H):
            s = scale * (q[b, :, h].double() @ k[b, :, h // g].double().T)
            s = torch.where(on, s, torch.full_like(s, -1e300))
            p = torch.where(on, torch.softmax(s, -1), torch.zeros_like(s))
            # what no row sees is not multiplied: it may hold anything
            vv = torch.where(on.any(0)[:, None], v[b, :, h // g].double(), torch.zeros((), dtype=torch.float64, device=q.device))
            heads.append(p @ vv)
        out.append(torch.stack(heads, 1))
    return torch.stack(out)


def decode(q, k, v, lengths, window, sinks, scale=None):
    B, H, D = q.shape
    g = H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), k.shape[1])
        at = [j for j in range(n) if n - 1 - j < window or j < sinks]
        for h in range(H):
            if at:
                s = scale * (k[b, at, h // g].double() @ q[b, h].double())
                out[b, h] = torch.softmax(s, 0) @ v[b, at, h // g].double()
    return out


def rotate(x, positions, freqs, amplitude, interleaved, inverse=False):
    """x [B, T, H, D]; positions [B, T]; freqs: radians per position (list)."""
    r = 2 * len(freqs)
    f = torch.tensor(freqs, dtype=torch.float64, device=x.device)
    angle = positions.double()[..., None] * f  # [B, T, r/2]
    c, s = (angle.cos() * amplitude)[:, :, None], (angle.sin() * amplitude)[:, :, None]
    if inverse:
        s = -s
    x = x.double()
    y = x.clone()
    ia = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    ib = ia + (1 if interleaved else r // 2)
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def distill(z, ids, t, y, tau, w, reduction="mean"):
    """float64, differentiable in z."""
    N, V = z.shape
    losses, count = [], 0
    for n in range(N):
        if y is not None and not 0 <= int(y[n]) < V:
            losses.append(torch.zeros((), dtype=torch.float64, device=z.device))
            continue
        count += 1
        row = z[n].double()
        ok = [k for k in range(ids.shape[1]) if 0 <= int(ids[n, k]) < V]
        loss = torch.zeros((), dtype=torch.float64, device=z.device)
        if ok and w < 1:
            p = torch.softmax(t[n, ok].double() / tau, 0)
            lq = torch.log_softmax(row / tau, 0)[ids[n, ok].long()]
            keep = p > 0
            loss = loss + (1 - w) * tau * tau * (p[keep] * (p[keep].log() - lq[keep])).sum()
        if w > 0:
            loss = loss - w * torch.log_softmax(row, 0)[int(y[n])]
        losses.append(loss)
    rows = torch.stack(losses) if losses else torch.zeros(0, dtype=torch.float64, device=z.device)
    if reduction == "none":
        return rows
    return rows.sum() / (max(count, 1) if reduction == "mean" else 1)


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def rel(x, want):
    """2-norm of the difference over 2-norm of what is wanted."""
    x, want = x.detach().double(), want.detach().double()
    n = float(want.norm())
    d = float((x - want).norm())
    return d if n == 0.0 else d / n


SQRT = math.sqrt
