"""Attention over packed sequences and paged caches from its definition, in 64 bits on the CPU, one (sequence, head) at a time, and
what the kernels' roundings can add to it."""

import torch

BF16 = 2.0 ** -8          # half a step of bfloat16, relative


def rho(x):
    root = torch.sqrt(1.0 + x * x)
    return torch.where(x >= 0, x + root, 1.0 / (root - x))


def lengths_to_cu(lens, start=0):
    cu = [start]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def attend(q, k, v, sink, first, n, c):
    """q (Lq, D), k, v (Lk, D) float64, token i at position first + i.  Returns (o, spread): spread is
    sum_j p_ij |v_j|, what a relative error of the weights is multiplied by."""
    Lq, D = q.shape
    x = (q @ k.t()) / (D ** 0.5 * c)
    a = n * torch.asinh(x)                                        # rho = exp(asinh)
    a = a.masked_fill(torch.arange(k.shape[0])[None] > first + torch.arange(Lq)[:, None], -float("inf"))
    b = torch.full((Lq, 1), -float("inf"), dtype=torch.float64) if sink is None else (n * torch.asinh(sink.double() / c)).expand(Lq, 1)
    top = torch.cat([a, b], dim=1).amax(dim=1, keepdim=True)
    empty = top == -float("inf")
    top = torch.where(empty, torch.zeros_like(top), top)
    w, ws = torch.exp(a - top), torch.exp(b - top)
    p = torch.where(empty, torch.zeros_like(w), w / (w.sum(1, keepdim=True) + ws))
    seen = (p != 0).any(dim=0)                                    # a key that no token sees may hold anything
    v = torch.where(seen[:, None], v, torch.zeros_like(v))
    return p @ v, p @ v.abs()


def weight_error(q, k, n, c):
    """Relative error of a weight formed in 32 bits: n times that of rho(x), x from a dot product of D terms."""
    D = q.shape[-1]
    size = q.norm(dim=-1).max() * k.norm(dim=-1).max() if k.numel() and q.numel() else torch.zeros(())
    return float(n * (D * 2.0 ** -24 * size / (D ** 0.5 * c) + 2.0 ** -20))


def packed(q, k, v, cu, sink, n, c):
    """(o, spread, weight error), (T, H, D) and a number; rows of no sequence are zero."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    H, Hkv = q.shape[1], k.shape[1]
    o, spread, err = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for h in range(H):
            if b > a:
                g = h // (H // Hkv)
                o[a:b, h], spread[a:b, h] = attend(q[a:b, h], k[a:b, g], v[a:b, g], None if sink is None else sink[h].cpu(), 0, n, c)
                err = max(err, weight_error(q[a:b, h], k[a:b, g], n, c))
    return o, spread, err


def paged(q, k_pages, v_pages, table, lens, cu, sink, n, c):
    q, k_pages, v_pages, table = q.double().cpu(), k_pages.double().cpu(), v_pages.double().cpu(), table.cpu()
    H, (pages, page, Hkv, D) = q.shape[1], k_pages.shape
    o, spread, err = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for s, length in enumerate(lens):
        a, b = (s, s + 1) if cu is None else (int(cu[s]), int(cu[s + 1]))
        at = table[s, : -(-length // page)].long()
        inside = (at >= 0) & (at < pages)
        for g in range(Hkv):
            k, v = (torch.where(inside[:, None, None], t[at.clamp(0, pages - 1), :, g], torch.zeros((), dtype=torch.float64))
                    .reshape(-1, D)[:length] for t in (k_pages, v_pages))
            for h in range(g * H // Hkv, (g + 1) * H // Hkv):
                if b > a:
                    o[a:b, h], spread[a:b, h] = attend(q[a:b, h], k, v, None if sink is None else sink[h].cpu(), length - (b - a), n, c)
                    err = max(err, weight_error(q[a:b, h], k, n, c))
    return o, spread, err


def assert_close(got, o, spread, err, weights=BF16, result=BF16):
    """|got - o| within: the weights' rounding (`weights`) and 32-bit error (`err`) times sum p |v|, the result's own rounding."""
    got = got.detach().double().cpu()
    if got.numel() == 0:
        return
    bound = (weights + 2 * err) * 1.01 * spread + result * 1.01 * (o.abs() + (weights + 2 * err) * spread) + 1e-30
    off = (got - o).abs()
    assert torch.isfinite(got).all(), f"{int((~torch.isfinite(got)).sum())} values are not finite"
    worst = float((off / bound).max())
    assert worst <= 1.0, f"{worst} times the bound, at {torch.nonzero(off / bound == (off / bound).max())[0].tolist()}"


def packed_gradients(q, k, v, d_o, cu, sink, n, c):
    """The formulas of the gradients, one (sequence, head) at a time, with what the kernels' roundings can add to each:
    ((dq, dk, dv, dsink), their bounds).  p and dS are rounded to bf16 ahead of the products, delta comes from an output of 16 bits,
    the rest is 32-bit arithmetic."""
    q, k, v, d_o = (t.double().cpu() for t in (q, k, v, d_o))
    H, Hkv, D = q.shape[1], k.shape[1], q.shape[2]
    out = [torch.zeros_like(t) for t in (q, k, v)] + [torch.zeros(H, dtype=torch.float64)]
    bound = [torch.zeros_like(t) for t in out]
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for h in range(H):
            if b <= a:
                continue
            g = h // (H // Hkv)
            Q, K, V, G = q[a:b, h], k[a:b, g], v[a:b, g], d_o[a:b, h]
            scale = 1.0 / (D ** 0.5 * c)
            x = (Q @ K.t()) * scale
            hidden = torch.arange(b - a)[None] > torch.arange(b - a)[:, None]
            logw = (n * torch.asinh(x)).masked_fill(hidden, -float("inf"))
            z = torch.tensor(-float("inf"), dtype=torch.float64) if sink is None else sink[h].double().cpu() / c
            logs = n * torch.asinh(z) if sink is not None else z
            top = torch.maximum(logw.amax(1, keepdim=True), logs)
            w, ws = torch.exp(logw - top), torch.exp(logs - top)
            total = w.sum(1, keepdim=True) + ws
            p, ps = w / total, ws / total
            o, spread = p @ V, p @ V.abs()
            dP, delta = G @ V.t(), (G * o).sum(1, keepdim=True)
            f = n * scale / torch.sqrt(1 + x * x)
            dS = f * p * (dP - delta)
            out[0][a:b, h] += dS @ K
            out[1][a:b, g] += dS.t() @ Q
            out[2][a:b, g] += p.t() @ G
            err = weight_error(Q, K, n, c)
            e_delta = (G.abs() * (2.0 ** -15 + 4 * err) * spread).sum(1, keepdim=True) + D * 2.0 ** -23 * G.norm(dim=1, keepdim=True) * V.norm(dim=1).max()
            eS = f * p * ((BF16 + 2 * err) * (dP - delta).abs() + 1.01 * e_delta)
            bound[0][a:b, h] += eS @ K.abs()
            bound[1][a:b, g] += eS.t() @ Q.abs()
            bound[2][a:b, g] += (BF16 + 2 * err) * (p.t() @ G.abs())
            if sink is not None:
                slope = n / c / torch.sqrt(1 + z * z)
                out[3][h] -= slope * (ps * delta).sum()
                bound[3][h] += slope * (ps * (e_delta + 2 * err * delta.abs())).sum()
    for i in range(3):
        bound[i] = 1.05 * bound[i] + BF16 * (out[i].abs() + bound[i]) + 1e-30
    bound[3] = 1.05 * bound[3] + 2.0 ** -20 * out[3].abs() + 1e-30
    return out, bound
