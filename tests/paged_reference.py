"""Plain 64-bit forms of the paged operators, with the bounds that the kernels' roundings allow, for the tests."""
import math

import torch


def plan(ctx, new, table, page, max_tokens, max_new, free=None, count=0):
    """The plan of a step on the host, from its description.  Returns a dict of lists; ``table`` (list of lists) and ``free`` are changed."""
    width = len(table[0])
    kept, total = [], 0
    for n in new:
        m = min(max(n, 0), max_new, max_tokens - total)
        kept.append(m)
        total += m
    cu = [0]
    for m in kept:
        cu.append(cu[-1] + m)
    ctx = [min(max(c, 0), width * page) for c in ctx]
    pages = lambda c: min(-(-c // page), width)
    taken = missing = back = 0
    if free is not None:
        stack = free[:count]
        for b, n in enumerate(new):
            if n < 0:
                held = table[b][:pages(ctx[b])]
                held = held[:held.index(-1)] if -1 in held else held  # its pages ran out
                stack += held
                back += len(held)
        for i in range(count, min(len(stack), len(free))):
            free[i] = stack[i]
        for b, n in enumerate(new):
            if n < 0:
                continue
            for col in range(pages(ctx[b]), pages(ctx[b] + kept[b])):
                table[b][col] = stack.pop() if stack else -1
                taken, missing = taken + (table[b][col] >= 0), missing + (table[b][col] < 0)
        count = len(stack)
    positions, slots = [-1] * max_tokens, [-1] * max_tokens
    for b in range(len(ctx)):
        for i in range(kept[b]):
            pos = ctx[b] + i
            positions[cu[b] + i] = pos
            pg = table[b][pos // page] if pos // page < width else -1
            slots[cu[b] + i] = pg * page + pos % page if pg >= 0 else -1
    kv = [0 if n < 0 else c + m for c, n, m in zip(ctx, new, kept)]
    return dict(cu=cu, kv=kv, positions=positions, slots=slots, count=count,
                info=[total, taken, back, missing, sum(max(n, 0) - m for n, m in zip(new, kept))])


def prestep(x, w, positions, rotary, theta, eps):
    """(normed, normed and rotated) of (tokens, heads, d), in 64 bits."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        x = x * w.double()
    half = rotary // 2
    if half == 0:
        return x, x
    freq = torch.tensor([theta ** (-2.0 * i / rotary) for i in range(half)], dtype=torch.float64, device=x.device)
    angle = positions.double()[:, None, None] * freq
    a, b = x[..., :half], x[..., half:rotary]
    return x, torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), x[..., rotary:]], -1)


def attention(q, k_cache, v_cache, table, ctx, new, scale, gate=None):
    """out, lse, the bound on out's error and the one on lse's in 64 bits.  ``table``: list of lists; a page outside the cache is not attended.

    The bound, for outputs o = sum w v of weights w: half a step of the output's type relative to o; half a step of the weights' type
    (the same) relative to sum w |v|; for fp16 weights below their normal range half of 2^-24, on a scale whose sum of weights is
    L >= 1; twice the error of the scores, which is d products and sums in fp32 (d 2^-24 of sum |q| |k| scale, at most) and 2^-21 for the scaling, the
    exponential (2^-22) and the sigmoid and division (2^-22 each).  lse: the scores' error, and 2^-20 for the sum and the logarithm."""
    T, H_q, d = q.shape
    page, H_kv = k_cache.shape[1], k_cache.shape[2]
    rep, n_pages, dev = H_q // H_kv, k_cache.shape[0], q.device
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(T, H_q, d, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    lse = torch.full((T, H_q), -math.inf, dtype=torch.float64, device=dev)
    lse_tol = torch.zeros_like(lse)
    t0 = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        n = max(n, 0)
        kv = c + n
        cols = -(-kv // page)
        pg = torch.tensor(([table[b][i] if i < len(table[b]) else -1 for i in range(cols)] or [-1]), device=dev)
        there = ((pg >= 0) & (pg < n_pages)).repeat_interleave(page)[:kv]
        safe = torch.where((pg >= 0) & (pg < n_pages), pg, torch.zeros_like(pg))
        for h in range(H_kv):
            k = k_cache[safe, :, h].reshape(-1, d)[:kv].double()
            v = v_cache[safe, :, h].reshape(-1, d)[:kv].double()
            k, v = k * there[:, None], torch.where(there[:, None], v, torch.zeros_like(v))
            k = torch.where(there[:, None], k, torch.zeros_like(k))
            for i in range(0, n, 256):
                m = min(256, n - i)
                rows, heads = slice(t0 + i, t0 + i + m), slice(h * rep, (h + 1) * rep)
                x = torch.einsum("mrd,kd->mrk", q[rows, heads].double(), k) * scale
                big = torch.einsum("mrd,kd->mrk", q[rows, heads].double().abs(), k.abs()).amax(-1, keepdim=True) * scale if kv else 0.0
                pos = c + i + torch.arange(m, device=dev)
                seen = (torch.arange(kv, device=dev)[None, :] <= pos[:, None]) & there[None, :]
                x = x.masked_fill(~seen[:, None, :], -math.inf)
                total = torch.logsumexp(x, -1, keepdim=True)
                w = torch.where(torch.isfinite(total), torch.exp(x - total), torch.zeros_like(x))
                o = torch.einsum("mrk,kd->mrd", w, v)
                spread = torch.einsum("mrk,kd->mrd", w, v.abs())
                err = half * o.abs() + (half + 2 * (d * 2.0 ** -24 * big + 2.0 ** -21)) * spread + 2.0 ** -20 * o.abs()
                if q.dtype is torch.float16:
                    top = torch.exp(x.amax(-1, keepdim=True) - total)  # the largest weight is 1 or more on the kernel's scale
                    top = torch.where(torch.isfinite(total), top, torch.zeros_like(top))
                    err = err + 2.0 ** -25 * top * torch.einsum("mk,kd->md", seen.double(), v.abs())[:, None, :] + 2.0 ** -25
                lse_tol[rows, heads] = (d * 2.0 ** -24 * big + 2.0 ** -20 * (1 + torch.nan_to_num(total.abs(), posinf=0.0))).squeeze(-1)
                if gate is not None:
                    s = torch.sigmoid(gate[rows, heads].double())
                    o, err = o * s, err * s + (2.0 ** -25 if q.dtype is torch.float16 else 0.0)
                out[rows, heads], tol[rows, heads], lse[rows, heads] = o, err + 1e-30, total.squeeze(-1)
        t0 += n
    return out, lse, tol, lse_tol
