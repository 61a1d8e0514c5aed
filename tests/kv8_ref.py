"""Plain implementations of the batched-serving operators over a paged 8-bit KV cache (tests only): the
plan request by request with a Python list for the free stack, the store in float32 arithmetic step by
step, the attention row by row in float64."""
import math

import numpy as np
import torch

LIMIT = {0: 127.0, 1: 448.0}  # FENCE_KV8_INT8, FENCE_KV8_E4M3


def ceil(a, b):
    return -(-a // b)


def plan(ctx, new, table, free, n_tokens, page, max_pages, n_pages):
    """Everything fence_paged_plan writes, as Python lists; `table` rows and `free` (the live stack) are copied."""
    table = [list(r) for r in table]
    stack = list(free)
    for r, n in enumerate(new):  # the ended requests' pages first
        if n < 0:
            stack += table[r][:ceil(ctx[r], page)]
    avail, before = len(stack), 0
    start, kv, ctx_out, slot, pos, touch = [0], [], [], [], [], []
    handed = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        start.append(start[-1] + max(0, n))
        if n < 0:
            kv.append(0)
            ctx_out.append(0)
            continue
        fits = c + n <= max_pages * page
        need = ceil(c + n, page) - ceil(c, page) if fits else 0
        placed = fits and (need == 0 or before + need <= avail)
        if placed:
            for j in range(need):
                table[r][ceil(c, page) + j] = stack[avail - 1 - before - j]
            handed = before + need if need else handed
        before += need
        kv.append(c + n if placed else 0)
        ctx_out.append(c + n if placed else c)
        for i in range(n):
            if placed:
                p = c + i
                pos.append(p)
                slot.append(table[r][p // page] * page + p % page)
                if i == 0 or p % page == 0:
                    touch.append([table[r][p // page], p % page, start[r] + i, 0])
                touch[-1][3] += 1
            else:
                pos.append(-1)
                slot.append(-1)
    slot += [-1] * (n_tokens - len(slot))
    pos += [-1] * (n_tokens - len(pos))
    return dict(n_free_out=[avail - handed], ctx_out=ctx_out, kv_len=kv, new_start=start, slot=slot, pos=pos, touch=touch,
                block_table=table, stack=stack[:avail - handed])


def values(codes, fmt):
    """uint8 codes -> float64 values (before the scale)."""
    return (codes.view(torch.int8) if fmt == 0 else codes.view(torch.float8_e4m3fn)).double()


def to_codes(x, fmt):
    """float32 x / scale -> uint8 codes (numpy-like rounding to nearest even); NaN gives 0."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x)
    if fmt == 0:
        return x.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def store_page(codes, scale, rows, first, fmt):
    """One page and head: codes [P][hd] uint8, scale float32 scalar, rows [n][hd] float32 from row `first` on. In
    float32 arithmetic, one operation at a time. Returns (codes, scale)."""
    n = rows.shape[0]
    f = np.float32
    s0 = f(scale) if first > 0 else f(0)
    a = rows.abs()
    big = f(float("nan")) if bool(torch.isnan(a).any()) else f(a.max().item())
    with np.errstate(all="ignore"):
        s1 = f(big * f(1.0 / LIMIT[fmt]))
        if s1 < f(1.1754944e-38):
            s1 = f(0)
        grown = bool(np.isnan(s1)) and not np.isnan(s0) or s1 > s0
        if not grown:
            s1 = s0
        inv = f(1) / s1 if s1 > 0 else f(0)
    out = codes.clone()
    if grown and first > 0:
        old = values(codes[:first], fmt).float() * torch.tensor(s0) * torch.tensor(inv)
        out[:first] = to_codes(old, fmt)
    out[first:first + n] = to_codes(rows * torch.tensor(inv), fmt)
    return out, s1


def attention(k, v, ks, vs, fmt, table, kv_len, start, q, hkv, scale, window, page):
    """(out, lse) in float64 of q [T][hq][hd], row by row of the definition."""
    T, hq, hd = q.shape
    out = torch.zeros(T, hq, hd, dtype=torch.float64, device=q.device)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=q.device)
    for r, n in enumerate(kv_len):
        rows = start[r + 1] - start[r]
        if n == 0 or rows == 0:
            continue
        ids = torch.tensor(table[r][:ceil(n, page)], device=q.device)
        K = (values(k[ids], fmt) * ks[ids].double()[:, :, None, None]).transpose(1, 2).reshape(-1, hkv, hd)[:n]
        V = (values(v[ids], fmt) * vs[ids].double()[:, :, None, None]).transpose(1, 2).reshape(-1, hkv, hd)[:n]
        key = torch.arange(n, device=q.device)
        at = n - rows + torch.arange(rows, device=q.device)[:, None]
        hide = key > at
        if window > 0:
            hide = hide | (key <= at - window)
        empty = hide.all(1)
        for h in range(hq):
            g = h // (hq // hkv)
            x = q[start[r]:start[r + 1], h].double() @ K[:, g].T * scale
            x = x.masked_fill(hide, -math.inf)
            w = torch.logsumexp(x, 1)
            p = torch.exp(x - w[:, None])
            p[empty] = 0
            out[start[r]:start[r + 1], h] = p @ V[:, g]
            lse[start[r]:start[r + 1], h] = w
    return out, lse
