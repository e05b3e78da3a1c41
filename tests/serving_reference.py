"""Plain forms of the serving operators in 64 bits, row by row from their definitions, and the bounds their bf16 kernels have to keep."""
import math

import torch

BF16_HALF = 2.0 ** -8          # half a step of bf16, relative to the value
F32_HALF = 2.0 ** -24


def quantise(x):
    """Rows of the last axis -> (codes as float, scale bytes). 64 bits on the CPU."""
    x = x.double().cpu()
    amax = x.abs().amax(-1)
    e = torch.full_like(amax, -100.0)
    some = amax > 0
    e[some] = torch.ceil(torch.log2(amax[some] / 448))
    e = e.clamp(-100, 7)
    u = (x / 2.0 ** e[..., None]).clamp(-448, 448)
    step = 2.0 ** (torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(u / step) * step, (e + 127).to(torch.uint8)


def cached(cache, which, page, at):
    """One cached row of all heads, [n_kv_heads, head_dim], as the values it stands for."""
    x = getattr(cache, which)[page, :, at].cpu()
    if cache.k_scale is None:
        return x.double()
    b = getattr(cache, which + "_scale")[page, :, at].cpu().long()
    return torch.where(b[:, None] == 255, torch.full((), math.nan, dtype=torch.float64), x.double() * 2.0 ** (b.double() - 127)[:, None])


def context(cache, table, i, n):
    """Keys and values [n, n_kv_heads, head_dim] of sequence i's first n positions; rows without a page are None-like: a mask says which are there."""
    k = torch.zeros(n, cache.n_kv_heads, cache.head_dim, dtype=torch.float64)
    v, there = torch.zeros_like(k), torch.zeros(n, dtype=torch.bool)
    for p in range(n):
        idx = p // cache.page_size
        page = int(table[i, idx]) if idx < table.shape[1] else -1
        if 0 <= page < cache.n_pages:
            there[p] = True
            k[p], v[p] = cached(cache, "k", page, p % cache.page_size), cached(cache, "v", page, p % cache.page_size)
    return k, v, there


def attention(cache, q_start, kv_len, table, q, scale, causal=True, window=0):
    """(out, lse, bound of |out - exact|, bound of |lse - exact|), rows of no sequence are NaN.

    The bound: a key's score is a sum of d products in fp32, wrong by at most (d + 16) 2^-23 of the sum of their magnitudes (each addition and the scaling half a
    step, doubled for units that cut instead of rounding), and its exponential by as much relatively (twice: it and the sum it is divided by) plus 2^-20 for the exponential
    itself; a probability is rounded to bf16 (2^-8) before it meets its value; the result is rounded to bf16 once (2^-8)."""
    rows, heads, d = q.shape
    q, group = q.double().cpu(), heads // cache.n_kv_heads
    out = torch.full((rows, heads, d), math.nan, dtype=torch.float64)
    lse, tol, tol_lse = torch.full((rows, heads), math.nan, dtype=torch.float64), torch.zeros(rows, heads, d, dtype=torch.float64), torch.zeros(rows, heads, dtype=torch.float64)
    for i in range(len(kv_len)):
        s, e, n = int(q_start[i]), int(q_start[i + 1]), int(kv_len[i])
        if e <= s:
            continue
        k, v, there = context(cache, table, i, max(n, 0))
        pos, key = torch.arange(n - (e - s), n)[:, None], torch.arange(max(n, 0))
        see = there.expand(e - s, -1).clone()
        if causal:
            see &= key <= pos
        if window:
            see &= key > pos - window
        for h in range(heads):
            kk, vv = k[:, h // group], v[:, h // group]
            for t in range(e - s):
                at = see[t].nonzero().flatten()
                if not len(at):
                    out[s + t, h], lse[s + t, h] = 0, -math.inf
                    continue
                x = kk[at] @ q[s + t, h] * scale
                z = torch.logsumexp(x, 0)
                p = torch.exp(x - z)
                out[s + t, h] = p @ vv[at]
                lse[s + t, h] = z
                off = float((kk[at].abs() @ q[s + t, h].abs()).max()) * abs(scale) * (d + 16) * 2.0 ** -23 + 2.0 ** -20
                mag = p @ vv[at].abs()
                tol[s + t, h] = mag * (BF16_HALF + 2 * off) + out[s + t, h].abs() * BF16_HALF * (1 + BF16_HALF) + 1e-37
                tol_lse[s + t, h] = off + abs(float(z)) * 2.0 ** -22
    return out, lse, tol, tol_lse


def logits(x, tokens=None, n_tokens=None, n_prompt=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, mask=None):
    """(values in 64 bits, bound of the error before the result's own rounding)"""
    y = x.double().cpu().clone()
    rows, vocab = y.shape
    mag = y.abs().clone()
    for b in range(rows):
        if tokens is not None:
            n = min(max(int(n_tokens[b]), 0), tokens.shape[1]) if n_tokens is not None else tokens.shape[1]
            first = int(n_prompt[b]) if n_prompt is not None else 0
            seen, count = set(), {}
            for j, t in enumerate(tokens[b, :n].tolist()):
                if 0 <= t < vocab:
                    seen.add(t)
                    if j >= first:
                        count[t] = count.get(t, 0) + 1
            for t in seen:
                if repetition is not None:
                    r = float(repetition[b])
                    y[b, t] = y[b, t] / r if y[b, t] > 0 else y[b, t] * r
                mag[b, t] = max(float(mag[b, t]), abs(float(y[b, t])))
            for t, c in count.items():
                f, p = float(frequency[b]) if frequency is not None else 0.0, float(presence[b]) if presence is not None else 0.0
                y[b, t] -= f * c + p
                mag[b, t] += abs(f) * c + abs(p)
        if bias is not None:
            for t, w in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= t < vocab:
                    y[b, t] += w
                    mag[b, t] += abs(w)
        if mask is not None:
            words = mask[b].cpu().tolist()
            for t in range(vocab):
                if not (words[t // 32] >> (t % 32)) & 1:
                    y[b, t] = -math.inf
    # a division, a product and four additions and as many more as an id's biases, half a step of fp32 each
    return y, mag * (8 + (bias.shape[1] if bias is not None else 0)) * F32_HALF
