"""Inputs for the attention and rotary tests, and both operators from their definitions in 64 bits.

Tolerances. The kernels hold everything in 32 bits but two roundings to the cache's type, of unit u (2^-8 in bf16,
2^-11 in fp16): the softmax weights ahead of the second product and the output. With weights p_j (sum L) and output o,
the first moves an element by at most u * sum(p_j |v_j|) / L =: u * A, the second by u |o|, so every element lies within
(u + 2^-12) (A + |o|), where 2^-12 covers 32-bit scores, exp2 and sums. fp16 weights below 2^-24 vanish: n keys lose at
most n 2^-25 max|v| more. The roundings are independent, so a row's root mean square error is at most
u * rms(sqrt(sum(p_j^2 v_j^2)) / L) + u * rms(o) (uniform roundings reach 1/sqrt(3) of each term), plus the 2^-12 term:
that is the sharper check, which one missing key of some hundreds fails.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def paged_case(q_lens, kv_lens, heads, kv_heads, dim, block, dtype, hnd=True, seed=0, shared=0, spare=2, garbage=True,
               fused=False):
    """Caches whose every row outside the sequences is NaN (with `garbage`), block ids in any order, table entries past
    a sequence's blocks far outside the cache."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // block) for n in kv_lens]
    shared_blocks = -(-shared // block)
    blocks = sum(need) + shared_blocks + spare
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    shape = (2, blocks, kv_heads, block, dim) if hnd else (2, blocks, block, kv_heads, dim)
    cache = torch.full(shape, math.nan, device="cuda", dtype=dtype)
    if not garbage:
        cache.zero_()
    view = cache.transpose(2, 3) if hnd else cache
    tables = torch.full((len(kv_lens), max(need + [1])), 2**30, dtype=torch.int32, device="cuda")
    at = shared_blocks
    keys, values = [], []

    def fill(ids, n):
        both = torch.randn(2, n, kv_heads, dim, generator=g, device="cuda").to(dtype)
        i = torch.arange(n, device="cuda")
        view[:, ids[i // block].long(), i % block] = both
        return both

    prefix = fill(order[:shared_blocks], shared) if shared else torch.zeros(2, 0, kv_heads, dim, device="cuda", dtype=dtype)
    for s, n in enumerate(kv_lens):
        ids = order[at : at + need[s]]
        tables[s, : need[s]] = ids
        at += need[s]
        both = torch.cat([prefix, fill(ids, n) if n else prefix[:, :0]], 1)
        keys.append(both[0])
        values.append(both[1])
    tokens = sum(q_lens)
    if fused:  # queries as a view into a wider product
        q = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g, device="cuda").to(dtype)[:, :heads]
    else:
        q = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(dtype)
    starts = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32, device="cuda")
    return dict(q=q, k_cache=view[0], v_cache=view[1], tables=tables, prefix_table=order[:shared_blocks].contiguous(),
                kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device="cuda"), q_starts=starts, q_lens=q_lens,
                keys=keys, values=values, shared=shared)


def attention64(case, scale=None, softcap=0.0, window=0, slopes=None, prefix_lens=None):
    """(output, weighted |v|, sqrt of the weighted squares of v) of every row, from the definition."""
    q = case["q"].double()
    heads, dim = q.shape[1:]
    kv_heads = case["keys"][0].size(1)
    scale = dim**-0.5 if scale is None else scale
    out, bound, spread = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    row = 0
    for s, n in enumerate(case["q_lens"]):
        k, v = case["keys"][s].double(), case["values"][s].double()
        total = k.size(0)
        j = torch.arange(total, device="cuda")[None]
        i = torch.arange(total - n, total, device="cuda")[:, None]
        seen = j <= i
        if window:
            seen &= j > i - window
        if prefix_lens is not None:
            seen |= j < min(int(prefix_lens[s]), total)
        seen |= j < case["shared"]
        for h in range(heads):
            kh = h // (heads // kv_heads)
            x = (q[row : row + n, h] @ k[:, kh].T) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x + float(slopes[h]) * (j - i)
            x = x.masked_fill(~seen, -math.inf)
            top = x.amax(-1, keepdim=True).clamp_min(-1e300) if total else x.new_zeros(n, 1)
            p = (x - top).exp().masked_fill(~seen, 0.0)
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            out[row : row + n, h] = p @ v[:, kh]
            bound[row : row + n, h] = p @ v[:, kh].abs()
            spread[row : row + n, h] = (p.square() @ v[:, kh].square()).sqrt()
        row += n
    return out, bound, spread


def check_attention(got, case, **options):
    want, bound, spread = attention64(case, **options)
    u = UNIT[got.dtype]
    most = max([k.size(0) for k in case["keys"]] + [1])
    biggest = max([float(v.abs().max()) for v in case["values"] if v.numel()] + [0.0])
    lost = most * 2.0**-25 * biggest if got.dtype == torch.float16 else 0.0
    error = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    limit = (u + 2.0**-12) * (bound + want.abs()) + lost
    assert bool((error <= limit).all()), f"largest excess {float((error - limit).max())}"

    def rms(x):
        return x.square().mean(-1).sqrt()

    row_limit = u * (rms(spread) + rms(want)) + 2.0**-12 * rms(bound) + lost
    assert bool((rms(error) <= row_limit).all()), f"largest row excess {float((rms(error) - row_limit).max())}"


def rotate64(x, weight, norm_dim, rotary_first, table, positions, interleaved, eps=1e-6):
    """(rows normed and rotated in 64 bits, the size of the terms each element is made of)."""
    y = x.double().clone()
    if weight is not None:
        head = y[..., :norm_dim]
        y[..., :norm_dim] = head / (head.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = y.abs()
    r = table.size(1)
    angle = table.double()[positions.long().clamp(0, table.size(0) - 1)][:, None]
    c, s = angle[..., : r // 2], angle[..., r // 2 :]
    p = torch.arange(r // 2, device=x.device)
    i, j = (rotary_first + 2 * p, rotary_first + 2 * p + 1) if interleaved else (rotary_first + p, rotary_first + p + r // 2)
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    size[..., i], size[..., j] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def check_rotated(got, want, size):
    """One rounding to the rows' type; 32-bit arithmetic before it (2^-20 of the terms' size covers the sum of squares,
    the reciprocal root and three products); fp16's smallest step, 2^-24."""
    error = (got.double() - want).abs()
    limit = UNIT[got.dtype] * want.abs() + 2.0**-20 * size + 2.0**-25
    assert bool((error <= limit).all()), f"largest excess {float((error - limit).max())}"
