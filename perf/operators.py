"""The operators around the paged KV cache: what they are called with, what they compute and what that costs.

Four operators, each in a plain form (elementary torch operations in 32 bits) and through the package's entry points:

- rotate_store_kvcache: per-head norms of queries and keys, the rotation by position, and the append of keys and
  values to a paged cache, in one pass;
- rotate_store_latents: the same for latent rows (normed part | rotated part) and the queries' rotated part;
- paged_attention: attention that reads the paged cache, for single tokens and for prompt chunks, with an optional
  tanh cap, distance bias, sliding window and prefix mask;
- shared_prefix_attention: attention of a batch whose sequences share one long prefix, the prefix read once for all.

A case is a dict of plain values; sequence lengths are derived from its numbers, tensors from the seed.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases


def _append(name, tokens, q_heads, kv_heads, dim, rotary, **more):
    case = dict(name=name, op="append", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                interleaved=False, norm=True, dtype="bf16", hnd=True, block=256, fused=True, padding=0)
    case.update(more)
    return case


def _latents(name, tokens, heads, **more):
    case = dict(name=name, op="latents", tokens=tokens, heads=heads, rank=512, rotary=64, interleaved=True, norm=True,
                dtype="bf16", block=64, padding=0)
    case.update(more)
    return case


def _paged(name, batch, q_max, kv_max, q_heads, kv_heads, dim, **more):
    case = dict(name=name, op="paged", batch=batch, q_max=q_max, kv_max=kv_max, kv_min=kv_max, mix=0, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, dtype="bf16", hnd=True, block=256, softcap=0.0, window=0, bias=False,
                prefix=0)
    case.update(more)
    return case


def _shared(name, batch, prefix, kv_max, q_heads, kv_heads, dim, **more):
    case = dict(name=name, op="shared", batch=batch, q_max=1, prefix=prefix, kv_max=kv_max, kv_min=1, mix=0,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype="bf16", hnd=True, block=256, softcap=0.0)
    case.update(more)
    return case


def listed():
    return [
        # One new token of one request: a decode step's smallest append, where the launch is what counts.
        _append("append_1", 1, 32, 8, 128, 128),
        # A whole prompt of 8k tokens of an 8-KV-head model, out of its fused qkv product into 256-token HND blocks.
        _append("append_8192", 8192, 32, 8, 128, 128),
        # A ragged chunk of a small model: interleaved pairs over half of a 64-wide head, no norms, NHD cache with
        # 24-token blocks (not a power of two), some rows padding.
        _append("append_777_partial", 777, 14, 2, 64, 32, interleaved=True, norm=False, dtype="fp16", hnd=False,
                block=24, padding=13),
        # A decode step of 64 requests of a latent-attention model: one 576-wide latent row each.
        _latents("latents_64", 64, 16),
        # A prompt of 8k tokens of that model, less one: an odd row count.
        _latents("latents_8191", 8191, 16),
        # One request early in its answer: a short cache, where latency counts.
        _paged("decode_1_short", 1, 1, 317, 32, 8, 128),
        # A busy decode step: 64 requests of very different lengths.
        _paged("decode_64_ragged", 64, 1, 16384, 32, 8, 128, kv_min=200, mix=1),
        # One request with a long document: all the parallelism has to come from the cache's length.
        _paged("decode_1_long", 1, 1, 131071, 32, 8, 128),
        # A prompt of 8k tokens prefilled at once, causal.
        _paged("prompt_8192", 1, 8192, 8192, 32, 8, 128),
        # Chunks of seven requests beside single tokens: capped scores, a sliding window, 64-wide fp16 heads in an
        # NHD cache of 24-token blocks, seven query heads a KV head.
        _paged("chunks_7_capped", 7, 700, 4099, 14, 2, 64, kv_min=50, mix=2, dtype="fp16", hnd=False, block=24,
               softcap=30.0, window=1000),
        # 64 requests that share an 8k system prompt, each with its own turn behind it.
        _shared("shared_64", 64, 8192, 700, 32, 8, 128, mix=3),
        # Few requests over a long shared document of odd length, four drafted tokens each, 16-token blocks.
        _shared("shared_5_drafts", 5, 30011, 129, 32, 8, 128, q_max=4, mix=4, block=16),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.choice(["append", "latents", "paged", "paged", "shared"])
    if kind == "append":
        kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 128])
        return _append("", _log(rng, 1, 8192), kv_heads * group, kv_heads, dim, rng.choice([dim, dim // 2, dim // 4]),
                       interleaved=rng.random() < 0.4, norm=rng.random() < 0.6, dtype=rng.choice(["bf16", "fp16"]),
                       hnd=rng.random() < 0.6, block=rng.choice([16, 24, 64, 256]), fused=rng.random() < 0.6,
                       padding=rng.choice([0, 0, 7, 31]))
    if kind == "latents":
        return _latents("", _log(rng, 1, 8192), rng.choice([8, 16, 32]), interleaved=rng.random() < 0.6,
                        norm=rng.random() < 0.7, dtype=rng.choice(["bf16", "fp16"]), block=rng.choice([16, 24, 64]),
                        padding=rng.choice([0, 0, 7]))
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8]), rng.choice([64, 128])
    while kv_heads * group > 32:
        group = rng.choice([1, 2, 4])
    common = dict(mix=rng.randrange(1 << 30), dtype=rng.choice(["bf16", "fp16"]), hnd=rng.random() < 0.6,
                  block=rng.choice([16, 24, 64, 256]))
    if kind == "shared":
        batch = _log(rng, 1, 128)
        return _shared("", batch, _log(rng, 1, 32768), _log(rng, 1, 700), kv_heads * group, kv_heads, dim,
                       q_max=rng.choice([1, 1, 1, 2, 4]), softcap=rng.choice([0.0, 0.0, 20.0]), **common)
    if rng.random() < 0.5:
        batch = _log(rng, 1, 128)
        kv_max = _log(rng, 1, min(131072, (1 << 19) // batch))
        q_max = rng.choice([1, 1, 1, 1, 3])
    else:
        batch = _log(rng, 1, 16)
        kv_max = _log(rng, 16, 8192 // (1 if batch < 4 else 2))
        q_max = _log(rng, 2, max(2, min(kv_max, 8192 // batch)))
    return _paged("", batch, q_max, max(kv_max, q_max), kv_heads * group, kv_heads, dim,
                  kv_min=_log(rng, 1, max(kv_max, q_max)), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                  window=rng.choice([0, 0, 0, _log(rng, 1, 2048)]), bias=rng.random() < 0.2,
                  prefix=rng.choice([0, 0, 0, _log(rng, 1, 1024)]), **common)


def _lengths(case):
    """Per sequence: query tokens and cached tokens (the query's own included), fixed by the case's numbers."""
    rng = random.Random(case["mix"])
    batch, kv_max = case["batch"], case["kv_max"]
    kv = [kv_max] + [_log(rng, min(case["kv_min"], kv_max), kv_max) for _ in range(batch - 1)]
    q = [min(kv[0], case["q_max"])]
    for n in kv[1:]:
        most = min(n, case["q_max"])
        q.append(1 if rng.random() < 0.3 else _log(rng, 1, most))
    both = list(zip(q, kv))
    rng.shuffle(both)
    return [a for a, _ in both], [b for _, b in both]


def _prefix_of(case, kv_len):
    return min(case["prefix"], kv_len)


def _pairs(case, q_len, kv_len):
    """How many (query, key) pairs a sequence's mask leaves, and how many of its keys any query sees."""
    prefix, window = _prefix_of(case, kv_len), case["window"]
    pairs, first = 0, kv_len
    for p in range(kv_len - q_len, kv_len):
        low = max(0, p + 1 - window) if window else 0
        pairs += max(p + 1, prefix) if low <= prefix else prefix + p + 1 - low
        first = min(first, low)
    return pairs, kv_len if first <= prefix else prefix + kv_len - first


def work(case):
    if case["op"] == "append":
        rows = case["tokens"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        rotated = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        # rows in and out, the rows of cos and sin, slots and positions
        return {"bytes": 2 * rows * 2 + case["tokens"] * (case["rotary"] * 4 + 16),
                "flops": rotated * (3 * case["rotary"] + (4 * case["dim"] if case["norm"] else 0))}
    if case["op"] == "latents":
        row = case["rank"] + case["rotary"] + case["heads"] * case["rotary"]
        return {"bytes": 2 * case["tokens"] * row * 2 + case["tokens"] * (case["rotary"] * 4 + 16),
                "flops": case["tokens"] * (3 * (case["heads"] + 1) * case["rotary"] + 4 * case["rank"])}
    q_lens, kv_lens = _lengths(case)
    dim, heads, kv_heads = case["dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "paged":
        seen = [_pairs(case, q, n) for q, n in zip(q_lens, kv_lens)]
        pairs, keys = sum(p for p, _ in seen), sum(k for _, k in seen)
    else:
        pairs = sum(q * (case["prefix"] + n - q) + q * (q + 1) // 2 for q, n in zip(q_lens, kv_lens))
        keys = case["prefix"] + sum(kv_lens)
    return {"bytes": (2 * sum(q_lens) * heads + 2 * keys * kv_heads) * dim * 2, "flops": 4 * dim * heads * pairs}


# ------------------------------------------------------------------------------------------------ inputs


def _table(rows, rotary, base=1000000.0):
    """cos of every pair's angle, then sin, for positions 0..rows-1."""
    freq = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _randn(g, *shape, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(0.0, scale, generator=g)


def _kv_cache(g, case, blocks):
    shape = ((2, blocks, case["kv_heads"], case["block"], case["dim"]) if case["hnd"] else
             (2, blocks, case["block"], case["kv_heads"], case["dim"]))
    cache = _randn(g, *shape, dtype=DTYPES[case["dtype"]])
    return cache.transpose(2, 3) if case["hnd"] else cache  # (2, blocks, block, heads, dim) by strides


def _slots(g, case, blocks):
    """Slots as an engine hands them out: whole blocks in any order, a request's tokens one after another in them."""
    tokens, block = case["tokens"], case["block"]
    table = torch.randperm(blocks, generator=g, device="cuda")
    at = torch.arange(tokens, device="cuda")
    slots = table[at // block] * block + at % block
    if case["padding"]:
        slots[case["padding"] - 1 :: case["padding"]] = -1
    return slots


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] in ("append", "latents"):
        tokens = case["tokens"]
        blocks = -(-tokens // case["block"]) + 2
        state["slots"] = _slots(g, case, blocks)
        start = int(torch.randint(0, 4096, (1,), generator=g, device="cuda"))
        state["positions"] = torch.arange(start, start + tokens, device="cuda")
        state["table"] = _table(16384, case["rotary"])
    if case["op"] == "append":
        q_heads, kv_heads, dim = case["q_heads"], case["kv_heads"], case["dim"]
        if case["fused"]:  # views into one product's output, as a model's qkv projection leaves them
            qkv = _randn(g, tokens, q_heads + 2 * kv_heads, dim, dtype=dtype)
            state["q"], state["k"], state["v"] = qkv.split([q_heads, kv_heads, kv_heads], 1)
        else:
            state["q"] = _randn(g, tokens, q_heads, dim, dtype=dtype)
            state["k"] = _randn(g, tokens, kv_heads, dim, dtype=dtype)
            state["v"] = _randn(g, tokens, kv_heads, dim, dtype=dtype)
        state["k_cache"], state["v_cache"] = _kv_cache(g, case, blocks)
        state["q_weight"] = state["k_weight"] = None
        if case["norm"]:
            state["q_weight"] = (1 + _randn(g, dim, dtype=torch.float32, scale=0.2)).to(dtype)
            state["k_weight"] = (1 + _randn(g, dim, dtype=torch.float32, scale=0.2)).to(dtype)
    elif case["op"] == "latents":
        state["latent"] = _randn(g, tokens, case["rank"] + case["rotary"], dtype=dtype)
        # The queries' rotated parts lie behind each head's unrotated 128: a strided view.
        state["query_pe"] = _randn(g, tokens, case["heads"], 128 + case["rotary"], dtype=dtype)[..., 128:]
        state["cache"] = _randn(g, blocks, case["block"], case["rank"] + case["rotary"], dtype=dtype)
        state["weight"] = (1 + _randn(g, case["rank"], dtype=torch.float32, scale=0.2)).to(dtype) if case["norm"] else None
    else:
        q_lens, kv_lens = _lengths(case)
        block, prefix = case["block"], case["prefix"] if case["op"] == "shared" else 0
        need = [-(-n // block) for n in kv_lens]
        prefix_blocks = -(-prefix // block)
        blocks = sum(need) + prefix_blocks + 1
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        tables = torch.full((case["batch"], max(need)), -1, dtype=torch.int32, device="cuda")
        at = prefix_blocks
        for s, n in enumerate(need):
            tables[s, :n] = order[at : at + n]
            at += n
        state["tables"], state["prefix_table"] = tables, order[:prefix_blocks].contiguous()
        state["q"] = _randn(g, sum(q_lens), case["q_heads"], case["dim"], dtype=dtype)
        state["k_cache"], state["v_cache"] = _kv_cache(g, case, blocks)
        state["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        state["q_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        state["q_lens_host"], state["kv_lens_host"] = q_lens, kv_lens
        state["slopes"] = state["prefix_lens"] = None
        if case["op"] == "paged":
            if case["bias"]:
                state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["q_heads"] + 1, device="cuda") / case["q_heads"])
            if case["prefix"]:
                state["prefix_lens"] = torch.tensor([_prefix_of(case, n) for n in kv_lens], dtype=torch.int32,
                                                    device="cuda")
    if own:
        from lean_vllm_b200.attention import kvx_attention, kvx_rotary

        state["rotary_ops"], state["attention_ops"] = kvx_rotary, kvx_attention
        if case["op"] in ("append", "latents"):
            state["rotary"] = kvx_rotary.RotaryTable(state["table"], interleaved=case["interleaved"])
        else:
            state["workspace"] = kvx_attention.AttentionWorkspace(torch.device("cuda", torch.cuda.current_device()))
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def _plain_norm(x, weight, eps=1e-6):
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()


def _plain_rotate(x, table, positions, interleaved):
    """The first table.size(1) elements of each row, rotated pair by pair; the rest as they are."""
    rotary = table.size(1)
    row = table[positions]
    cos, sin = row[:, None, : rotary // 2], row[:, None, rotary // 2 :]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., : rotary // 2], turned[..., rotary // 2 :]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(st):
    case, slots = st["case"], st["slots"]
    q = _plain_rotate(_plain_norm(st["q"].float(), st["q_weight"]), st["table"], st["positions"], case["interleaved"])
    k = _plain_rotate(_plain_norm(st["k"].float(), st["k_weight"]), st["table"], st["positions"], case["interleaved"])
    keep = slots >= 0
    block, offset = slots[keep] // case["block"], slots[keep] % case["block"]
    st["k_cache"][block, offset] = k[keep].to(st["k_cache"].dtype)
    st["v_cache"][block, offset] = st["v"][keep]
    return q.to(st["q"].dtype), st["k_cache"], st["v_cache"]


def _plain_latents(st):
    case, slots = st["case"], st["slots"]
    rank = case["rank"]
    latent = st["latent"].float()
    c = _plain_norm(latent[:, :rank], st["weight"])
    pe = _plain_rotate(latent[:, None, rank:], st["table"], st["positions"], case["interleaved"])[:, 0]
    q = _plain_rotate(st["query_pe"].float(), st["table"], st["positions"], case["interleaved"])
    keep = slots >= 0
    st["cache"][slots[keep] // case["block"], slots[keep] % case["block"]] = torch.cat([c, pe], 1)[keep].to(st["cache"].dtype)
    return q.to(st["query_pe"].dtype), st["cache"]


def _plain_gather(cache, table, n):
    return cache[table[: -(-n // cache.size(1))].long()].flatten(0, 1)[:n].float()  # (tokens, heads, dim)


def _plain_rows(st, q, keys, values, positions, kv_len, prefix_len):
    """Attention of q (tokens, heads, dim) in 32 bits over keys and values of one sequence, some query rows and one
    KV head at a time so that the scores fit."""
    case = st["case"]
    group = case["q_heads"] // case["kv_heads"]
    out = torch.empty_like(q, dtype=torch.float32)
    at = torch.arange(kv_len, device=q.device)
    step = max(1, (1 << 28) // max(1, kv_len * group))
    for t in range(0, q.size(0), step):
        pos = positions[t : t + step, None]
        seen = at[None] <= pos
        if case.get("window"):
            seen &= at[None] > pos - case["window"]
        if prefix_len:
            seen |= at[None] < prefix_len
        for h in range(case["kv_heads"]):
            rows = q[t : t + step, h * group : (h + 1) * group].float()
            scores = torch.matmul(rows.transpose(0, 1), keys[:, h].T) / math.sqrt(case["dim"])  # (group, tokens, keys)
            if case["softcap"]:
                scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
            if st["slopes"] is not None:
                scores = scores + st["slopes"][h * group : (h + 1) * group, None, None] * (at[None] - pos).float()
            scores = scores.masked_fill(~seen, float("-inf"))
            scores = scores - scores.amax(-1, keepdim=True)
            weights = scores.exp()
            weights = weights / weights.sum(-1, keepdim=True)
            out[t : t + step, h * group : (h + 1) * group] = torch.matmul(weights, values[:, h]).transpose(0, 1)
    return out


def _plain_attention(st):
    case, q = st["case"], st["q"]
    out = torch.empty_like(q)
    prefix = case["prefix"] if case["op"] == "shared" else 0
    if prefix:
        prefix_k = _plain_gather(st["k_cache"], st["prefix_table"], prefix)
        prefix_v = _plain_gather(st["v_cache"], st["prefix_table"], prefix)
    start = 0
    for s, (q_len, kv_len) in enumerate(zip(st["q_lens_host"], st["kv_lens_host"])):
        keys = _plain_gather(st["k_cache"], st["tables"][s], kv_len)
        values = _plain_gather(st["v_cache"], st["tables"][s], kv_len)
        if prefix:
            keys, values = torch.cat([prefix_k, keys]), torch.cat([prefix_v, values])
        total = prefix + kv_len
        positions = torch.arange(total - q_len, total, device=q.device)
        both_ways = _prefix_of(case, kv_len) if case["op"] == "paged" else 0
        rows = _plain_rows(st, q[start : start + q_len], keys, values, positions, total, both_ways)
        out[start : start + q_len] = rows.to(q.dtype)
        start += q_len
    return out


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "latents": _plain_latents, "paged": _plain_attention,
                "shared": _plain_attention}[case["op"]](state)
    if case["op"] == "append":
        q = state["rotary_ops"].rotate_store_kvcache(
            state["q"], state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"], state["positions"],
            state["rotary"], q_weight=state["q_weight"], k_weight=state["k_weight"])
        return q, state["k_cache"], state["v_cache"]
    if case["op"] == "latents":
        q = state["rotary_ops"].rotate_store_latents(
            state["latent"], state["cache"], state["slots"], state["positions"], state["rotary"],
            query_pe=state["query_pe"], weight=state["weight"])
        return q, state["cache"]
    ops, many = state["attention_ops"], case["q_max"] > 1
    more = {"q_starts": state["q_starts"], "max_q_len": case["q_max"]} if many else {}
    if case["op"] == "paged":
        return ops.paged_attention(
            state["q"], state["k_cache"], state["v_cache"], state["tables"], state["kv_lens"],
            max_kv_len=case["kv_max"], softcap=case["softcap"], window=case["window"], slopes=state["slopes"],
            prefix_lens=state["prefix_lens"], workspace=state["workspace"], **more)
    return ops.shared_prefix_attention(
        state["q"], state["k_cache"], state["v_cache"], state["prefix_table"], case["prefix"], state["tables"],
        state["kv_lens"], max_kv_len=case["kv_max"], softcap=case["softcap"], workspace=state["workspace"], **more)


# ------------------------------------------------------------------------------------------------ 64 bits


def _exact_turn(x, table, positions, interleaved):
    """Pairs as complex numbers, turned by cos + i sin."""
    rotary = table.size(1)
    half = rotary // 2
    turn = torch.complex(table[positions, :half].double(), table[positions, half:].double()).unsqueeze(1)
    x = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:rotary:2], x[..., 1:rotary:2]) * turn
        x[..., 0:rotary:2], x[..., 1:rotary:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half], x[..., half:rotary]) * turn
        x[..., :half], x[..., half:rotary] = z.real, z.imag
    return x


def _exact_normed(x, weight):
    if weight is None:
        return x
    return weight.double() * x / (x.square().sum(-1, keepdim=True) / x.size(-1) + 1e-6).sqrt()


def _exact_store(cache, rows, slots):
    out = cache.double()
    for_rows = torch.nonzero(slots >= 0)[:, 0]
    s = slots[for_rows]
    out[torch.div(s, cache.size(1), rounding_mode="floor"), s.remainder(cache.size(1))] = rows[for_rows]
    return out


def exact(case, seed):
    global own
    was, own = own, False  # the inputs alone
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "append":
        q = _exact_turn(_exact_normed(st["q"].double(), st["q_weight"]), st["table"], st["positions"], case["interleaved"])
        k = _exact_turn(_exact_normed(st["k"].double(), st["k_weight"]), st["table"], st["positions"], case["interleaved"])
        return q, _exact_store(st["k_cache"], k, st["slots"]), _exact_store(st["v_cache"], st["v"].double(), st["slots"])
    if case["op"] == "latents":
        rank, latent = case["rank"], st["latent"].double()
        pe = _exact_turn(latent[:, None, rank:], st["table"], st["positions"], case["interleaved"])[:, 0]
        rows = torch.cat([_exact_normed(latent[:, :rank], st["weight"]), pe], -1)
        q = _exact_turn(st["query_pe"].double(), st["table"], st["positions"], case["interleaved"])
        return q, _exact_store(st["cache"], rows, st["slots"])
    heads, kv_heads, dim, block = case["q_heads"], case["kv_heads"], case["dim"], case["block"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    head_of = torch.arange(heads, device="cuda") // (heads // kv_heads)
    shared = case["prefix"] if case["op"] == "shared" else 0
    row = 0
    for s, (q_len, own_len) in enumerate(zip(st["q_lens_host"], st["kv_lens_host"])):
        # Every key's (block, offset): the shared prefix's, then the sequence's own.
        mine = torch.arange(own_len, device="cuda")
        ids, offsets = st["tables"][s][mine // block].long(), mine % block
        if shared:
            front = torch.arange(shared, device="cuda")
            ids = torch.cat([st["prefix_table"][front // block].long(), ids])
            offsets = torch.cat([front % block, offsets])
        total = shared + own_len
        key_at = torch.arange(total, device="cuda")
        for h in range(heads):
            kh = int(head_of[h])
            keys = st["k_cache"][ids, offsets, kh].double()
            values = st["v_cache"][ids, offsets, kh].double()
            chunk = max(1, (1 << 26) // total)
            for a in range(0, q_len, chunk):
                b = min(q_len, a + chunk)
                at = torch.arange(total - q_len + a, total - q_len + b, device="cuda").unsqueeze(1)
                e = (st["q"][row + a : row + b, h].double() @ keys.t()) * dim ** -0.5
                if case["softcap"]:
                    e = case["softcap"] * (e / case["softcap"]).tanh()
                if st["slopes"] is not None:
                    e -= st["slopes"][h].double() * (at - key_at)
                hidden = key_at > at
                if case.get("window"):
                    hidden = hidden | (at - key_at >= case["window"])
                if case["op"] == "paged" and case["prefix"]:
                    hidden = hidden & (key_at >= min(case["prefix"], own_len))
                e[hidden] = -math.inf
                out[row + a : row + b, h] = (e - e.logsumexp(-1, keepdim=True)).exp() @ values
        row += q_len
    return out
