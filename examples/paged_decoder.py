"""A small decoder over the paged cache, with the operators that stand around it used together: `python
examples/paged_decoder.py` on a B200.

A batch of requests shares a system prompt. Its blocks are filled once; each request's own prompt is prefilled behind it and
decoded greedily, every layer one rotate_store_kvcache (per-head norms, rotation, append) and one shared_prefix_attention.
The blocks then move to a second cache, as they move from a prefill to a decode GPU (transport.copy), and decoding goes on
from there -- the same tokens, bit for bit the same logits; and once more with paged_attention, each request's table naming
the system prompt's blocks itself, where only the order of the sums differs (a near tie between two tokens may fall the
other way, and that request goes on differently).
"""

from __future__ import annotations

import math
import os
import sys
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from lean_vllm_b200.attention.kvx_attention import AttentionWorkspace, paged_attention, shared_prefix_attention
from lean_vllm_b200.attention.kvx_rotary import RotaryTable, rotate_store_kvcache
from lean_vllm_b200.kv_transfer import transport
from lean_vllm_b200.kv_transfer.transport import CacheTable, CopyJob


@dataclass
class Shape:
    vocab: int = 512
    hidden: int = 512
    layers: int = 3
    heads: int = 8
    kv_heads: int = 2
    dim: int = 64
    block: int = 64


class Decoder:
    """A random-init decoder: RMSNorm, per-head norms of queries and keys, rotary positions, grouped-query attention over
    per-layer HND caches (2, blocks, kv heads, block, dim), SwiGLU."""

    def __init__(self, shape: Shape, seed: int = 0, positions: int = 4096):
        self.shape = s = shape
        g = torch.Generator(device="cuda").manual_seed(seed)

        def w(rows, cols, gain=1.0):
            return (torch.randn(rows, cols, generator=g, device="cuda") * gain / math.sqrt(rows)).to(torch.bfloat16)

        self.embed = w(s.vocab, s.hidden, math.sqrt(s.vocab))
        self.layers = [dict(qkv=w(s.hidden, (s.heads + 2 * s.kv_heads) * s.dim), o=w(s.heads * s.dim, s.hidden),
                            up=w(s.hidden, 8 * s.hidden), down=w(4 * s.hidden, s.hidden),
                            q_norm=(1 + 0.1 * torch.randn(s.dim, generator=g, device="cuda")).to(torch.bfloat16),
                            k_norm=(1 + 0.1 * torch.randn(s.dim, generator=g, device="cuda")).to(torch.bfloat16))
                       for _ in range(s.layers)]
        self.head = w(s.hidden, s.vocab)
        self.rotary = RotaryTable.build(positions, s.dim)
        self.workspace = AttentionWorkspace("cuda")

    def cache(self, blocks: int) -> list[torch.Tensor]:
        s = self.shape
        return [torch.zeros(2, blocks, s.kv_heads, s.block, s.dim, dtype=torch.bfloat16, device="cuda")
                for _ in range(s.layers)]

    @staticmethod
    def norm(x):
        x32 = x.float()
        return (x32 * torch.rsqrt(x32.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, tokens, positions, slots, caches, attend):
        """Logits of `tokens` at `positions`, whose keys and values go to `slots`; attend(query, k_cache, v_cache) reads the
        cache."""
        s = self.shape
        x = self.embed[tokens]
        for layer, cache in zip(self.layers, caches):
            qkv = (self.norm(x) @ layer["qkv"]).view(len(tokens), s.heads + 2 * s.kv_heads, s.dim)
            q, k, v = qkv.split([s.heads, s.kv_heads, s.kv_heads], 1)
            keys, values = cache.transpose(2, 3)  # (blocks, block, heads, dim), by strides
            q = rotate_store_kvcache(q, k, v, keys, values, slots, positions, self.rotary, q_weight=layer["q_norm"],
                                     k_weight=layer["k_norm"])
            x = x + attend(q, keys, values).flatten(1) @ layer["o"]
            gate, up = (self.norm(x) @ layer["up"]).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ layer["down"]
        return self.norm(x) @ self.head


class Batch:
    """Requests behind one system prompt: `prefix` blocks shared by all, a table of own blocks each."""

    def __init__(self, decoder: Decoder, caches, prefix_blocks, own_blocks, prefix_len: int, own_lens: list[int]):
        self.decoder, self.caches, self.prefix_len = decoder, caches, prefix_len
        self.prefix = torch.tensor(prefix_blocks, dtype=torch.int32, device="cuda")
        self.own = torch.tensor(own_blocks, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(own_lens, dtype=torch.int32, device="cuda")  # own tokens in the cache
        self.longest = max(own_lens)

    def slots(self, request, at):
        """Where a request's own token `at` goes."""
        block = self.decoder.shape.block
        return self.own[request, at // block].long() * block + at % block

    def prefill(self, prompts: list[torch.Tensor]):
        """Every request's own prompt in one ragged pass behind the system prompt: the last logits of each."""
        lens = [len(p) for p in prompts]
        starts = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        request = torch.repeat_interleave(torch.arange(len(prompts), device="cuda"), torch.tensor(lens, device="cuda"))
        at = torch.cat([torch.arange(n, device="cuda") for n in lens])
        self.lens, self.longest = torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens)

        def attend(q, keys, values):
            return shared_prefix_attention(q, keys, values, self.prefix, self.prefix_len, self.own, self.lens,
                                           q_starts=starts, max_q_len=max(lens), max_kv_len=max(lens),
                                           workspace=self.decoder.workspace)

        logits = self.decoder.forward(torch.cat(prompts), self.prefix_len + at, self.slots(request, at), self.caches, attend)
        return logits[starts[1:].long() - 1]

    def step(self, tokens, shared: bool = True):
        """One token of every request: its logits. `shared`: the system prompt is read once for all; else by each, from a
        table that begins with its blocks."""
        at = self.lens.long()
        self.lens = self.lens + 1
        self.longest += 1
        request = torch.arange(len(tokens), device="cuda")
        if shared:
            def attend(q, keys, values):
                return shared_prefix_attention(q, keys, values, self.prefix, self.prefix_len, self.own, self.lens,
                                               max_kv_len=self.longest, workspace=self.decoder.workspace)
        else:
            tables = torch.cat([self.prefix.expand(len(tokens), -1), self.own], 1).contiguous()

            def attend(q, keys, values):
                return paged_attention(q, keys, values, tables, self.lens + self.prefix_len,
                                       max_kv_len=self.longest + self.prefix_len, workspace=self.decoder.workspace)

        return self.decoder.forward(tokens, self.prefix_len + at, self.slots(request, at), self.caches, attend)

    def greedy(self, first, steps: int, shared: bool = True):
        """Tokens (steps, requests) and the logits they were taken from."""
        tokens, logits, token = [], [], first
        for _ in range(steps):
            logits.append(self.step(token, shared))
            token = logits[-1].argmax(-1)
            tokens.append(token)
        return torch.stack(tokens), torch.stack(logits)


def run(requests: int = 6, prefix_blocks: int = 5, steps: int = 12, seed: int = 0):
    """(tokens and logits decoded in place, from the moved blocks, and without sharing)."""
    shape = Shape()
    decoder = Decoder(shape, seed)
    g = torch.Generator().manual_seed(seed + 1)
    block = shape.block
    prefix_len = prefix_blocks * block  # whole blocks, so that a plain table can name them too
    system = torch.randint(0, shape.vocab, (prefix_len,), generator=g).cuda()
    prompts = [torch.randint(0, shape.vocab, (int(n),), generator=g).cuda()
               for n in torch.randint(1, 150, (requests,), generator=g)]
    own = -(-(max(len(p) for p in prompts) + steps) // block)
    total = prefix_blocks + requests * own
    prefill_order = torch.randperm(total, generator=g).tolist()
    decode_order = torch.randperm(total + 3, generator=g)[:total].tolist()

    def batch(order, caches):
        tables = [order[prefix_blocks + r * own : prefix_blocks + (r + 1) * own] for r in range(requests)]
        return Batch(decoder, caches, order[:prefix_blocks], tables, prefix_len, [len(p) for p in prompts])

    # The system prompt, once: a prompt of its own in its blocks.
    caches = decoder.cache(total)
    table = torch.tensor([prefill_order[:prefix_blocks]], dtype=torch.int32, device="cuda")
    at = torch.arange(prefix_len, device="cuda")
    starts = torch.tensor([0, prefix_len], dtype=torch.int32, device="cuda")
    decoder.forward(system, at, table[0, at // block].long() * block + at % block, caches,
                    lambda q, k, v: paged_attention(q, k, v, table, starts[1:], q_starts=starts, max_q_len=prefix_len,
                                                    workspace=decoder.workspace))
    here = batch(prefill_order, caches)
    first = here.prefill(prompts).argmax(-1)

    # The blocks move to a decode instance's cache, other ids there.
    moved = decoder.cache(total + 3)
    transport.copy([CacheTable.from_tensors(caches), CacheTable.from_tensors(moved)],
                   [CopyJob(0, 1, prefill_order, decode_order, 0, 0, shape.kv_heads)],
                   stream=torch.cuda.current_stream().cuda_stream)
    alone = [c.clone() for c in moved]
    return (here.greedy(first, steps), batch(decode_order, moved).greedy(first, steps),
            batch(decode_order, alone).greedy(first, steps, shared=False))


def main():
    (tokens, logits), (moved_tokens, moved_logits), (alone_tokens, alone_logits) = run()
    torch.cuda.synchronize()
    print("tokens of the first request:", tokens[:, 0].tolist())
    print("after the move: the same tokens", torch.equal(tokens, moved_tokens), "and logits", torch.equal(logits, moved_logits))
    agree = int((tokens == alone_tokens).all(0).sum())
    print(f"without sharing the prefix: first logits within {float((logits[0].float() - alone_logits[0].float()).abs().max()):.3f},",
          f"all tokens the same for {agree} of {tokens.size(1)} requests")


if __name__ == "__main__":
    main()
