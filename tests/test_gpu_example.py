"""The example decoder: rotary stores, prompt and decode attention and the shared prefix together, around a block move."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    import sys

    spec = importlib.util.spec_from_file_location("paged_decoder", os.path.join(ROOT, "examples", "paged_decoder.py"))
    module = importlib.util.module_from_spec(spec)
    sys.modules["paged_decoder"] = module  # its dataclasses look themselves up there
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("requests, prefix_blocks", [(1, 1), (6, 5), (40, 3)])
def test_decoding_goes_on_from_moved_blocks_and_without_sharing(example, requests, prefix_blocks):
    """From the moved blocks, bit for bit; reading the prefix per request, up to the order of the sums: the logits differ by
    bf16 roundings along the layers (a few hundredths at logits of about 1), as long as the tokens fed back are the same."""
    (tokens, logits), (moved, moved_logits), (alone, alone_logits) = example.run(requests, prefix_blocks, steps=8)
    assert torch.equal(tokens, moved) and torch.equal(logits, moved_logits)
    assert torch.isfinite(logits).all() and len(torch.unique(tokens)) > 1
    same = torch.ones(requests, dtype=torch.bool, device="cuda")
    for step in range(8):
        off = (logits[step].float() - alone_logits[step].float()).abs().amax(-1)
        assert bool((off[same] < 0.25).all()), float(off[same].max())
        same &= tokens[step] == alone[step]
    assert int(same.sum()) * 2 >= requests


def test_a_step_is_the_plain_computation(example):
    """One decode step's attention input and output against a plain float32 computation of the layer's queries, keys and
    values from the same cache."""
    shape = example.Shape()
    decoder = example.Decoder(shape, seed=3)
    caches = decoder.cache(8)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, shape.vocab, (200,), generator=g).cuda()
    table = torch.tensor([[6, 1, 3, 0]], dtype=torch.int32, device="cuda")
    at = torch.arange(200, device="cuda")
    slots = table[0, at // shape.block].long() * shape.block + at % shape.block
    starts = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    seen = []

    def attend(q, keys, values):
        out = example.paged_attention(q, keys, values, table, starts[1:], q_starts=starts, max_q_len=200,
                                      workspace=decoder.workspace)
        k = keys[table[0].long()].flatten(0, 1)[:200].float().repeat_interleave(shape.heads // shape.kv_heads, 1)
        v = values[table[0].long()].flatten(0, 1)[:200].float().repeat_interleave(shape.heads // shape.kv_heads, 1)
        scores = torch.einsum("qhd,khd->hqk", q.float(), k) / shape.dim**0.5
        scores = scores.masked_fill(torch.ones(200, 200, device="cuda").triu(1).bool(), float("-inf"))
        want = torch.einsum("hqk,khd->qhd", scores.softmax(-1), v)
        seen.append(float((out.float() - want).abs().max() / want.abs().max()))
        return out

    decoder.forward(prompt, at, slots, caches, attend)
    assert len(seen) == shape.layers and max(seen) < 2.0**-7  # two bf16 roundings of 2^-8 each, at the largest element
