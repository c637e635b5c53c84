"""Attention over the paged KV cache as sm_100a kernels (kvx_attention): single tokens, prompt chunks and mixtures of
both, reading the blocks a prefill stored or a transfer brought, in the NHD or HND layout the caches have.

`paged_attention` is the general call; `shared_prefix_attention` is for a batch whose sequences all begin with the same
cached prefix, which is read once for all of them. Lengths and block tables stay on the device: no call here waits for
it. For serving: inputs that require a gradient are refused while gradients are recorded. There is no fallback: without
libkvx.so the calls raise.
"""

from __future__ import annotations

import torch

from lean_vllm_b200 import _native
from lean_vllm_b200._native import check, lib
from lean_vllm_b200.attention.device import call, calls, no_gradient, output_like, raw_stream, stream_of

_INT32_MAX = 2**31 - 1
_DTYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16}


class AttentionWorkspace:
    """Device memory in which the parts of a call's work join. A workspace serves one call at a time, in stream order:
    keep one per stream (and one per captured graph), and pass it to every call there. Allocated and cleared once, on
    the current stream (or `stream`, a cudaStream_t as int)."""

    def __init__(self, device: torch.device | str = "cuda", stream: int | None = None):
        size = lib().kvx_attention_workspace_bytes()
        device = torch.device(device)
        where = torch.cuda.current_stream(device) if stream is None else stream_of(stream, device)
        with torch.cuda.stream(where):
            self.tensor = torch.empty(size, dtype=torch.uint8, device=device)
            self.tensor[: _native.ATTENTION_ZEROED].zero_()
        self.address = self.tensor.data_ptr()
        self.device = self.tensor.device
        self.index = self.tensor.get_device()


def _int32(name: str, t: torch.Tensor, shape: tuple, device: int) -> int:
    if t.dtype != torch.int32 or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor {shape} on the queries' device, not "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _attention(query, k_cache, v_cache, block_tables, kv_lens, scale, q_starts, max_q_len, max_kv_len, softcap, window,
               slopes, prefix_lens, shared_table, shared_len, out, workspace, stream, flags, status):
    if out is None and stream is None and workspace is not None and (native := calls()) is not None:
        done = native.attention(query, k_cache, v_cache, block_tables, kv_lens, scale, q_starts, max_q_len, max_kv_len,
                                softcap, window, slopes, prefix_lens, shared_table, shared_len, workspace.address,
                                workspace.index, flags, status)
        if type(done) is int:
            check(done)
        elif done is not None:
            return done
    no_gradient(query, k_cache, v_cache, slopes)
    shape, cache_shape = query.shape, k_cache.shape
    if len(shape) != 3 or len(cache_shape) != 4 or cache_shape != v_cache.shape:
        raise ValueError(f"queries {tuple(query.shape)} [num_tokens, heads, dim] over caches {tuple(k_cache.shape)} / "
                         f"{tuple(v_cache.shape)} [num_blocks, block_size, heads, dim]")
    num_tokens, q_heads, head_dim = shape
    num_blocks, block_size, kv_heads, cache_dim = cache_shape
    if cache_dim != head_dim or kv_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"{q_heads} query heads of {head_dim} over {kv_heads} KV heads of {cache_dim}")
    dtype, device = query.dtype, query.get_device()
    if dtype not in _DTYPES or not dtype == k_cache.dtype == v_cache.dtype:
        raise TypeError(f"queries and caches must share a dtype, bfloat16 or float16: {dtype}, {k_cache.dtype}, "
                        f"{v_cache.dtype}")
    if not device == k_cache.get_device() == v_cache.get_device():
        raise ValueError("queries and caches must be on one device")
    (q0, q1, q2), strides = query.stride(), k_cache.stride()
    if strides != v_cache.stride() or strides[3] != 1 or q2 != 1:
        raise ValueError("key and value caches must share strides; a head's elements must be contiguous")
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or block_tables.get_device() != device:
        raise ValueError("block tables are an int32 tensor [batch, blocks] on the queries' device")
    batch, max_blocks = block_tables.shape
    table_stride, unit = block_tables.stride()
    if max_blocks > 1 and unit != 1:
        raise ValueError("a sequence's block ids must be contiguous")
    lens = _int32("kv_lens", kv_lens, (batch,), device)
    starts = prefixes = biases = shared = shared_blocks = 0
    if q_starts is not None:
        starts = _int32("q_starts", q_starts, (batch + 1,), device)
    elif num_tokens != batch:
        raise ValueError(f"{num_tokens} query tokens of {batch} sequences: more than one each needs q_starts")
    if prefix_lens is not None:
        prefixes = _int32("prefix_lens", prefix_lens, (batch,), device)
    if slopes is not None:
        if (slopes.dtype != torch.float32 or slopes.get_device() != device or not slopes.is_contiguous()
                or slopes.shape != (q_heads,)):
            raise ValueError(f"slopes are {q_heads} contiguous float32 on the queries' device")
        biases = slopes.data_ptr()
    if shared_table is not None:
        shared_blocks = shared_table.numel()
        shared = _int32("prefix_table", shared_table, (shared_blocks,), device)
    if out is None:
        out = output_like(query, stream)
        o0, o1 = q_heads * head_dim, head_dim
    else:
        o0, o1, o2 = out.stride() if out.dim() == 3 else (0, 0, 0)
        if out.shape != shape or out.dtype != dtype or out.get_device() != device or o2 != 1:
            raise ValueError("`out` must have the queries' shape, dtype and device, a head's elements contiguous")
    if workspace is None:
        workspace = AttentionWorkspace(query.device, stream)  # on the launch's stream, and freed there
    elif workspace.index != device:
        raise ValueError("the workspace must be on the queries' device")
    args = _native.ATTENTION_ARGS.pack(
        query.data_ptr(), 2 * q0, 2 * q1, out.data_ptr(), 2 * o0, 2 * o1, k_cache.data_ptr(), v_cache.data_ptr(),
        2 * strides[0], 2 * strides[1], 2 * strides[2], block_tables.data_ptr(), table_stride, lens, starts, biases,
        prefixes, shared, workspace.address, status, shared_len, shared_blocks, block_size, num_blocks, max_blocks, batch,
        num_tokens, q_heads, kv_heads, head_dim, _DTYPES[dtype], min(max_q_len, _INT32_MAX),
        min(max_blocks * block_size if max_kv_len is None else max_kv_len, _INT32_MAX), window,
        head_dim**-0.5 if scale is None else scale, softcap)
    call(device, lib().kvx_attention, args, flags, raw_stream(device) if stream is None else stream)
    return out


def paged_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    kv_lens: torch.Tensor, *, scale: float | None = None, q_starts: torch.Tensor | None = None,
                    max_q_len: int = 1, max_kv_len: int | None = None, softcap: float = 0.0, window: int = 0,
                    slopes: torch.Tensor | None = None, prefix_lens: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, workspace: AttentionWorkspace | None = None,
                    stream: int | None = None, flags: int = 0, status: int = 0) -> torch.Tensor:
    """Attention of queries [num_tokens, heads, dim] over [num_blocks, block_size, kv_heads, dim] caches (HND caches by
    their transposed view), through int32 `block_tables` [batch, blocks] and `kv_lens` [batch] (cached tokens, the
    query's own included). One query token per sequence, or those from q_starts[s] to q_starts[s + 1] (int32,
    [batch + 1]), of which the last stands at the sequence's last position. Query tokens of no sequence get no defined output.

    A row sees the keys up to its own position; with `window`, only the last `window` of them; with `prefix_lens` (int32
    [batch]), also every key below its sequence's, whatever its position. Scores are `scale` (1/sqrt(dim)) times q.k,
    capped to softcap * tanh(score / softcap) when `softcap` is given, plus slopes[head] * (key - query position) when
    `slopes` (float32 [heads]) are. A row that sees nothing gets zeros. Cache rows past a sequence's length, ahead of its
    first row's window and between a prefix and that window are never used, whatever they or the table there hold. A value
    that one row sees must be finite for the rows beside it too (they multiply it by zero).

    `max_q_len` and `max_kv_len` bound the lengths (the device holds them): they choose the launch's shape only. Without
    q_starts `max_q_len` means nothing.
    `flags` may be STORE_SERIAL: plain launches, no overlap with the kernel before.
    `status` (a StatusWord's address) gets bit 2 for a block id outside the cache, which reads as zeros, or a length past
    its table, which is cut to it."""
    return _attention(query, k_cache, v_cache, block_tables, kv_lens, scale, q_starts, max_q_len, max_kv_len, softcap,
                      window, slopes, prefix_lens, None, 0, out, workspace, stream, flags, status)


def shared_prefix_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_len: int, block_tables: torch.Tensor,
                            kv_lens: torch.Tensor, *, scale: float | None = None,
                            q_starts: torch.Tensor | None = None, max_q_len: int = 1, max_kv_len: int | None = None,
                            softcap: float = 0.0, slopes: torch.Tensor | None = None,
                            out: torch.Tensor | None = None, workspace: AttentionWorkspace | None = None,
                            stream: int | None = None, flags: int = 0, status: int = 0) -> torch.Tensor:
    """paged_attention for sequences that all begin with the same `prefix_len` cached tokens, in the blocks of
    `prefix_table` (int32): `block_tables` and `kv_lens` hold each sequence's own tokens behind it (the query's
    included), which begin in a block of their own. Every row sees the whole prefix and its sequence's own keys up to
    its position. With up to 128 query rows a sequence and KV head (`max_q_len` times the query heads of one) and blocks of
    a multiple of 8 tokens, the prefix is read once for the batch (once for every 65,536 rows of it, where it has more),
    not once per sequence; behind prompts, for each of their tiles of rows."""
    if prefix_len < 0:
        raise ValueError(f"a prefix of {prefix_len} tokens")
    return _attention(query, k_cache, v_cache, block_tables, kv_lens, scale, q_starts, max_q_len, max_kv_len, softcap,
                      0, slopes, None, prefix_table, prefix_len, out, workspace, stream, flags, status)


__all__ = ["AttentionWorkspace", "paged_attention", "shared_prefix_attention"]
