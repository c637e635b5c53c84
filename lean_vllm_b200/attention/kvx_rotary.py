"""Norm, rotation by position and the paged cache store as one sm_100a kernel (kvx_rotate_store).

What an attention layer does to a step's rows between its projections and its attention: each query and key head's
norm (where the model has one), the rotation of its pairs by the token's position, and store_kvcache -- here in one
pass over the rows, with the store's slots, padding, layouts and pushes to decode ranks (PushTarget) unchanged.
`rotate_store_latents` is the same for a latent-attention model's cached rows, [normed part | rotated part], and the
rotated part of its queries. Computed in 32 bits and rounded once. There is no fallback: without libkvx.so the calls
raise.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from lean_vllm_b200 import _native
from lean_vllm_b200._native import RotateArgs, RotateRows, StoreDest, check, lib
from lean_vllm_b200.attention.kvx_cache import PushTarget, _dest, _slots, _target_slots

_DTYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16}


@dataclass
class RotaryTable:
    """The angles of every position: `table` is a float32 device tensor [positions, rotary_dim], the cos of each of a
    position's rotary_dim / 2 angles, then their sin. Pairs are elements (2p, 2p + 1) when `interleaved`, else
    (p, p + rotary_dim / 2). A rotary_dim below the head's rotates its leading elements and leaves the rest."""

    table: torch.Tensor
    interleaved: bool = False

    def __post_init__(self):
        t = self.table
        if t.dim() != 2 or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("a rotary table is a contiguous float32 tensor [positions, rotary_dim]")
        if t.size(0) < 1 or t.size(1) % 2:
            raise ValueError(f"a rotary table of {t.size(0)} positions and rotary_dim {t.size(1)}")

    @classmethod
    def build(cls, positions: int, rotary_dim: int, base: float = 10000.0, interleaved: bool = False,
              scaling: dict | None = None, device="cuda") -> "RotaryTable":
        """The table of angles position * base ** (-2p / rotary_dim), computed in 64 bits. `scaling` stretches it for
        contexts longer than the model was trained on, by `factor`:

        - {"type": "linear", "factor"}: positions divided by factor;
        - {"type": "ntk", "factor"}: base times factor ** (rotary_dim / (rotary_dim - 2)), which leaves the fastest
          pair alone and slows the slowest by factor;
        - {"type": "yarn", "factor", "original_positions", "fast" (32), "slow" (1), "magnitude"}: pairs that turn more
          than `fast` times over original_positions stay, those that turn less than `slow` times are divided by
          factor, a ramp between them, and cos and sin are multiplied by `magnitude` (0.1 ln(factor) + 1).
        """
        if positions < 1 or rotary_dim < 2 or rotary_dim % 2:
            raise ValueError(f"a rotary table of {positions} positions and rotary_dim {rotary_dim}")
        pairs = torch.arange(rotary_dim // 2, dtype=torch.float64)
        magnitude = 1.0
        kind = scaling["type"] if scaling else None
        factor = float(scaling["factor"]) if scaling else 1.0
        if factor < 1.0:
            raise ValueError(f"a scaling factor of {factor}: contexts are stretched, not shrunk")
        if kind == "ntk" and rotary_dim > 2:
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        speed = base ** (-2.0 * pairs / rotary_dim)  # radians a position
        if kind == "linear":
            speed = speed / factor
        elif kind == "yarn":
            original = scaling["original_positions"]

            def pair_turning(turns):  # the (fractional) pair that turns this often over the original context
                return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

            low = max(math.floor(pair_turning(scaling.get("fast", 32))), 0)
            high = min(math.ceil(pair_turning(scaling.get("slow", 1))), rotary_dim - 1)
            ramp = ((pairs - low) / max(high - low, 0.001)).clamp(0, 1)
            speed = speed * (1 - ramp) + speed / factor * ramp
            magnitude = scaling.get("magnitude", 0.1 * math.log(factor) + 1.0)
        elif kind not in (None, "ntk"):
            raise ValueError(f"unknown rotary scaling {kind!r}, expected 'linear', 'ntk' or 'yarn'")
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * speed
        table = torch.cat([angle.cos(), angle.sin()], 1) * magnitude
        return cls(table.float().to(device), interleaved)


def _positions(positions: torch.Tensor, num_tokens: int, device) -> torch.Tensor:
    if positions.numel() != num_tokens:
        raise ValueError(f"{positions.numel()} positions for {num_tokens} rows")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions are int32 or int64, not {positions.dtype}")
    if positions.device != device or not positions.is_contiguous():
        raise ValueError("positions must be contiguous on the storing device")
    return positions


def _rows(x: torch.Tensor, weight, norm_dim: int, rotary_first: int) -> RotateRows:
    if weight is None:
        norm_dim = 0
    elif weight.dtype != x.dtype or weight.numel() != norm_dim or weight.device != x.device or not weight.is_contiguous():
        raise ValueError(f"a norm's weight is {norm_dim} contiguous elements of the rows' dtype on their device")
    if x.stride(-1) != 1:
        raise ValueError("a head's elements must be contiguous")
    size = x.element_size()
    head_stride, heads = (x.stride(1) * size, x.size(1)) if x.dim() == 3 else (0, 1)
    return RotateRows(x.data_ptr(), x.stride(0) * size, head_stride, heads, x.size(-1), norm_dim, rotary_first,
                      weight.data_ptr() if norm_dim else None)


def _launch(rows, out, rotary, positions, num_tokens, dtype, eps, dests, stream, flags, status, device):
    query, key, value = rows
    table = rotary.table
    if table.device != device:
        raise ValueError("the rotary table must be on the storing device")
    size = 2
    args = RotateArgs(query, key, value, out.data_ptr() if out is not None else None,
                      out.stride(0) * size if out is not None else 0, out.stride(1) * size if out is not None else 0,
                      table.data_ptr(), positions.data_ptr(), table.size(0), table.size(1), int(rotary.interleaved),
                      positions.element_size(), num_tokens, dtype, eps, 0)
    array = (StoreDest * len(dests))(*dests)
    s = stream if stream is not None else torch.cuda.current_stream(device).cuda_stream
    check(lib().kvx_rotate_store(args, array, len(dests), status or None, flags, s))


def _output(query, out, stream):
    if out is None:
        if stream is not None and query.is_cuda:  # the caching allocator has to know who writes it
            out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
            out.record_stream(torch.cuda.ExternalStream(stream, query.device))
            return out
        return torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or out.stride(-1) != 1:
        raise ValueError("`out` must have the queries' shape, dtype and device, a head's elements contiguous")
    return out


def rotate_store_kvcache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
                         rotary: RotaryTable, *, q_weight: torch.Tensor | None = None,
                         k_weight: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None,
                         push_to=(), stream: int | None = None, flags: int = 0, status: int = 0) -> torch.Tensor:
    """Norms (with `q_weight` / `k_weight`) and rotates queries and keys [num_tokens, heads, dim], stores keys and
    values into [num_blocks, block_size, heads, dim] caches by `slot_mapping` (as store_kvcache, `push_to` and
    `status` too) and returns the queries, in `out` when given (which may be `query` itself). Rows may be strided over
    tokens and heads (views into a fused qkv product). A position outside the table takes its nearest row and sets bit
    8 of `status`."""
    if query.dim() != 3 or key.dim() != 3:
        raise ValueError("queries, keys and values are [num_tokens, heads, dim]")
    num_tokens, num_heads, head_dim = key.shape
    if value.shape != key.shape or k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"keys {tuple(key.shape)} and values {tuple(value.shape)} into caches "
                         f"{tuple(k_cache.shape)} / {tuple(v_cache.shape)}: shapes must match")
    if k_cache.size(2) != num_heads or k_cache.size(3) != head_dim:
        raise ValueError(f"{num_heads} heads of {head_dim} into a cache of {k_cache.size(2)} heads of "
                         f"{k_cache.size(3)}")
    if query.size(0) != num_tokens or query.size(2) != head_dim:
        raise ValueError(f"queries {tuple(query.shape)} beside keys {tuple(key.shape)}")
    dtype = query.dtype
    if dtype not in _DTYPES or not dtype == key.dtype == value.dtype == k_cache.dtype == v_cache.dtype:
        raise TypeError(f"queries, keys, values and caches must share a dtype, bfloat16 or float16: {dtype}, "
                        f"{key.dtype}, {value.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    device = query.device
    if not device == key.device == value.device == k_cache.device == v_cache.device:
        raise ValueError("queries, keys, values and the local caches must be on one device")
    strides = k_cache.stride()
    if strides != v_cache.stride() or strides[3] != 1:
        raise ValueError("key and value caches must share strides with contiguous head_dim")
    if rotary.table.size(1) > head_dim:
        raise ValueError(f"a rotary table of {rotary.table.size(1)} elements for heads of {head_dim}")
    if len(push_to) > 8:
        raise ValueError("at most 8 peers per store")
    slots = _slots(slot_mapping, num_tokens, device)
    _positions(positions, num_tokens, device)
    rows = (_rows(query, q_weight, head_dim, 0), _rows(key, k_weight, head_dim, 0), _rows(value, None, 0, 0))
    dests = [_dest(k_cache.data_ptr(), v_cache.data_ptr(), strides[0] * 2, strides[1] * 2, strides[2] * 2,
                   k_cache.size(1), k_cache.size(0), slots, 0, num_heads, 0)]
    for target in push_to:
        t_slots = _target_slots(target, num_tokens, device)
        count = num_heads - target.src_first_head if target.num_heads is None else target.num_heads
        dests.append(_dest(target.k_cache, target.v_cache, target.block_stride, target.token_stride,
                           target.head_stride, target.block_size, target.num_blocks, t_slots, target.src_first_head,
                           count, target.dst_first_head, target.block_map))
    out = _output(query, out, stream)
    _launch(rows, out, rotary, positions, num_tokens, _DTYPES[dtype], eps, dests, stream, flags, status, device)
    return out


def rotate_store_latents(latent: torch.Tensor, latent_cache: torch.Tensor, slot_mapping: torch.Tensor,
                         positions: torch.Tensor, rotary: RotaryTable, *, query_pe: torch.Tensor | None = None,
                         weight: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None,
                         push_to=(), stream: int | None = None, flags: int = 0,
                         status: int = 0) -> torch.Tensor | None:
    """Stores latents [num_tokens, rank + rotary_dim] into a [num_blocks, block_size, rank + rotary_dim] cache by
    `slot_mapping` (as store_latents), the leading `rank` elements normed with `weight` (where given) and the last
    rotary_dim rotated, and returns the queries' rotated part `query_pe` [num_tokens, heads, rotary_dim] rotated, in
    `out` when given (None without queries)."""
    if latent.dim() != 2 or latent_cache.dim() != 3 or latent_cache.size(2) != latent.size(1):
        raise ValueError(f"latents {tuple(latent.shape)} into a cache {tuple(latent_cache.shape)}")
    num_tokens, dim = latent.shape
    rotary_dim = rotary.table.size(1)
    if rotary_dim > dim:
        raise ValueError(f"a rotary table of {rotary_dim} elements for latents of {dim}")
    dtype, device = latent.dtype, latent.device
    if dtype not in _DTYPES or dtype != latent_cache.dtype or (query_pe is not None and query_pe.dtype != dtype):
        raise TypeError(f"latents, queries and cache must share a dtype, bfloat16 or float16: {dtype}, "
                        f"{latent_cache.dtype}")
    if device != latent_cache.device or (query_pe is not None and query_pe.device != device):
        raise ValueError("latents, queries and the local cache must be on one device")
    if latent_cache.stride(-2) != dim or latent_cache.stride(-1) != 1:
        raise ValueError("cache tokens must be contiguous")
    if query_pe is not None and (query_pe.dim() != 3 or query_pe.size(0) != num_tokens or query_pe.size(2) != rotary_dim):
        raise ValueError(f"queries' rotated part {tuple(query_pe.shape)} for {num_tokens} rows of {rotary_dim}")
    if len(push_to) > 8:
        raise ValueError("at most 8 peers per store")
    slots = _slots(slot_mapping, num_tokens, device)
    _positions(positions, num_tokens, device)
    rank = dim - rotary_dim
    rows = (_rows(query_pe, None, 0, 0) if query_pe is not None else RotateRows(),
            _rows(latent, weight, rank, rank), RotateRows())
    dests = [_dest(latent_cache.data_ptr(), 0, latent_cache.stride(0) * 2, dim * 2, 0, latent_cache.size(1),
                   latent_cache.size(0), slots, 0, 1, 0)]
    for target in push_to:
        t_slots = _target_slots(target, num_tokens, device)
        dests.append(_dest(target.k_cache, 0, target.block_stride, target.token_stride, 0, target.block_size,
                           target.num_blocks, t_slots, 0, 1, 0, target.block_map))
    if query_pe is not None:
        out = _output(query_pe, out, stream)
    else:
        out = None
    _launch(rows, out, rotary, positions, num_tokens, _DTYPES[dtype], eps, dests, stream, flags, status, device)
    return out


__all__ = ["PushTarget", "RotaryTable", "rotate_store_kvcache", "rotate_store_latents"]
