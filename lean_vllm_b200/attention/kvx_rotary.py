"""Norm, rotation by position and the paged cache store as one sm_100a kernel (kvx_rotate_store).

What an attention layer does to a step's rows between its projections and its attention: each query and key head's
norm (where the model has one), the rotation of its pairs by the token's position, and store_kvcache -- here in one
pass over the rows, with the store's slots, padding, layouts and pushes to decode ranks (PushTarget) unchanged.
`rotate_store_latents` is the same for a latent-attention model's cached rows, [normed part | rotated part], and the
rotated part of its queries. Computed in 32 bits and rounded once. For serving: inputs that require a gradient are refused
while gradients are recorded. There is no fallback: without libkvx.so the calls raise.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from lean_vllm_b200 import _native
from lean_vllm_b200._native import check, lib
from lean_vllm_b200.attention.device import call, calls, no_gradient, output_like, raw_stream
from lean_vllm_b200.attention.kvx_cache import PushTarget, _dest, _slots, _target_slots

_DTYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}


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


def _positions(positions: torch.Tensor, num_tokens: int, device: int) -> int:
    """The positions' element size, after checking them."""
    if positions.numel() != num_tokens:
        raise ValueError(f"{positions.numel()} positions for {num_tokens} rows")
    size = _INDEX_BYTES.get(positions.dtype)
    if size is None:
        raise TypeError(f"positions are int32 or int64, not {positions.dtype}")
    if positions.get_device() != device or not positions.is_contiguous():
        raise ValueError("positions must be contiguous on the storing device")
    return size


def _weight(weight: torch.Tensor | None, dim: int, dtype, device: int) -> tuple[int, int]:
    """(normed elements, address) of a norm's weight."""
    if weight is None:
        return 0, 0
    if weight.dtype != dtype or weight.numel() != dim or weight.get_device() != device or not weight.is_contiguous():
        raise ValueError(f"a norm's weight is {dim} contiguous elements of the rows' dtype on their device")
    return dim, weight.data_ptr()


_NO_ROWS = (0, 0, 0, 0, 0, 0, 0, 0)


def _dests(k_addr: int, v_addr: int, strides: tuple, block_size: int, num_blocks: int, slots: torch.Tensor, heads: int,
           push_to, num_tokens: int, device) -> bytes:
    packed = _native.STORE_DEST.pack(k_addr, v_addr, *strides, block_size, num_blocks, slots.data_ptr(),
                                     _INDEX_BYTES[slots.dtype], 0, heads, 0, 0, 0, 0)
    for target in push_to:
        t_slots = _target_slots(target, num_tokens, device)
        count = heads - target.src_first_head if target.num_heads is None else target.num_heads
        dest = _dest(target.k_cache, target.v_cache if v_addr else 0, target.block_stride, target.token_stride,
                     target.head_stride if v_addr else 0, target.block_size, target.num_blocks, t_slots,
                     target.src_first_head if v_addr else 0, count if v_addr else 1,
                     target.dst_first_head if v_addr else 0, target.block_map)
        packed += bytes(dest)
    return packed


def _launch(rows: tuple, out, rotary: RotaryTable, positions: torch.Tensor, position_bytes: int, num_tokens: int, dtype,
            eps: float, dests: bytes, stream, flags: int, status: int, device: int) -> None:
    table = rotary.table
    if table.get_device() != device:
        raise ValueError("the rotary table must be on the storing device")
    if out is not None:
        o0, o1, _ = out.stride()
        to = (out.data_ptr(), 2 * o0, 2 * o1)
    else:
        to = (0, 0, 0)
    table_rows, rotary_dim = table.shape
    args = _native.ROTATE_ARGS.pack(*rows, *to, table.data_ptr(), positions.data_ptr(), table_rows, rotary_dim,
                                    rotary.interleaved, position_bytes, num_tokens, _DTYPES[dtype], eps, 0)
    s = raw_stream(device) if stream is None else stream
    call(device, lib().kvx_rotate_store, args, dests, len(dests) // _native.STORE_DEST.size, status or None, flags, s)


def _output(query: torch.Tensor, out: torch.Tensor | None, stream: int | None) -> torch.Tensor:
    if out is None:
        return output_like(query, stream)
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or out.stride(-1) != 1:
        raise ValueError("`out` must have the queries' shape, dtype and device, a head's elements contiguous")
    return out


def rotate_store_kvcache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
                         rotary: RotaryTable, *, q_weight: torch.Tensor | None = None,
                         k_weight: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None,
                         push_to=(), stream: int | None = None, flags: int = 0,
                         status: int = 0) -> torch.Tensor | None:
    """Norms (with `q_weight` / `k_weight`) and rotates queries and keys [num_tokens, heads, dim], stores keys and
    values into [num_blocks, block_size, heads, dim] caches by `slot_mapping` (as store_kvcache, `push_to` and
    `status` too) and returns the queries, in `out` when given (which may be `query` itself). Rows may be strided over
    tokens and heads (views into a fused qkv product). A position outside the table takes its nearest row and sets bit
    8 of `status`. With STORE_PEERS_ONLY in `flags`, the push half of a store whose local half came before, only the
    peers are written: the queries are left alone, and `out` is returned as it is (None without one)."""
    push_half = flags & _native.STORE_PEERS_ONLY
    if out is None and stream is None and not push_to and not push_half and (native := calls()) is not None:
        done = native.rotate_store(query, key, value, k_cache, v_cache, slot_mapping, positions, rotary.table,
                                   rotary.interleaved, q_weight, k_weight, eps, flags, status)
        if type(done) is int:
            check(done)
        elif done is not None:
            return done
    no_gradient(query, key, value, q_weight, k_weight, rotary.table)
    if query.dim() != 3 or key.dim() != 3:
        raise ValueError("queries, keys and values are [num_tokens, heads, dim]")
    num_tokens, num_heads, head_dim = key.shape
    cache_shape, dtype, device = k_cache.shape, query.dtype, query.get_device()
    if value.shape != key.shape or len(cache_shape) != 4 or cache_shape != v_cache.shape:
        raise ValueError(f"keys {tuple(key.shape)} and values {tuple(value.shape)} into caches "
                         f"{tuple(k_cache.shape)} / {tuple(v_cache.shape)}: shapes must match")
    num_blocks, block_size, cache_heads, cache_dim = cache_shape
    if cache_heads != num_heads or cache_dim != head_dim:
        raise ValueError(f"{num_heads} heads of {head_dim} into a cache of {cache_heads} heads of {cache_dim}")
    q_tokens, q_heads, q_dim = query.shape
    if q_tokens != num_tokens or q_dim != head_dim:
        raise ValueError(f"queries {tuple(query.shape)} beside keys {tuple(key.shape)}")
    if dtype not in _DTYPES or not dtype == key.dtype == value.dtype == k_cache.dtype == v_cache.dtype:
        raise TypeError(f"queries, keys, values and caches must share a dtype, bfloat16 or float16: {dtype}, "
                        f"{key.dtype}, {value.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    if not device == key.get_device() == value.get_device() == k_cache.get_device() == v_cache.get_device():
        raise ValueError("queries, keys, values and the local caches must be on one device")
    (q0, q1, q2), (k0, k1, k2), (v0, v1, v2) = query.stride(), key.stride(), value.stride()
    if q2 != 1 or k2 != 1 or v2 != 1:
        raise ValueError("a head's elements must be contiguous")
    strides = k_cache.stride()
    if strides != v_cache.stride() or strides[3] != 1:
        raise ValueError("key and value caches must share strides with contiguous head_dim")
    if rotary.table.size(1) > head_dim:
        raise ValueError(f"a rotary table of {rotary.table.size(1)} elements for heads of {head_dim}")
    if len(push_to) > 8:
        raise ValueError("at most 8 peers per store")
    slots = _slots(slot_mapping, num_tokens, key.device)
    position_bytes = _positions(positions, num_tokens, device)
    q_norm, q_scale = _weight(q_weight, head_dim, dtype, device)
    k_norm, k_scale = _weight(k_weight, head_dim, dtype, device)
    rows = (query.data_ptr(), 2 * q0, 2 * q1, q_heads, head_dim, q_norm, 0, q_scale,
            key.data_ptr(), 2 * k0, 2 * k1, num_heads, head_dim, k_norm, 0, k_scale,
            value.data_ptr(), 2 * v0, 2 * v1, num_heads, head_dim, 0, 0, 0)
    dests = _dests(k_cache.data_ptr(), v_cache.data_ptr(), (2 * strides[0], 2 * strides[1], 2 * strides[2]), block_size,
                   num_blocks, slots, num_heads, push_to, num_tokens, key.device)
    if out is not None or not push_half:
        out = _output(query, out, stream)
    _launch(rows, out, rotary, positions, position_bytes, num_tokens, dtype, eps, dests, stream, flags, status, device)
    return out


def rotate_store_latents(latent: torch.Tensor, latent_cache: torch.Tensor, slot_mapping: torch.Tensor,
                         positions: torch.Tensor, rotary: RotaryTable, *, query_pe: torch.Tensor | None = None,
                         weight: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None,
                         push_to=(), stream: int | None = None, flags: int = 0,
                         status: int = 0) -> torch.Tensor | None:
    """Stores latents [num_tokens, rank + rotary_dim] into a [num_blocks, block_size, rank + rotary_dim] cache by
    `slot_mapping` (as store_latents), the leading `rank` elements normed with `weight` (where given) and the last
    rotary_dim rotated, and returns the queries' rotated part `query_pe` [num_tokens, heads, rotary_dim] rotated, in
    `out` when given (None without queries). STORE_PEERS_ONLY in `flags` as for rotate_store_kvcache."""
    push_half = flags & _native.STORE_PEERS_ONLY
    if out is None and stream is None and not push_to and not push_half and (native := calls()) is not None:
        done = native.rotate_latents(latent, latent_cache, slot_mapping, positions, rotary.table, rotary.interleaved,
                                     query_pe, weight, eps, flags, status)
        if type(done) is int:
            check(done)
        elif done is not None:
            return done if query_pe is not None else None
    no_gradient(latent, query_pe, weight, rotary.table)
    if latent.dim() != 2 or latent_cache.dim() != 3 or latent_cache.size(2) != latent.size(1):
        raise ValueError(f"latents {tuple(latent.shape)} into a cache {tuple(latent_cache.shape)}")
    num_tokens, dim = latent.shape
    num_blocks, block_size, _ = latent_cache.shape
    rotary_dim = rotary.table.size(1)
    if rotary_dim > dim:
        raise ValueError(f"a rotary table of {rotary_dim} elements for latents of {dim}")
    dtype, device = latent.dtype, latent.get_device()
    if dtype not in _DTYPES or dtype != latent_cache.dtype or (query_pe is not None and query_pe.dtype != dtype):
        raise TypeError(f"latents, queries and cache must share a dtype, bfloat16 or float16: {dtype}, "
                        f"{latent_cache.dtype}")
    if device != latent_cache.get_device() or (query_pe is not None and query_pe.get_device() != device):
        raise ValueError("latents, queries and the local cache must be on one device")
    block_stride, token_stride, unit = latent_cache.stride()
    if token_stride != dim or unit != 1:
        raise ValueError("cache tokens must be contiguous")
    l0, l1 = latent.stride()
    if l1 != 1:
        raise ValueError("a latent's elements must be contiguous")
    if len(push_to) > 8:
        raise ValueError("at most 8 peers per store")
    slots = _slots(slot_mapping, num_tokens, latent.device)
    position_bytes = _positions(positions, num_tokens, device)
    rank = dim - rotary_dim
    normed, scale = _weight(weight, rank, dtype, device)
    if query_pe is not None:
        if query_pe.dim() != 3 or query_pe.size(0) != num_tokens or query_pe.size(2) != rotary_dim:
            raise ValueError(f"queries' rotated part {tuple(query_pe.shape)} for {num_tokens} rows of {rotary_dim}")
        q0, q1, q2 = query_pe.stride()
        if q2 != 1:
            raise ValueError("a head's elements must be contiguous")
        query = (query_pe.data_ptr(), 2 * q0, 2 * q1, query_pe.size(1), rotary_dim, 0, 0, 0)
        if out is not None or not push_half:
            out = _output(query_pe, out, stream)
    else:
        query, out = _NO_ROWS, None
    rows = (*query, latent.data_ptr(), 2 * l0, 0, 1, dim, normed, rank, scale, *_NO_ROWS)
    dests = _dests(latent_cache.data_ptr(), 0, (2 * block_stride, 2 * dim, 0), block_size, num_blocks, slots, 1, push_to,
                   num_tokens, latent.device)
    _launch(rows, out, rotary, positions, position_bytes, num_tokens, dtype, eps, dests, stream, flags, status, device)
    return out


__all__ = ["PushTarget", "RotaryTable", "rotate_store_kvcache", "rotate_store_latents"]
