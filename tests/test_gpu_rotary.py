"""kvx_rotate_store on the GPU: norm, rotation and store against the definition in 64 bits, what it leaves alone bit
for bit, and what it flags."""

import pytest
import torch

from lean_vllm_b200._native import STORE_PEERS_ONLY
from lean_vllm_b200.attention.kvx_cache import PushTarget, store_kvcache, store_latents
from lean_vllm_b200.attention.kvx_rotary import RotaryTable, rotate_store_kvcache, rotate_store_latents
from lean_vllm_b200.kv_transfer import transport
from tests.attention_cases import check_rotated, rotate64

pytestmark = pytest.mark.gpu


def rows_case(tokens, q_heads, kv_heads, dim, rotary, block, dtype, hnd=True, fused=True, seed=0, norm=True,
              slot_dtype=torch.int64, positions=512):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if fused:
        q, k, v = randn(tokens, q_heads + 2 * kv_heads, dim).to(dtype).split([q_heads, kv_heads, kv_heads], 1)
    else:
        q, k, v = (randn(tokens, n, dim).to(dtype) for n in (q_heads, kv_heads, kv_heads))
    blocks = -(-tokens // block) + 2
    cache = randn(*((2, blocks, kv_heads, block, dim) if hnd else (2, blocks, block, kv_heads, dim))).to(dtype)
    slots = torch.randperm(blocks * block, generator=g, device="cuda")[:tokens].to(slot_dtype)
    slots[3::11] = -1
    table = RotaryTable.build(positions, rotary, base=1e4) if rotary else RotaryTable(torch.zeros(1, 0, device="cuda"))
    at = torch.randint(0, positions, (tokens,), generator=g, device="cuda").to(slot_dtype)
    weights = [(1 + 0.3 * randn(dim)).to(dtype) if norm else None for _ in range(2)]
    return q, k, v, cache, slots, table, at, weights


def expected_cache(before, rows, slots, hnd):
    """The cache with `rows` in their slots, for comparing whole: (blocks, block, heads, dim)."""
    out = before.double().clone()
    keep = slots >= 0
    s = slots[keep].long()
    out[s // before.size(1), s % before.size(1)] = rows[keep]
    return out


def check_case(q, k, v, cache, slots, table, at, weights, hnd, interleaved, **more):
    table = RotaryTable(table.table, interleaved)
    dim = q.size(2)
    view = cache.transpose(2, 3) if hnd else cache
    before = view.clone()
    want_q, size_q = rotate64(q, weights[0], dim, 0, table.table, at, interleaved)
    want_k, size_k = rotate64(k, weights[1], dim, 0, table.table, at, interleaved)
    word = transport.StatusWord()
    out = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0], k_weight=weights[1],
                               status=word.address, **more)
    torch.cuda.synchronize()
    assert word.bits() == 0
    word.close()
    check_rotated(out, want_q, size_q)
    check_rotated(view[0], expected_cache(before[0], want_k, slots, hnd), expected_cache(before[0].abs(), size_k, slots, hnd))
    keep = slots >= 0
    want_v = before[1].clone()
    s = slots[keep].long()
    want_v[s // view.size(2), s % view.size(2)] = v[keep]
    assert torch.equal(view[1], want_v)
    untouched = torch.ones(view.size(1) * view.size(2), dtype=torch.bool, device="cuda")
    untouched[s] = False
    assert torch.equal(view[0].flatten(0, 1)[untouched], before[0].flatten(0, 1)[untouched])
    return out


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens, q_heads, kv_heads, dim, rotary, block, dtype, hnd, fused, norm", [
    (1, 32, 8, 128, 128, 256, torch.bfloat16, True, True, True),      # one decoded token
    (1, 1, 1, 64, 64, 16, torch.float16, True, False, False),         # the least there is
    (333, 8, 2, 128, 128, 64, torch.bfloat16, True, True, True),
    (97, 14, 2, 64, 32, 24, torch.float16, False, True, False),       # part of the head, block size not a power of two
    (50, 7, 1, 128, 32, 16, torch.bfloat16, False, False, True),      # a quarter of the head
    (40, 5, 5, 64, 64, 256, torch.bfloat16, True, False, True),       # no grouping, odd head count
    (29, 4, 2, 80, 80, 16, torch.bfloat16, True, True, True),         # a width no variant is made for
    (31, 3, 3, 12, 6, 16, torch.float16, True, True, True),           # rows of 24 bytes, 3 pairs
    (17, 2, 1, 128, 100, 16, torch.bfloat16, False, True, True),      # 50 pairs: their halves not on vector bounds
    (19, 4, 1, 256, 64, 16, torch.float16, True, True, True),
    (23, 4, 2, 128, 0, 16, torch.bfloat16, True, True, True),         # norms alone
])
def test_rows_are_normed_rotated_and_stored(tokens, q_heads, kv_heads, dim, rotary, block, dtype, hnd, fused, norm,
                                            interleaved):
    case = rows_case(tokens, q_heads, kv_heads, dim, rotary, block, dtype, hnd, fused, seed=tokens, norm=norm,
                     slot_dtype=torch.int32 if tokens % 2 else torch.int64)
    check_case(*case, hnd=hnd, interleaved=interleaved)


def test_many_tokens_are_the_same_as_few():
    """More rows than one wave of CTAs holds, and one token at a time: the same bits."""
    q, k, v, cache, slots, table, at, weights = rows_case(3001, 16, 4, 128, 128, 64, torch.bfloat16)
    out = check_case(q, k, v, cache, slots, table, at, weights, hnd=True, interleaved=False)
    again = torch.zeros_like(cache)
    view = again.transpose(2, 3)
    for t in range(0, 3001, 750):
        one = rotate_store_kvcache(q[t : t + 1], k[t : t + 1], v[t : t + 1], view[0], view[1], slots[t : t + 1],
                                   at[t : t + 1], table, q_weight=weights[0], k_weight=weights[1])
        assert torch.equal(one, out[t : t + 1])
        if slots[t] >= 0:
            s = int(slots[t])
            assert torch.equal(view[0, s // 64, s % 64], cache.transpose(2, 3)[0, s // 64, s % 64])


def test_queries_can_be_rotated_in_place_and_into_a_strided_output():
    q, k, v, cache, slots, table, at, weights = rows_case(65, 6, 2, 64, 64, 16, torch.bfloat16, fused=False)
    view = cache.transpose(2, 3)
    want = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0], k_weight=weights[1])
    wide = torch.zeros(65, 9, 64, dtype=q.dtype, device="cuda")
    got = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0], k_weight=weights[1],
                               out=wide[:, 2:8])
    assert got.data_ptr() == wide[:, 2:8].data_ptr() and torch.equal(wide[:, 2:8], want)
    assert not wide[:, :2].any() and not wide[:, 8:].any()
    same = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0], k_weight=weights[1],
                                out=q)
    assert same.data_ptr() == q.data_ptr() and torch.equal(q, want)


def test_rows_that_begin_off_vector_bounds_are_the_same_as_aligned_ones():
    """A head's rows two bytes past a 16-byte boundary, and a cache whose rows are: only the access width differs."""
    q, k, v, cache, slots, table, at, weights = rows_case(37, 4, 2, 128, 128, 16, torch.bfloat16, fused=False)
    view = cache.transpose(2, 3)
    want = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0], k_weight=weights[1])

    def shifted(x):
        flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
        flat[1:] = x.reshape(-1)
        return flat[1:].view(x.shape)

    odd_cache = shifted(torch.zeros_like(cache))
    odd = odd_cache.transpose(2, 3)
    got = rotate_store_kvcache(shifted(q), shifted(k), shifted(v), odd[0], odd[1], slots, at, table,
                               q_weight=shifted(weights[0]), k_weight=shifted(weights[1]))
    keep = slots[slots >= 0]
    # The sums of squares run in another order: the last bit of the norm's 32 bits may differ, and round another way.
    assert (got.double() - want.double()).abs().max() <= 2.0**-7 * want.abs().max()
    for part in (0, 1):
        a, b = odd[part][keep // 16, keep % 16].double(), view[part][keep // 16, keep % 16].double()
        assert (a - b).abs().max() <= (2.0**-7 * b.abs().max() if part == 0 else 0)


def test_no_tokens_launch_nothing():
    q, k, v, cache, slots, table, at, weights = rows_case(4, 2, 1, 64, 64, 16, torch.bfloat16)
    view = cache.transpose(2, 3)
    before = transport.launch_count()
    out = rotate_store_kvcache(q[:0], k[:0], v[:0], view[0], view[1], slots[:0], at[:0], table)
    assert out.shape == (0, 2, 64) and transport.launch_count() == before


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens, heads, rank, rotary, block, dtype, norm", [
    (1, 16, 512, 64, 64, torch.bfloat16, True),
    (200, 16, 512, 64, 64, torch.float16, True),
    (75, 5, 512, 64, 24, torch.bfloat16, False),
    (33, 3, 96, 32, 16, torch.bfloat16, True),   # a rank no variant is made for
    (20, 0, 512, 64, 64, torch.bfloat16, True),  # no queries
    (9, 2, 256, 6, 16, torch.float16, True),     # 3 pairs
])
def test_latents_are_normed_rotated_and_stored(tokens, heads, rank, rotary, block, dtype, norm, interleaved):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    latent = torch.randn(tokens, rank + rotary, generator=g, device="cuda").to(dtype)
    pe = torch.randn(tokens, heads, 128 + rotary, generator=g, device="cuda").to(dtype)[..., 128:] if heads else None
    blocks = -(-tokens // block) + 2
    cache = torch.randn(blocks, block, rank + rotary, generator=g, device="cuda").to(dtype)
    slots = torch.randperm(blocks * block, generator=g, device="cuda")[:tokens]
    slots[2::9] = -1
    at = torch.randint(0, 300, (tokens,), generator=g, device="cuda")
    table = RotaryTable.build(300, rotary, interleaved=interleaved)
    weight = (1 + 0.3 * torch.randn(rank, generator=g, device="cuda")).to(dtype) if norm else None
    before = cache.clone()
    out = rotate_store_latents(latent, cache, slots, at, table, query_pe=pe, weight=weight)
    torch.cuda.synchronize()
    want, size = rotate64(latent[:, None], weight, rank, rank, table.table, at, interleaved)
    check_rotated(cache, expected_cache(before, want[:, 0], slots, False), expected_cache(before.abs(), size[:, 0], slots, False))
    if heads:
        want_q, size_q = rotate64(pe, None, 0, 0, table.table, at, interleaved)
        check_rotated(out, want_q, size_q)
    else:
        assert out is None


def test_peers_get_the_rotated_heads_they_take():
    """The push of a layer-by-layer transfer: two peers' caches hold, bit for bit, the heads the local cache got; one by
    its own slots, one through a block map that leaves a block out."""
    q, k, v, cache, slots, table, at, weights = rows_case(300, 8, 4, 128, 128, 16, torch.bfloat16, seed=5)
    view = cache.transpose(2, 3)
    peers = [torch.zeros(2, 30, 2, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    peer_slots = torch.randperm(480, device="cuda")[:300]
    block_map = torch.randperm(30, device="cuda")[: view.size(1)].to(torch.int32)
    block_map[2] = -1
    targets = [PushTarget.of(peers[0].transpose(2, 3)[0], peers[0].transpose(2, 3)[1], peer_slots, src_first_head=0,
                             num_heads=2),
               PushTarget.of(peers[1].transpose(2, 3)[0], peers[1].transpose(2, 3)[1], None, src_first_head=2,
                             num_heads=2, block_map=block_map)]
    before = transport.launch_count()
    rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0], k_weight=weights[1],
                         push_to=targets)
    torch.cuda.synchronize()
    assert transport.launch_count() - before == 1
    rows = torch.zeros(2, 300, 4, 128, device="cuda", dtype=torch.bfloat16)
    keep = slots >= 0
    rows[:, keep] = view[:, slots[keep] // 16, slots[keep] % 16]
    # Rows without a local slot still go to the first peer: take them from a store of the same rows elsewhere.
    spare = torch.zeros(2, 19, 16, 4, 128, device="cuda", dtype=torch.bfloat16)
    rotate_store_kvcache(q, k, v, spare[0], spare[1], torch.arange(300, device="cuda"), at, table, q_weight=weights[0],
                         k_weight=weights[1])
    everything = spare.flatten(1, 2)[:, :300]
    assert torch.equal(everything[:, keep], rows[:, keep])
    want = torch.zeros_like(peers[0]).transpose(2, 3)
    want[:, peer_slots // 16, peer_slots % 16] = everything[:, :, :2]
    assert torch.equal(peers[0].transpose(2, 3), want)
    want = torch.zeros_like(peers[1]).transpose(2, 3)
    mapped = torch.where(keep, block_map[(slots // 16).clamp(min=0)].long(), -1)
    ok = mapped >= 0
    want[:, mapped[ok], slots[ok] % 16] = everything[:, ok, 2:]
    assert torch.equal(peers[1].transpose(2, 3), want)


def test_without_norm_or_turn_the_store_is_the_plain_one():
    """At position 0 every angle is 0: what lands is what store_kvcache and store_latents land, bit for bit."""
    q, k, v, cache, slots, table, at, _ = rows_case(123, 8, 4, 128, 128, 16, torch.bfloat16, norm=False)
    other = cache.clone()
    a, b = cache.transpose(2, 3), other.transpose(2, 3)
    out = rotate_store_kvcache(q, k, v, a[0], a[1], slots, torch.zeros_like(at), table)
    store_kvcache(k, v, b[0], b[1], slots)
    assert torch.equal(cache, other) and torch.equal(out, q)
    latent = torch.randn(123, 576, device="cuda").to(torch.bfloat16)
    one, two = torch.zeros(2, cache.size(1), 16, 576, device="cuda", dtype=torch.bfloat16)
    rotate_store_latents(latent, one, slots, torch.zeros_like(at), RotaryTable.build(4, 64))
    store_latents(latent, two, slots)
    assert torch.equal(one, two)


def test_slots_past_the_cache_and_positions_past_the_table_are_flagged():
    q, k, v, cache, slots, table, at, weights = rows_case(64, 4, 2, 128, 128, 16, torch.bfloat16)
    view = cache.transpose(2, 3)
    transport.device_error()
    word = transport.StatusWord()
    slots[10] = view.size(1) * 16
    before = view.clone()
    rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, status=word.address)
    torch.cuda.synchronize()
    assert word.bits() == 2 and transport.device_error() == 2
    word.close()
    s = slots[(slots >= 0) & (slots < view.size(1) * 16)]
    untouched = torch.ones(view.size(1) * 16, dtype=torch.bool, device="cuda")
    untouched[s] = False
    assert torch.equal(view[1].flatten(0, 1)[untouched], before[1].flatten(0, 1)[untouched])
    slots[10] = -1
    at[10] = 10**6  # padding: its position means nothing
    word = transport.StatusWord()
    rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, status=word.address)
    torch.cuda.synchronize()
    assert word.bits() == 0
    for bad, near in ((-5, 0), (512, 511), (10**12, 511)):
        at[1], slots[1] = bad, 1
        out = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, status=word.address)
        torch.cuda.synchronize()
        assert word.bits() == 8 and transport.device_error() == 8
        at[1] = near
        assert torch.equal(out, rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table))
    word.close()


def test_a_cache_past_four_gigabytes_is_addressed_whole():
    """Blocks whose byte offsets pass 2^32, through both kinds of rows."""
    blocks = 9000
    cache = torch.zeros(2, blocks, 8, 256, 128, dtype=torch.bfloat16, device="cuda")  # 2 x 4.7 GB
    view = cache.transpose(2, 3)
    k, v = torch.randn(2, 3, 8, 128, device="cuda").to(torch.bfloat16)
    slots = torch.tensor([blocks * 256 - 1, 0, 8500 * 256 + 7], device="cuda")
    rotate_store_kvcache(k, k, v, view[0], view[1], slots, torch.zeros(3, dtype=torch.int64, device="cuda"),
                         RotaryTable.build(4, 128))
    for t, (b, o) in enumerate([(blocks - 1, 255), (0, 0), (8500, 7)]):
        assert torch.equal(view[0, b, o], k[t]) and torch.equal(view[1, b, o], v[t])
    assert int((view[0].float().abs().amax((-1, -2)) > 0).sum()) == 3


def test_another_stream_runs_the_call_in_its_own_order():
    q, k, v, cache, slots, table, at, weights = rows_case(500, 8, 2, 128, 128, 16, torch.bfloat16)
    view = cache.transpose(2, 3)
    want = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        for _ in range(20):
            late.copy_(q)  # the rows arrive on this stream only
        got = rotate_store_kvcache(late, k, v, view[0], view[1], slots, at, table)
    side.synchronize()
    assert torch.equal(got, want)
    raw = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(raw, want)


def test_an_output_made_for_another_stream_waits_for_nobody():
    """Work still queued on the current stream on memory that was freed there does not reach the queries made for a call on
    another stream (stream 0 among them)."""
    q, k, v, cache, slots, table, at, weights = rows_case(500, 8, 2, 128, 128, 16, torch.bfloat16)
    view = cache.transpose(2, 3)
    want = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table)
    side = torch.cuda.Stream()
    for current, other in ((torch.cuda.current_stream(), side), (side, torch.cuda.default_stream())):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        with torch.cuda.stream(current):
            taken = torch.empty_like(want)
            torch.cuda._sleep(50_000_000)  # tens of ms
            taken.fill_(1)
            del taken
            got = rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, stream=other.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dim, rotary", [(128, 128), (80, 80)], ids=["vector", "any"])
def test_the_push_half_of_a_store_leaves_the_queries_alone(dim, rotary):
    """STORE_PEERS_ONLY: the peers get the rows that the local half stored, the local cache and the queries, rotated by the
    local half (in place, here), stay as they are, and without `out` there are none to return."""
    q, k, v, cache, slots, table, at, weights = rows_case(65, 6, 2, dim, rotary, 16, torch.bfloat16, fused=False)
    view, peer = cache.transpose(2, 3), torch.zeros_like(cache)
    target = PushTarget.of(peer.transpose(2, 3)[0], peer.transpose(2, 3)[1], slots)

    def call(**more):
        return rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, q_weight=weights[0],
                                    k_weight=weights[1], **more)

    call(out=q)
    rotated, local = q.clone(), cache.clone()
    assert call(out=q, push_to=[target], flags=STORE_PEERS_ONLY) is q
    assert call(push_to=[target], flags=STORE_PEERS_ONLY) is None and call(flags=STORE_PEERS_ONLY) is None
    torch.cuda.synchronize()
    assert torch.equal(q, rotated) and torch.equal(cache, local)
    s = slots[slots >= 0]
    assert torch.equal(peer.transpose(2, 3)[:, s // 16, s % 16], view[:, s // 16, s % 16])


@pytest.mark.parametrize("rank, rotary", [(512, 64), (96, 32)], ids=["vector", "any"])
def test_peers_get_the_latents_too_and_the_push_half_alone(rank, rotary):
    g = torch.Generator(device="cuda").manual_seed(7)
    latent = torch.randn(90, rank + rotary, generator=g, device="cuda").to(torch.bfloat16)
    pe = torch.randn(90, 5, rotary, generator=g, device="cuda").to(torch.bfloat16)
    weight = (1 + 0.3 * torch.randn(rank, generator=g, device="cuda")).to(torch.bfloat16)
    table, at = RotaryTable.build(300, rotary), torch.randint(0, 300, (90,), generator=g, device="cuda")
    slots, other = (torch.randperm(160, generator=g, device="cuda")[:90] for _ in range(2))
    cache, peers = (torch.zeros(n, 10, 16, rank + rotary, dtype=torch.bfloat16, device="cuda") for n in (1, 2))
    block_map = torch.randperm(10, generator=g, device="cuda").to(torch.int32)
    targets = [PushTarget.of(peers[0], None, other), PushTarget.of(peers[1], None, None, block_map=block_map)]

    def call(**more):
        return rotate_store_latents(latent, cache[0], slots, at, table, query_pe=pe, weight=weight, **more)

    want = call(push_to=targets)
    rows = cache[0].flatten(0, 1)[slots]
    assert torch.equal(peers[0].flatten(0, 1)[other], rows)
    assert torch.equal(peers[1][block_map[slots // 16].long(), slots % 16], rows)
    peers.zero_()
    kept = cache.clone()
    turned = pe.clone()
    assert call(push_to=targets, out=turned, flags=STORE_PEERS_ONLY) is turned and torch.equal(turned, pe)
    assert torch.equal(cache, kept) and torch.equal(peers[0].flatten(0, 1)[other], rows)
    assert call(push_to=targets, flags=STORE_PEERS_ONLY) is None
    assert torch.equal(call(out=turned), want)


def test_a_gradient_is_refused_not_lost():
    q, k, v, cache, slots, table, at, weights = rows_case(5, 4, 2, 64, 64, 16, torch.bfloat16, fused=False)
    view = cache.transpose(2, 3)
    weights[1].requires_grad_()
    with pytest.raises(ValueError, match="no gradient passes"):
        rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, k_weight=weights[1])
    with torch.no_grad():
        rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, k_weight=weights[1])
    latent, rows = torch.zeros(5, 96, dtype=torch.bfloat16, device="cuda", requires_grad=True), view[0].new_zeros(9, 16, 96)
    with pytest.raises(ValueError, match="no gradient passes"):
        rotate_store_latents(latent, rows, slots, at, RotaryTable.build(512, 32))


def test_a_graph_replays_the_call():
    q, k, v, cache, slots, table, at, weights = rows_case(16, 8, 2, 128, 128, 16, torch.bfloat16, fused=False)
    view = cache.transpose(2, 3)
    out = torch.empty_like(q)
    rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotate_store_kvcache(q, k, v, view[0], view[1], slots, at, table, out=out)
    q.copy_(torch.randn_like(q))
    at.add_(1).remainder_(512)
    graph.replay()
    want, size = rotate64(q, None, 0, 0, table.table, at, False)
    check_rotated(out, want, size)
