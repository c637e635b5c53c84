"""kvx_attention on the GPU against the definition in 64 bits: lengths from nothing to long, masks that leave a row
empty, garbage wherever nothing is to be read, layouts, streams and graphs."""

import math

import pytest
import torch

from lean_vllm_b200._native import STORE_SERIAL
from lean_vllm_b200.attention.kvx_attention import AttentionWorkspace, paged_attention, shared_prefix_attention
from lean_vllm_b200.kv_transfer import transport
from tests.attention_cases import attention64, check_attention, paged_case

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def workspace():
    return AttentionWorkspace("cuda")


def run(case, workspace, **options):
    more = {}
    if any(n != 1 for n in case["q_lens"]):
        more = dict(q_starts=case["q_starts"], max_q_len=max(case["q_lens"]))
    if case["shared"]:
        return shared_prefix_attention(case["q"], case["k_cache"], case["v_cache"], case["prefix_table"],
                                       case["shared"], case["tables"], case["kv_lens"], workspace=workspace, **more,
                                       **options)
    return paged_attention(case["q"], case["k_cache"], case["v_cache"], case["tables"], case["kv_lens"],
                           workspace=workspace, **more, **options)


def check(case, workspace, **options):
    transport.device_error()
    word = transport.StatusWord()
    got = run(case, workspace, status=word.address, **options)
    torch.cuda.synchronize()
    assert word.bits() == 0 and transport.device_error() == 0
    word.close()
    check_attention(got, case, **options)
    return got


@pytest.mark.parametrize("kv_lens, heads, kv_heads, dim, block, dtype, hnd", [
    ([1], 1, 1, 64, 16, BF16, True),
    ([317], 32, 8, 128, 256, BF16, True),
    ([1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000], 8, 2, 128, 16, BF16, True),
    ([0, 5, 0, 700, 0], 4, 2, 64, 16, FP16, True),                    # nothing cached: zeros
    ([333, 77], 14, 2, 64, 24, FP16, False),                          # 7 heads a KV head, 24-token blocks, NHD
    ([401, 90, 3], 10, 2, 128, 256, BF16, False),                     # 5 heads a KV head
    ([2500, 10], 32, 1, 128, 64, BF16, True),                         # one KV head for 32
    ([130, 131], 3, 3, 128, 1, FP16, True),                           # one token a block, no grouping
    ([255, 256, 257], 4, 4, 64, 7, BF16, False),                      # odd blocks
    ([9000, 31, 4097], 8, 1, 128, 16, BF16, True),
    ([40] * 200, 4, 1, 64, 16, BF16, True),                           # more sequences than threads that look at them
], ids=lambda v: None if not isinstance(v, list) else f"{len(v)}x{max(v)}")
def test_single_tokens(kv_lens, heads, kv_heads, dim, block, dtype, hnd, workspace):
    check(paged_case([1] * len(kv_lens), kv_lens, heads, kv_heads, dim, block, dtype, hnd, fused=True), workspace)


@pytest.mark.parametrize("q_lens, kv_lens, heads, kv_heads, dim, block, dtype, hnd", [
    ([5], [5], 4, 1, 64, 16, BF16, True),                             # a whole prompt
    ([300], [300], 8, 2, 128, 64, BF16, True),
    ([129, 1, 0, 64, 3], [129, 500, 77, 1000, 3], 8, 2, 128, 16, BF16, True),  # chunks, single tokens, none
    ([257, 128], [1000, 128], 14, 2, 64, 24, FP16, False),
    ([700], [4099], 4, 1, 128, 256, FP16, True),
    ([33, 40], [40, 300], 6, 2, 128, 5, BF16, True),                  # blocks of 5
    ([4, 4, 4], [4, 600, 2100], 32, 4, 128, 16, BF16, True),          # drafted tokens
    ([10], [3], 4, 2, 64, 16, BF16, True),                            # more queries than keys: the first see nothing
], ids=lambda v: None if not isinstance(v, list) else f"{len(v)}x{max(v)}")
def test_chunks(q_lens, kv_lens, heads, kv_heads, dim, block, dtype, hnd, workspace):
    check(paged_case(q_lens, kv_lens, heads, kv_heads, dim, block, dtype, hnd), workspace)


MASKS = {
    "capped": dict(softcap=3.0),
    "window": dict(window=100),
    "window1": dict(window=1),
    "bias": dict(slopes=True),
    "prefix": dict(prefix_lens=True),
    "all": dict(softcap=5.0, window=33, slopes=True, prefix_lens=True, scale=0.3),
}


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("q_lens, kv_lens, heads, kv_heads, dim, block, dtype", [
    ([1, 1, 1, 1], [1, 64, 333, 1500], 8, 2, 128, 16, BF16),
    ([1, 1], [1000, 100], 4, 4, 64, 24, FP16),
    ([200, 7, 1], [260, 1003, 300], 8, 2, 128, 16, BF16),
    ([513], [777], 7, 1, 64, 64, FP16),
], ids=["decode128", "decode64", "chunks128", "chunk64"])
def test_masks_caps_and_biases(q_lens, kv_lens, heads, kv_heads, dim, block, dtype, mask, workspace):
    options = dict(MASKS[mask])
    if options.get("slopes"):
        options["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    if options.get("prefix_lens"):
        options["prefix_lens"] = torch.tensor([0, 50, 2000, 3][: len(kv_lens)] if len(kv_lens) > 1 else [300],
                                              dtype=torch.int32, device="cuda")
    case = paged_case(q_lens, kv_lens, heads, kv_heads, dim, block, dtype)
    check(case, workspace, **options)


@pytest.mark.parametrize("q_lens, kv_lens, heads, kv_heads, dim, dtype, shared", [
    ([300], [900], 8, 2, 128, BF16, 0),
    ([300], [900], 8, 2, 64, FP16, 0),
    ([40, 1, 90], [2000, 400, 90], 4, 1, 64, BF16, 0),
    ([700, 300], [1500, 300], 16, 8, 128, BF16, 0),
    ([1] * 40, [300] * 40, 8, 2, 128, FP16, 700),
], ids=["prompt128", "prompt64", "chunks64", "prompts128", "shared"])
@pytest.mark.parametrize("window", [0, 350])
def test_caps_near_and_far(q_lens, kv_lens, heads, kv_heads, dim, dtype, shared, window, workspace):
    """Scores well below the cap; scores of which some tiles of keys are near it and beyond, others not; scores beyond it
    everywhere."""
    if shared and window:
        pytest.skip("a shared prefix takes no window")
    for softcap, factor in ((40.0, 1.0), (20.0, 8.0), (0.5, 1.0)):
        case = paged_case(q_lens, kv_lens, heads, kv_heads, dim, 16, dtype, shared=shared)
        if factor != 1.0:  # some stretches of 160 keys
            for s, keys in enumerate(case["keys"]):
                if not shared:
                    i = torch.arange(0, keys.size(0), device="cuda")
                    chosen = i[i // 160 % 3 == 1]
                    keys[chosen] *= factor
                    case["k_cache"][case["tables"][s][chosen // 16].long(), chosen % 16] = keys[chosen]
        check(case, workspace, softcap=softcap, **(dict(window=window) if window else {}))


@pytest.mark.parametrize("kv_heads, group", [(3, 7), (2, 20), (4, 3), (2, 5)])
@pytest.mark.parametrize("q_lens, kv_lens, dim, shared, window", [
    ([300], [900], 128, 0, 0), ([90], [971], 128, 0, 0), ([300, 40], [900, 500], 64, 0, 0), ([300], [900], 128, 0, 120),
    ([3] * 20, [30] * 20, 128, 700, 0), ([3] * 20, [30] * 20, 64, 700, 0),
], ids=["prompt", "short", "chunks64", "window", "shared", "shared64"])
def test_what_ran_before_a_capped_call_changes_no_bit(kv_heads, group, q_lens, kv_lens, dim, shared, window, workspace):
    """Tiles of 128 rows that groups of 3, 5, 7 or 20 heads do not fill: what is left in their last rows from a call before,
    queries near the cap or far beyond it, is no row's business."""
    options = dict(softcap=50.0, **(dict(window=window) if window else {}))
    case = paged_case(q_lens, kv_lens, kv_heads * group, kv_heads, dim, 16, BF16, shared=shared)
    filler = paged_case([400] * 8, [400] * 8, 8 * kv_heads, kv_heads, dim, 16, BF16)
    seen = []
    for factor in (0.0, 1000.0, 0.0, 1000.0):
        filler["q"].fill_(factor)
        run(filler, workspace)
        fill = paged_case([16] * 20, [16] * 20, 8 * kv_heads, kv_heads, dim, 16, BF16, shared=300)
        fill["q"].fill_(factor)
        run(fill, workspace)
        seen.append(run(case, workspace, **options))
    check_attention(seen[0], case, **options)
    assert all(torch.equal(x, seen[0]) for x in seen)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens, kv_lens, heads, shared", [
    ([1], [20000], 4, 0), ([4], [20000], 4, 0), ([3, 1], [9000, 17], 1, 0),  # one walk of the cache in hundreds of parts
    ([40], [20000], 4, 0), ([20, 1], [30000, 5], 8, 0),
    ([1, 2], [50, 0], 4, 20000),
], ids=["rows4", "rows16", "rows3", "tiles", "mixed", "shared"])
def test_many_parts(q_lens, kv_lens, heads, shared, dim, workspace):
    """One KV head and a long cache: parts in numbers that are joined in several rounds, the same each time."""
    case = paged_case(q_lens, kv_lens, heads, 1, dim, 16, BF16, shared=shared)
    first = check(case, workspace)
    for _ in range(3):
        assert torch.equal(run(case, workspace), first)


@pytest.mark.parametrize("dim", [64, 128])
def test_more_items_than_a_wave(dim, workspace):
    """Tiles of rows that CTAs take one after another."""
    check(paged_case([900, 3, 400], [900, 600, 1000], 32, 8, dim, 16, BF16), workspace)


def test_a_window_never_reads_what_lies_before_it(workspace):
    """Blocks ahead of every row's window may be gone: their table entries are stale and their rows NaN."""
    case = paged_case([1, 20], [1000, 700], 8, 2, 128, 16, BF16)
    for s, (q_len, n) in enumerate(zip(case["q_lens"], [1000, 700])):
        first = n - q_len - 100 + 1  # the first key that any row sees
        ids = case["tables"][s]
        for t in range(first):
            b, o = int(ids[t // 16]), t % 16
            case["k_cache"][b, o] = math.nan
            case["v_cache"][b, o] = math.nan
        case["tables"][s, : first // 16] = -1
    check(case, workspace, window=100)


@pytest.mark.parametrize("q_len, kv_len", [(4, 2), (10, 3), (300, 260), (5, 0)])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 200])
def test_the_widest_windows_see_everything(q_len, kv_len, window, workspace):
    """Also for queries that stand ahead of the first key."""
    check(paged_case([q_len], [kv_len], 4, 2, 64, 16, BF16), workspace, window=window)


@pytest.mark.parametrize("prefix", [1, 5, 64, 70, 200, 640, 899, 10000])
@pytest.mark.parametrize("q_lens, kv_lens, heads, kv_heads, dim, block, options", [
    ([1, 1, 1], [1000, 2001, 150], 8, 2, 128, 16, {}),
    ([4, 2], [1000, 777], 8, 2, 64, 24, {}),
    ([1, 3], [1000, 650], 4, 2, 128, 7, {}),                           # blocks that lie in no stage of keys
    ([20, 300], [1000, 900], 8, 2, 128, 16, {}),
    ([130, 1], [1500, 1300], 4, 1, 64, 64, {}),
    ([60], [9000], 4, 1, 128, 16, {}),                                 # cut along the keys
    ([200, 1], [1200, 1200], 8, 2, 128, 16, {"softcap": 20.0}),
], ids=["decode", "drafts64", "odd", "chunks", "chunks64", "cut", "capped"])
def test_what_lies_between_a_prefix_and_the_window_is_never_read(q_lens, kv_lens, heads, kv_heads, dim, block, options,
                                                                 prefix, workspace):
    """First tokens and a sliding window: keys and values between the two may be gone, NaN rows and stale table entries."""
    case = paged_case(q_lens, kv_lens, heads, kv_heads, dim, block, BF16)
    for s, (q_len, n) in enumerate(zip(q_lens, kv_lens)):
        gap = torch.arange(min(prefix, n), max(n - q_len - 100 + 1, min(prefix, n)), device="cuda")
        case["k_cache"][case["tables"][s][gap // block].long(), gap % block] = math.nan
        case["v_cache"][case["tables"][s][gap // block].long(), gap % block] = math.nan
        blocks = torch.arange(case["tables"].size(1), device="cuda")
        stale = (blocks * block >= prefix) & ((blocks + 1) * block <= n - q_len - 100 + 1)
        case["tables"][s][stale] = torch.where(blocks[stale] % 2 == 0, -1, 2**30).to(torch.int32)
    check(case, workspace, window=100, prefix_lens=torch.full((len(q_lens),), prefix, dtype=torch.int32, device="cuda"),
          **options)


@pytest.mark.parametrize("q_lens, kv_lens, shared, heads, kv_heads, dim, block, dtype, hnd", [
    ([1] * 3, [1, 17, 40], 100, 8, 2, 128, 16, BF16, True),
    ([1] * 64, list(range(1, 65)), 1000, 32, 8, 128, 256, BF16, True),
    ([4] * 5, [4, 129, 60, 30, 5], 3001, 32, 8, 128, 16, BF16, True),
    ([1, 3, 2], [20, 3, 77], 333, 14, 2, 64, 24, FP16, False),
    ([1, 1], [5, 6], 1, 4, 1, 64, 7, FP16, True),                     # a prefix of one token, odd blocks
    ([150, 1, 30], [150, 9, 400], 500, 8, 2, 128, 64, BF16, True),    # prompts behind a prefix
    ([1], [7], 5000, 16, 1, 128, 64, FP16, False),
    ([1] * 300, [3] * 300, 257, 8, 1, 64, 16, BF16, True),            # 2400 rows of one KV head
], ids=lambda v: None if not isinstance(v, list) else f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("options", [{}, {"softcap": 4.0}, {"slopes": True}], ids=["plain", "capped", "bias"])
def test_a_shared_prefix(q_lens, kv_lens, shared, heads, kv_heads, dim, block, dtype, hnd, options, workspace):
    options = dict(options)
    if options.get("slopes"):
        options["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    case = paged_case(q_lens, kv_lens, heads, kv_heads, dim, block, dtype, hnd, shared=shared)
    check(case, workspace, **options)


@pytest.mark.parametrize("q_lens, options", [([1] * 1100, {}), ([3, 1, 2, 4] * 300 + [1], {}),
                                             ([2, 3] * 250 + [2] * 3, {"slopes": True})],
                         ids=["single", "drafts", "bias"])
def test_more_rows_behind_a_prefix_than_parts_fit(q_lens, options, workspace):
    """A batch that goes in several runs: three launches each, sequences cut between two of them among the checked ones."""
    heads, options = 64, dict(options)
    if options:
        options["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    kv_lens = [n + i % 23 for i, n in enumerate(q_lens)]
    case = paged_case(q_lens, kv_lens, heads, 4, 64, 16, BF16, shared=300)
    run(case, workspace, **options)
    runs = -(-2 * sum(q_lens) * heads // 131072)
    each = -(-sum(q_lens) // runs)
    before = transport.launch_count()
    out = run(case, workspace, **options)
    assert runs > 1 and transport.launch_count() - before == 3 * runs
    starts = case["q_starts"].tolist()
    cut = [s for s in range(len(q_lens)) if starts[s] // each != (starts[s + 1] - 1) // each]
    assert len(cut) == (0 if max(q_lens) == 1 else runs - 1)
    chosen = sorted({*range(0, len(q_lens), 97), *cut, len(q_lens) - 1})
    rows = torch.cat([torch.arange(starts[s], starts[s + 1], device="cuda") for s in chosen])
    some = dict(case, q=case["q"][rows], q_lens=[q_lens[s] for s in chosen], keys=[case["keys"][s] for s in chosen],
                values=[case["values"][s] for s in chosen])
    check_attention(out[rows], some, **options)
    assert torch.isfinite(out).all()


def test_a_shared_prefix_with_nothing_behind_it(workspace):
    """kv_lens of 0: rows that see the prefix alone."""
    case = paged_case([1, 1], [0, 0], 8, 2, 128, 16, BF16, shared=200)
    case["q_lens"] = [1, 1]
    check(case, workspace)


def test_a_long_cache(workspace):
    """One sequence of 100,003 tokens, all the parallelism from its length, and a prefix as long."""
    check(paged_case([1], [100003], 8, 2, 128, 64, BF16), workspace)
    check(paged_case([1, 2], [5, 9], 8, 2, 128, 64, BF16, shared=70001), workspace)


def test_a_cache_past_four_gigabytes(workspace):
    blocks = 9000
    cache = torch.zeros(2, blocks, 8, 256, 128, dtype=BF16, device="cuda")  # 2 x 4.7 GB
    view = cache.transpose(2, 3)
    for q_len in (1, 100):
        case = paged_case([q_len], [700], 8, 8, 128, 256, BF16, seed=q_len)
        ids = torch.tensor([8999, 8500, 8700], dtype=torch.int32, device="cuda")
        both = torch.stack([case["k_cache"], case["v_cache"]])[:, case["tables"][0].long()]
        view[:, ids.long()] = both
        case.update(k_cache=view[0], v_cache=view[1], tables=ids[None].contiguous())
        check(case, workspace)


def test_scores_far_apart_and_large_values(workspace):
    """Scores in the hundreds (the running maximum grows from tile to tile) and keys that fall steadily."""
    for q_len in (1, 150):
        case = paged_case([q_len], [1500], 4, 1, 128, 16, BF16)
        case["q"].mul_(30)
        check(case, workspace)
        ramp = torch.linspace(-1, 1, 1500, device="cuda")[:, None, None]
        for sign in (1, -1):
            case = paged_case([q_len], [1500], 4, 1, 128, 16, BF16)
            keys = (torch.ones(1500, 1, 128, device="cuda") * ramp * sign).to(BF16)
            case["keys"] = [keys]
            i = torch.arange(1500, device="cuda")
            case["k_cache"][case["tables"][0][i // 16].long(), i % 16] = keys
            case["q"].abs_()
            check(case, workspace)


def test_block_ids_outside_the_cache_read_as_zeros_and_are_flagged(workspace):
    for q_len in (1, 200):
        case = paged_case([q_len], [500], 8, 2, 128, 16, BF16, garbage=False)
        case["tables"][0, 3] = 10**6
        case["tables"][0, 7] = -2
        keys, values = case["keys"][0], case["values"][0]
        for b in (3, 7):
            keys[b * 16 : b * 16 + 16] = 0
            values[b * 16 : b * 16 + 16] = 0
        transport.device_error()
        word = transport.StatusWord()
        got = run(case, workspace, status=word.address)
        torch.cuda.synchronize()
        assert word.bits() == 2 and transport.device_error() == 2
        word.close()
        check_attention(got, case)


def test_a_length_past_its_table_is_cut_and_flagged(workspace):
    for q_len in (1, 40):
        case = paged_case([q_len], [64], 8, 2, 128, 16, BF16)
        case["kv_lens"][0] = 5000
        transport.device_error()
        word = transport.StatusWord()
        got = run(case, workspace, status=word.address)
        torch.cuda.synchronize()
        assert word.bits() == 2 and transport.device_error() == 2
        word.close()
        check_attention(got, case)


@pytest.mark.parametrize("q_lens, kv_lens, shared", [([1] * 7, [900, 1, 30, 5000, 77, 64, 128], 0),
                                                      ([300, 1, 9], [4000, 700, 9], 0), ([1] * 9, [50] * 9, 3000)],
                         ids=["decode", "chunks", "shared"])
def test_the_same_call_gives_the_same_bits(q_lens, kv_lens, shared, workspace):
    """Parts join in a fixed order whichever CTA joins them, and the bounds on the lengths change the shape of the launch
    only: wrong ones cost time."""
    case = paged_case(q_lens, kv_lens, 8, 2, 128, 16, BF16, shared=shared)
    first = run(case, workspace)
    for _ in range(5):
        assert torch.equal(run(case, workspace), first)
    for bound in (1, 100000):
        check_attention(run(case, workspace, max_kv_len=bound), case)


def test_wrong_bounds_on_the_query_lengths_are_harmless(workspace):
    case = paged_case([70, 1, 200], [300, 900, 200], 8, 2, 128, 16, BF16)
    for bound in (1, 2, 17, 10000):
        got = paged_attention(case["q"], case["k_cache"], case["v_cache"], case["tables"], case["kv_lens"],
                              q_starts=case["q_starts"], max_q_len=bound, workspace=workspace)
        check_attention(got, case)


@pytest.mark.parametrize("kv_lens, heads, kv_heads, dim, shared", [
    ([4096, 77], 32, 8, 128, 0), ([600, 1, 0, 300], 32, 8, 128, 0), ([5000, 9], 14, 2, 64, 0), ([3, 40, 2], 32, 4, 128, 3000),
], ids=["long", "short", "dim64", "shared"])
@pytest.mark.parametrize("bound", [5, 16, 10000])
def test_single_tokens_are_single_whatever_the_bound(kv_lens, heads, kv_heads, dim, shared, bound, workspace):
    """Without q_starts a bound on the query lengths, a captured maximum say, means nothing: the same bits."""
    case = paged_case([1] * len(kv_lens), kv_lens, heads, kv_heads, dim, 16, BF16, shared=shared)
    want = check(case, workspace)
    assert torch.equal(run(case, workspace, max_q_len=bound), want)


def test_strided_queries_and_outputs(workspace):
    for q_lens in ([1, 1], [90, 5]):
        case = paged_case(q_lens, [200, 300], 6, 2, 128, 16, BF16, fused=True)
        want = run(case, workspace)
        wide = torch.zeros(sum(q_lens), 10, 128, dtype=BF16, device="cuda")
        got = run(case, workspace, out=wide[:, 3:9])
        assert got.data_ptr() == wide[:, 3:9].data_ptr() and torch.equal(got, want)
        assert not wide[:, :3].any() and not wide[:, 9:].any()


@pytest.mark.parametrize("q_lens, kv_lens", [([1, 1], [90, 333]), ([40, 200], [90, 333])], ids=["decode", "chunks"])
def test_block_tables_that_are_views(q_lens, kv_lens, workspace):
    """A batch's rows of a wider table, as an engine keeps for all its requests."""
    case = paged_case(q_lens, kv_lens, 8, 2, 128, 16, BF16)
    wide = torch.full((9, 50), -7, dtype=torch.int32, device="cuda")
    wide[3:5, : case["tables"].size(1)] = case["tables"]
    case["tables"] = wide[3:5, : case["tables"].size(1)]
    check(case, workspace)


@pytest.mark.parametrize("q_lens, kv_lens, heads, kv_heads, dim", [
    ([1, 1], [77, 900], 160, 1, 64),    # more heads on a KV head than a tile has rows
    ([3, 50], [77, 300], 160, 1, 128),
    ([2, 100], [20, 130], 72, 1, 64),   # one token a tile of 128 rows
    ([1, 33], [400, 400], 1, 1, 128),
])
def test_large_and_single_groups(q_lens, kv_lens, heads, kv_heads, dim, workspace):
    check(paged_case(q_lens, kv_lens, heads, kv_heads, dim, 16, BF16), workspace)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
def test_any_scale(scale, workspace):
    for q_lens, kv_lens in (([1, 1], [70, 500]), ([100, 30], [300, 400])):
        check(paged_case(q_lens, kv_lens, 8, 2, 128, 16, BF16), workspace, scale=scale)


@pytest.mark.parametrize("softcap", [5.0, 30.0, 50.0])
@pytest.mark.parametrize("q_lens, kv_lens, heads, kv_heads, dim, dtype, shared", [
    ([300], [900], 8, 2, 128, FP16, 0), ([300, 40], [900, 700], 4, 2, 64, FP16, 0), ([300], [900], 8, 2, 128, BF16, 0),
    ([1] * 20, [50] * 20, 8, 2, 128, FP16, 700), ([1, 2], [500, 300], 8, 2, 128, FP16, 0),
], ids=["prompt128", "chunks64", "bf16", "shared", "decode"])
def test_a_negative_scale_under_a_cap(q_lens, kv_lens, heads, kv_heads, dim, dtype, shared, softcap, workspace):
    """Capped scores fall as the products rise: the row's maximum is its smallest product."""
    check(paged_case(q_lens, kv_lens, heads, kv_heads, dim, 16, dtype, shared=shared), workspace, scale=-0.2,
          softcap=softcap)


def test_a_nan_that_is_seen_shows(workspace):
    """NaN in a key that every row sees makes every output of its head NaN, and of no other."""
    for q_lens, options in (([1], {}), ([70], {}), ([70], {"softcap": 5.0}), ([1], {"softcap": 5.0})):
        case = paged_case(q_lens, [300], 4, 2, 128, 16, BF16)
        case["k_cache"][int(case["tables"][0, 1]), 5, 1] = math.nan  # position 21, KV head 1
        out = run(case, workspace, **options)
        assert torch.isnan(out[:, 2:]).all() and torch.isfinite(out[:, :2]).all()


def test_no_tokens_launch_nothing(workspace):
    case = paged_case([1], [5], 4, 2, 64, 16, BF16)
    before = transport.launch_count()
    out = paged_attention(case["q"][:0], case["k_cache"], case["v_cache"], case["tables"][:0], case["kv_lens"][:0],
                          workspace=workspace)
    assert out.shape == (0, 4, 64) and transport.launch_count() == before


def test_other_streams(workspace):
    """A side stream with a workspace of its own beside the current one, and a raw stream handle."""
    for q_lens, kv_lens, shared in (([1, 1], [3000, 50], 0), ([200], [900], 0), ([1] * 8, [9] * 8, 2000)):
        case = paged_case(q_lens, kv_lens, 8, 2, 128, 16, BF16, shared=shared)
        want = run(case, workspace)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            own = AttentionWorkspace("cuda")
            late = dict(case, q=torch.zeros_like(case["q"]))
            for _ in range(20):
                late["q"].copy_(case["q"])  # the queries arrive on this stream only
            got = [run(late, own) for _ in range(3)]
        here = [run(case, workspace) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got + here)
        raw = run(case, None, stream=side.cuda_stream)
        side.synchronize()
        assert torch.equal(raw, want)


def test_an_output_made_for_another_stream_waits_for_nobody(workspace):
    """Work still queued on the current stream on memory that was freed there does not reach an output (or a workspace)
    made for a call on another stream."""
    case = paged_case([200], [900], 32, 8, 128, 16, BF16)
    want = run(case, workspace)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        own = AttentionWorkspace("cuda")
    for mine in (own, None):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        taken = [torch.empty_like(case["q"]), torch.empty_like(own.tensor)]
        torch.cuda._sleep(50_000_000)  # tens of ms
        for t in taken:
            t.fill_(1)
        del taken, t
        got = run(case, mine, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_stream_0_is_the_default_stream(workspace):
    """A workspace made for stream 0, and a call there, while another stream is the current one and busy."""
    case = paged_case([1, 40], [900, 300], 8, 2, 128, 16, BF16)
    want = run(case, workspace)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        dirty = torch.full((workspace.tensor.numel(),), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        del dirty
        torch.cuda._sleep(50_000_000)
        made = AttentionWorkspace("cuda", stream=0)
        with torch.cuda.stream(torch.cuda.default_stream()):
            head = made.tensor[:65536].clone()
    torch.cuda.synchronize()
    assert not head.any()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        got = run(case, None, stream=0)
        torch.cuda.default_stream().synchronize()
        assert not side.query()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_a_gradient_is_refused_not_lost(workspace):
    case = paged_case([1], [70], 4, 2, 64, 16, BF16)
    want = run(case, workspace)
    case["q"].requires_grad_()
    with pytest.raises(ValueError, match="no gradient passes"):
        run(case, workspace)
    with torch.no_grad():
        assert torch.equal(run(case, workspace), want)
    with torch.inference_mode():
        assert torch.equal(run(case, workspace), want)


def test_plain_launches_give_the_same_bits(workspace):
    for q_lens, kv_lens, shared in (([1, 1], [3000, 50], 0), ([200, 1], [900, 700], 0), ([40], [9000], 0),
                                    ([1] * 8, [9] * 8, 2000)):
        case = paged_case(q_lens, kv_lens, 8, 2, 128, 16, BF16, shared=shared)
        want = run(case, workspace)
        for _ in range(3):
            assert torch.equal(run(case, workspace, flags=STORE_SERIAL), want)


def test_a_graph_replays_the_call_at_other_lengths(workspace):
    """Lengths live on the device: a captured call follows them."""
    for q_lens, kv_lens, shared in (([1, 1, 1], [800, 300, 50], 0), ([64, 64], [500, 400], 0), ([1, 1], [40, 60], 700)):
        case = paged_case(q_lens, kv_lens, 8, 2, 128, 16, BF16, shared=shared)
        own = AttentionWorkspace("cuda")
        out = torch.empty_like(case["q"])
        run(case, own, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(case, own, out=out)
        for shorter in (0, 3):
            lens = [n - shorter for n in kv_lens]
            case["kv_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
            now = dict(case, keys=[k[: shared + n] for k, n in zip(case["keys"], lens)],
                       values=[v[: shared + n] for v, n in zip(case["values"], lens)])
            for _ in range(2):
                graph.replay()
            torch.cuda.synchronize()
            check_attention(out, now)


def test_the_reference_notices_one_missing_key():
    """The oracle's own check: leave out one key of 200 on the oracle's side and the row limit is passed."""
    case = paged_case([1], [200], 4, 4, 128, 16, BF16)
    want, _, _ = attention64(case)
    check_attention(want.to(BF16), case)
    wrong = dict(case, keys=[case["keys"][0][1:]], values=[case["values"][0][1:]])
    with pytest.raises(AssertionError):
        check_attention(attention64(wrong)[0].to(BF16), case)
