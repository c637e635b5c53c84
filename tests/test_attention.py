"""What the attention and rotary entry points refuse, before anything reaches a device (these run on CPU tensors), and
the rotary table's angles."""

import ctypes
import math
import os
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from lean_vllm_b200 import _native
from lean_vllm_b200.attention.kvx_attention import paged_attention, shared_prefix_attention
from lean_vllm_b200.attention.kvx_cache import PushTarget
from lean_vllm_b200.attention.kvx_rotary import RotaryTable, rotate_store_kvcache, rotate_store_latents

BF16 = torch.bfloat16


def store_args(**change):
    args = dict(query=torch.zeros(4, 4, 64, dtype=BF16), key=torch.zeros(4, 2, 64, dtype=BF16),
                value=torch.zeros(4, 2, 64, dtype=BF16), k_cache=torch.zeros(3, 16, 2, 64, dtype=BF16),
                v_cache=torch.zeros(3, 16, 2, 64, dtype=BF16), slot_mapping=torch.arange(4),
                positions=torch.arange(4), rotary=RotaryTable(torch.zeros(8, 64)))
    args.update(change)
    return args


@pytest.mark.parametrize("change, error, message", [
    (dict(query=torch.zeros(4, 256, dtype=BF16)), ValueError, "num_tokens, heads, dim"),
    (dict(query=torch.zeros(5, 4, 64, dtype=BF16)), ValueError, "beside keys"),
    (dict(value=torch.zeros(4, 1, 64, dtype=BF16)), ValueError, "shapes must match"),
    (dict(k_cache=torch.zeros(3, 16, 4, 64, dtype=BF16), v_cache=torch.zeros(3, 16, 4, 64, dtype=BF16)), ValueError,
     "2 heads of 64 into a cache of 4"),
    (dict(query=torch.zeros(4, 4, 64)), TypeError, "share a dtype"),
    (dict(query=torch.zeros(4, 4, 64), key=torch.zeros(4, 2, 64), value=torch.zeros(4, 2, 64),
          k_cache=torch.zeros(3, 16, 2, 64), v_cache=torch.zeros(3, 16, 2, 64)), TypeError, "bfloat16 or float16"),
    (dict(v_cache=torch.zeros(3, 2, 16, 64, dtype=BF16).transpose(1, 2)), ValueError, "share strides"),
    (dict(key=torch.zeros(4, 2, 128, dtype=BF16)[..., ::2]), ValueError, "elements must be contiguous"),
    (dict(slot_mapping=torch.arange(3)), ValueError, "3 slots for 4 rows"),
    (dict(slot_mapping=torch.zeros(4)), TypeError, "slots are int32 or int64"),
    (dict(positions=torch.arange(5)), ValueError, "5 positions for 4 rows"),
    (dict(positions=torch.zeros(4)), TypeError, "positions are int32 or int64"),
    (dict(positions=torch.arange(8)[::2]), ValueError, "positions must be contiguous"),
    (dict(rotary=RotaryTable(torch.zeros(8, 66))), ValueError, "66 elements for heads of 64"),
    (dict(q_weight=torch.zeros(32, dtype=BF16)), ValueError, "64 contiguous elements"),
    (dict(k_weight=torch.zeros(64)), ValueError, "rows' dtype"),
    (dict(out=torch.zeros(4, 4, 32, dtype=BF16)), ValueError, "`out` must have"),
    (dict(push_to=[PushTarget(1, 1, 0, 0, 0, 16, 1, None)] * 9), ValueError, "at most 8 peers"),
])
def test_rotate_store_refuses(change, error, message):
    with pytest.raises(error, match=message):
        rotate_store_kvcache(**store_args(**change))


def latent_args(**change):
    args = dict(latent=torch.zeros(4, 96, dtype=BF16), latent_cache=torch.zeros(3, 16, 96, dtype=BF16),
                slot_mapping=torch.arange(4), positions=torch.arange(4), rotary=RotaryTable(torch.zeros(8, 32)))
    args.update(change)
    return args


@pytest.mark.parametrize("change, error, message", [
    (dict(latent_cache=torch.zeros(3, 16, 64, dtype=BF16)), ValueError, "into a cache"),
    (dict(latent_cache=torch.zeros(3, 16, 96)), TypeError, "share a dtype"),
    (dict(latent_cache=torch.zeros(3, 96, 16, dtype=BF16).transpose(1, 2)), ValueError, "cache tokens must be contiguous"),
    (dict(rotary=RotaryTable(torch.zeros(8, 128))), ValueError, "128 elements for latents of 96"),
    (dict(query_pe=torch.zeros(4, 2, 64, dtype=BF16)), ValueError, "rotated part"),
    (dict(query_pe=torch.zeros(4, 2, 32)), TypeError, "share a dtype"),
    (dict(weight=torch.zeros(96, dtype=BF16)), ValueError, "64 contiguous elements"),
    (dict(positions=torch.arange(3)), ValueError, "3 positions for 4 rows"),
])
def test_rotate_store_latents_refuses(change, error, message):
    with pytest.raises(error, match=message):
        rotate_store_latents(**latent_args(**change))


@pytest.mark.parametrize("table, message", [
    (torch.zeros(8, 64, dtype=torch.float64), "float32"),
    (torch.zeros(8, 64).T, "contiguous"),
    (torch.zeros(64), "float32 tensor"),
    (torch.zeros(0, 64), "0 positions"),
    (torch.zeros(8, 63), "rotary_dim 63"),
])
def test_a_rotary_table_refuses(table, message):
    with pytest.raises(ValueError, match=message):
        RotaryTable(table)


def attention_args(**change):
    args = dict(query=torch.zeros(3, 4, 64, dtype=BF16), k_cache=torch.zeros(5, 16, 2, 64, dtype=BF16),
                v_cache=torch.zeros(5, 16, 2, 64, dtype=BF16), block_tables=torch.zeros(3, 2, dtype=torch.int32),
                kv_lens=torch.ones(3, dtype=torch.int32))
    args.update(change)
    return args


@pytest.mark.parametrize("change, error, message", [
    (dict(query=torch.zeros(3, 256, dtype=BF16)), ValueError, "over caches"),
    (dict(v_cache=torch.zeros(4, 16, 2, 64, dtype=BF16)), ValueError, "over caches"),
    (dict(query=torch.zeros(3, 3, 64, dtype=BF16)), ValueError, "3 query heads of 64 over 2 KV heads"),
    (dict(query=torch.zeros(3, 4, 128, dtype=BF16)), ValueError, "of 128 over 2 KV heads of 64"),
    (dict(query=torch.zeros(3, 4, 64)), TypeError, "share a dtype"),
    (dict(v_cache=torch.zeros(5, 2, 16, 64, dtype=BF16).transpose(1, 2)), ValueError, "share strides"),
    (dict(query=torch.zeros(3, 4, 128, dtype=BF16)[..., ::2]), ValueError, "contiguous"),
    (dict(block_tables=torch.zeros(3, 2)), ValueError, "int32 tensor"),
    (dict(block_tables=torch.zeros(6, dtype=torch.int32)), ValueError, "int32 tensor"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int32).T), ValueError, "block ids must be contiguous"),
    (dict(kv_lens=torch.ones(3, dtype=torch.int64)), ValueError, "kv_lens must be"),
    (dict(kv_lens=torch.ones(4, dtype=torch.int32)), ValueError, "kv_lens must be"),
    (dict(q_starts=torch.ones(3, dtype=torch.int32)), ValueError, "q_starts must be"),
    (dict(query=torch.zeros(5, 4, 64, dtype=BF16)), ValueError, "needs q_starts"),
    (dict(prefix_lens=torch.ones(2, dtype=torch.int32)), ValueError, "prefix_lens must be"),
    (dict(slopes=torch.ones(3)), ValueError, "slopes are 4"),
    (dict(slopes=torch.ones(4, dtype=BF16)), ValueError, "slopes are 4"),
    (dict(out=torch.zeros(3, 4, 64)), ValueError, "`out` must have"),
])
def test_attention_refuses(change, error, message):
    with pytest.raises(error, match=message):
        paged_attention(**attention_args(**change))


def test_shared_prefix_attention_refuses():
    args = attention_args()
    with pytest.raises(ValueError, match="a prefix of -1"):
        shared_prefix_attention(args["query"], args["k_cache"], args["v_cache"], torch.zeros(1, dtype=torch.int32), -1,
                                args["block_tables"], args["kv_lens"])
    with pytest.raises(ValueError, match="prefix_table must be"):
        shared_prefix_attention(args["query"], args["k_cache"], args["v_cache"], torch.zeros(1), 3,
                                args["block_tables"], args["kv_lens"])


@pytest.mark.parametrize("call, args, name", [
    (paged_attention, attention_args, "query"), (paged_attention, attention_args, "k_cache"),
    (rotate_store_kvcache, store_args, "query"), (rotate_store_kvcache, store_args, "key"),
    (rotate_store_kvcache, store_args, "value"), (rotate_store_latents, latent_args, "latent"),
])
def test_inputs_whose_gradient_would_be_lost_are_refused(call, args, name):
    given = args()
    given[name].requires_grad_()
    with pytest.raises(ValueError, match="no gradient passes"):
        call(**given)
    given["out"] = torch.zeros(1)  # with no gradient recorded the checks go on, to this one or the device's
    with torch.no_grad(), pytest.raises(Exception) as other:
        call(**given)
    assert "gradient" not in str(other.value)


def test_weights_and_slopes_whose_gradient_would_be_lost_are_refused():
    weight = torch.ones(64, dtype=BF16, requires_grad=True)
    for change in (dict(q_weight=weight), dict(k_weight=weight)):
        with pytest.raises(ValueError, match="no gradient passes"):
            rotate_store_kvcache(**store_args(**change))
    with pytest.raises(ValueError, match="no gradient passes"):
        rotate_store_latents(**latent_args(weight=weight))
    with pytest.raises(ValueError, match="no gradient passes"):
        paged_attention(**attention_args(slopes=torch.ones(4, requires_grad=True)))


def in_a_thread(fn):
    """fn(), in a thread of its own: the library's last error is per thread, and other tests look at this one's."""
    with ThreadPoolExecutor(1) as pool:
        return pool.submit(fn).result()


def attention_struct(**change):
    fields = dict(query=16, q_token_stride=512, q_head_stride=128, out=16, out_token_stride=512, out_head_stride=128,
                  k_cache=16, v_cache=16, block_stride=4096, token_stride=256, head_stride=128, block_tables=16,
                  table_stride=2, kv_lens=16, workspace=128, block_size=16, num_blocks=5, max_blocks=2, batch=3,
                  num_tokens=3, q_heads=4, kv_heads=2, head_dim=64, max_q_len=1, max_kv_len=32, scale=0.125)
    fields.update(change)
    return _native.AttentionArgs(**fields)


@pytest.mark.parametrize("change, message", [
    (dict(head_dim=96), "head_dim 96"),
    (dict(q_heads=5), "5 query heads over 2"),
    (dict(kv_heads=0), "over 0 KV heads"),
    (dict(dtype=7), "element type 7"),
    (dict(num_tokens=-1), "-1 tokens"),
    (dict(block_size=0), "bad block size"),
    (dict(block_size=1 << 20, max_blocks=1 << 12), "more than 2"),
    (dict(window=-3), "negative window"),
    (dict(softcap=-1.0), "negative window or softcap"),
    (dict(softcap=math.nan), "negative window or softcap"),
    (dict(shared_len=100, shared_blocks=6, shared_table=16), "100 tokens in 6 blocks"),
    (dict(shared_len=90, shared_blocks=6), "null pointer"),
    (dict(query=None), "null pointer"),
    (dict(workspace=None), "null pointer"),
    (dict(workspace=64), "128 bytes"),
    (dict(q_token_stride=510), "16-byte boundaries"),
    (dict(k_cache=8), "16-byte boundaries"),
    (dict(num_tokens=9), "need q_starts"),
    (dict(shared_len=90, shared_blocks=6, shared_table=16, window=5), "takes no window"),
])
def test_the_abi_refuses_attention_arguments(change, message):
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libkvx.so is not built here")
    with pytest.raises(_native.KvxError, match=message):
        struct = attention_struct(**change)
        in_a_thread(lambda: _native.check(_native.lib().kvx_attention(ctypes.addressof(struct), 0, None)))


@pytest.mark.parametrize("change", [
    dict(block_size=1, max_blocks=2**31 - 1), dict(block_size=128, max_blocks=2**24 - 1),
    dict(block_size=1 << 20, max_blocks=2047, shared_len=1 << 29, shared_blocks=1 << 9, shared_table=16),
    dict(block_size=1 << 20, shared_len=2**31 - 1, shared_blocks=1 << 11, shared_table=16),
], ids=["table", "last tile", "both", "shared"])
def test_the_abi_refuses_sequences_whose_positions_pass_31_bits(change):
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libkvx.so is not built here")
    with pytest.raises(_native.KvxError, match="tokens a sequence"):
        struct = attention_struct(**change)
        in_a_thread(lambda: _native.check(_native.lib().kvx_attention(ctypes.addressof(struct), 0, None)))


def test_the_abi_refuses_an_infinite_cap():
    """inf * tanh(s / inf) is no number."""
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libkvx.so is not built here")
    with pytest.raises(_native.KvxError, match="infinite softcap"):
        struct = attention_struct(softcap=math.inf)
        in_a_thread(lambda: _native.check(_native.lib().kvx_attention(ctypes.addressof(struct), 0, None)))


@pytest.mark.parametrize("flags", [_native.STORE_PEERS_ONLY, 2, 8 << 24, -1])
def test_the_abi_refuses_flags_that_attention_does_not_have(flags):
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libkvx.so is not built here")
    with pytest.raises(_native.KvxError, match="flags"):
        struct = attention_struct()
        in_a_thread(lambda: _native.check(_native.lib().kvx_attention(ctypes.addressof(struct), flags, None)))


def test_the_abi_refuses_rotate_arguments():
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libkvx.so is not built here")
    lib = _native.lib()
    dest = (_native.StoreDest * 1)(_native.StoreDest(4096, 4096, 4096, 256, 128, 16, 3, 16, 8, 0, 2, 0, None, 0, 0))

    def rows(**change):
        return _native.RotateRows(**{**dict(rows=16, token_stride=256, head_stride=128, num_heads=2, dim=64), **change})

    def call(dests=dest, n=1, **change):
        fields = dict(query=rows(), key=rows(), value=rows(), query_out=16, table=16, positions=16, num_positions=8,
                      rotary_dim=64, position_bytes=8, num_tokens=4, eps=1e-6)
        fields.update(change)
        args = _native.RotateArgs(**fields)
        in_a_thread(lambda: _native.check(lib.kvx_rotate_store(ctypes.addressof(args), ctypes.addressof(dests), n, None, 0,
                                                               None)))

    for change, message in [
        (dict(dtype=9), "element type 9"), (dict(num_tokens=-1), "-1 tokens"), (dict(rotary_dim=7), "not an even"),
        (dict(table=None), "needs a table"), (dict(num_positions=0), "needs a table"),
        (dict(position_bytes=2), "8-byte positions"), (dict(query_out=None), "null query output"),
        (dict(rotary_dim=66), r"rotated elements \[0, \+66\) of 64"), (dict(key=rows(num_heads=0)), "0 key heads"),
        (dict(key=rows(norm_dim=64)), "needs its weight"), (dict(key=rows(norm_dim=65)), "65 normed"),
        (dict(value=rows(dim=32)), "keys' shape"), (dict(value=rows(rows=None)), "null rows"),
        (dict(key=rows(rotary_first=1)), r"\[1, \+64\) of 64"), (dict(n=0), "0 destinations"),
        (dict(key=rows(num_heads=1), value=rows(num_heads=1)), "heads"),
    ]:
        with pytest.raises(_native.KvxError, match=message):
            call(**change)


def test_the_structs_are_the_header_s(tmp_path):
    """The ctypes structs have the sizes and field offsets the C compiler gives the header's."""
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    pairs = [("kvx_rotate_rows", _native.RotateRows), ("kvx_rotate_args", _native.RotateArgs),
             ("kvx_attention_args", _native.AttentionArgs), ("kvx_store_dest", _native.StoreDest)]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "kvx.h"', "int main(void) {"]
    for name, struct in pairs:
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {field}));' for field, _ in struct._fields_]
    lines += ['  printf("%d\\n", KVX_ATTENTION_ZEROED);', "  return 0;", "}"]
    (tmp_path / "s.c").write_text("\n".join(lines))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o",
                    str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()]
    want = []
    for _, struct in pairs:
        want.append(ctypes.sizeof(struct))
        want += [getattr(struct, field).offset for field, _ in struct._fields_]
    assert got == want + [_native.ATTENTION_ZEROED]


@pytest.mark.parametrize("struct, packed", [(_native.StoreDest, _native.STORE_DEST), (_native.RotateArgs, _native.ROTATE_ARGS),
                                            (_native.AttentionArgs, _native.ATTENTION_ARGS)])
def test_packed_structs_are_the_ctypes_structs(struct, packed):
    """A pack() of 1, 2, 3, ... reads back, field by field, as the ctypes struct's values in order."""
    def fields(s):
        for name, kind in s._fields_:
            value = getattr(s, name)
            if isinstance(value, ctypes.Structure):
                yield from fields(value)
            else:
                yield value

    assert packed.size == ctypes.sizeof(struct)
    n = len(packed.unpack(bytes(packed.size)))
    assert [int(v) for v in fields(struct.from_buffer_copy(packed.pack(*range(1, n + 1))))] == list(range(1, n + 1))


def test_rotary_angles():
    """position * base ** (-2p / r), and each way to stretch it."""
    plain = RotaryTable.build(50, 8, base=100.0, device="cpu").table.double()
    for p in range(4):
        angle = 37 * 100.0 ** (-2 * p / 8)
        assert abs(plain[37, p] - math.cos(angle)) < 1e-6 and abs(plain[37, 4 + p] - math.sin(angle)) < 1e-6
    linear = RotaryTable.build(50, 8, base=100.0, scaling={"type": "linear", "factor": 4}, device="cpu").table
    assert torch.allclose(linear[36].double(), plain[9], atol=1e-6)
    ntk = RotaryTable.build(50, 8, base=100.0, scaling={"type": "ntk", "factor": 3}, device="cpu").table.double()
    assert torch.allclose(ntk[:, 0], plain[:, 0])  # the fastest pair as it was ...
    assert abs(ntk[30, 3] - math.cos(30 * 100.0 ** (-6 / 8) / 3)) < 1e-6  # ... the slowest a third as fast
    yarn = RotaryTable.build(4000, 64, scaling={"type": "yarn", "factor": 4, "original_positions": 1000},
                             device="cpu").table.double()
    magnitude = 0.1 * math.log(4) + 1
    assert abs(yarn[3, 0] - magnitude * math.cos(3)) < 1e-6  # turns often: unchanged
    assert abs(yarn[2000, 31] - magnitude * math.cos(500 * 10000.0 ** (-62 / 64))) < 1e-6  # turns rarely: stretched
    for bad in ({"type": "other", "factor": 2}, {"type": "linear", "factor": 0.5}):
        with pytest.raises(ValueError):
            RotaryTable.build(4, 8, scaling=bad, device="cpu")
    with pytest.raises(ValueError, match="rotary_dim 7"):
        RotaryTable.build(4, 7, device="cpu")


@pytest.mark.parametrize("kind", ["absent", "does not load", "another torch"])
def test_a_marshalling_that_is_not_this_torch_s_is_left_alone(kind, monkeypatch):
    """The wrappers then marshal the calls themselves, and refuse and answer as ever."""
    import sys
    import types

    import lean_vllm_b200
    from lean_vllm_b200.attention import device

    class Broken:  # what the import system meets where a library asks for symbols that another torch had
        def find_spec(self, name, path=None, target=None):
            if name == "lean_vllm_b200._calls":
                raise ModuleNotFoundError(name) if kind == "absent" else ImportError("undefined symbol")

    monkeypatch.delattr(lean_vllm_b200, "_calls", raising=False)
    if kind == "another torch":
        other = types.SimpleNamespace(torch_version="1.0", bind=lambda *a: pytest.fail("bound"))
        monkeypatch.setattr(lean_vllm_b200, "_calls", other, raising=False)
        monkeypatch.setitem(sys.modules, "lean_vllm_b200._calls", other)
    else:
        monkeypatch.delitem(sys.modules, "lean_vllm_b200._calls", raising=False)
        monkeypatch.setattr(sys, "meta_path", [Broken(), *sys.meta_path])
    monkeypatch.setattr(device, "_bound", [])
    assert device.calls() is None
    with pytest.raises(ValueError, match="kv_lens must be"):
        paged_attention(**attention_args(kv_lens=torch.ones(4, dtype=torch.int32)))


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    from lean_vllm_b200 import build

    ran = []

    def compile(cmd, check):
        ran.append(cmd)
        open(build.CALLS + ".tmp", "w").close()

    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build, "CALLS_TORCH", str(tmp_path / "_calls.so.torch"))
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(build.subprocess, "run", compile)
    build.build_calls()
    build.build_calls()
    assert len(ran) == 1 and f'-DKVX_TORCH_VERSION="{torch.__version__}"' in ran[0]
    (tmp_path / "_calls.so.torch").write_text("1.0")
    build.build_calls()
    assert len(ran) == 2 and (tmp_path / "_calls.so.torch").read_text() == torch.__version__


def test_the_native_marshalling_loads_and_leaves_the_rest_to_the_wrappers():
    """Where it is built, the C++ module imports, binds, and answers None to what is not a plain call (CPU tensors)."""
    from lean_vllm_b200 import build

    if not os.path.exists(build.CALLS) or not os.path.exists(_native.LIB_PATH):
        pytest.skip("not built here")
    from lean_vllm_b200.attention.device import calls

    native = calls()
    a = attention_args()
    plain = (a["query"], a["k_cache"], a["v_cache"], a["block_tables"], a["kv_lens"], None, None, 1, 32, 0.0, 0, None,
             None, None, 0, 4096, 0, 0, 0)
    assert native.attention(*plain) is None
    for wrong in ((), plain[:-1], (None,) * 19, (*plain[:5], "x", *plain[6:]), (*plain[:7], 2**70, *plain[8:])):
        assert native.attention(*wrong) is None
    s = store_args()
    assert native.rotate_store(s["query"], s["key"], s["value"], s["k_cache"], s["v_cache"], s["slot_mapping"],
                               s["positions"], s["rotary"].table, False, None, None, 1e-6, 0, 0) is None
    assert native.rotate_store(*[None] * 14) is None and native.rotate_latents(*[3] * 11) is None
    with pytest.raises(TypeError):
        native.bind(1)
