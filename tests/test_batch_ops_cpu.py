"""The batched-decoding operators' argument checks and signatures, without a GPU. Every refusal happens before the first
CUDA call, so a zeroed block stands for the context here; no call below gets past the checks."""
import ctypes
import re

import pytest

import managedllama2_b200 as ml2
from managedllama2_b200 import _lib

E_INVALID = -1
P = 1 << 20  # stands for a device pointer, 16-byte aligned; never dereferenced


@pytest.fixture(scope="module")
def calls():
    lib = ml2.load()
    block = ctypes.create_string_buffer(4096)

    class Context:
        _lib = lib
        handle = ctypes.addressof(block)
        device = 0
    cfg = ml2.Config(256, 0, 1, 2, 2, 0, 0)
    keep = (ml2.BlockTables(Context, 16), ml2.QKNormRoPE(Context, cfg), ml2.PrefixAttention(Context, cfg, 16))  # set the argument types
    yield lib, Context.handle, (block, keep)


def call(function, arguments, values):
    return function(values.pop("ctx"), arguments.pack(*(values[name] for name in arguments.names)))


def refused(lib, rc, word):
    assert rc == E_INVALID, rc
    assert word in lib.ml2_last_error().decode(), lib.ml2_last_error()


@pytest.mark.parametrize("name,arguments", [("ml2_block_tables_args", _lib.BLOCK_TABLES), ("ml2_qk_norm_rope_args", _lib.QK_NORM_ROPE),
                                            ("ml2_prefix_attention_args", _lib.PREFIX_ATTENTION)])
def test_argument_structs_match_the_header(name, arguments):
    text = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    members = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    names, kinds = [], ""
    for line in members.split(";"):
        for one in filter(None, (x.strip() for x in line.split(","))):
            names.append(re.search(r"(\w+)$", one).group(1))
            kinds += "p" if "*" in one else "l" if "long long" in line or "size_t" in line else "f" if "float" in line else "i"
    assert names == arguments.names and kinds == arguments.kinds


TABLES = dict(ctx=None, lengths=P, new_lengths=2 * P, n_requests=4, page_size=16, table=3 * P, table_stride=8, free_pages=4 * P, free_count=5 * P,
              n_pages=64, lengths_out=6 * P, free_count_out=7 * P, query_start=8 * P, slots=9 * P, positions=10 * P, max_tokens=32,
              refused=11 * P, position_offset=0)


@pytest.mark.parametrize("change,word", [
    (dict(ctx=0), "null"), (dict(lengths=0), "null"), (dict(new_lengths=0), "null"), (dict(table=0), "null"), (dict(free_pages=0), "null"),
    (dict(free_count=0), "null"), (dict(lengths_out=0), "null"), (dict(free_count_out=0), "null"), (dict(query_start=0), "null"),
    (dict(refused=0), "null"), (dict(slots=0), "slots"), (dict(positions=0), "positions"), (dict(max_tokens=-1), "max_tokens"), (dict(max_tokens=2**31 - 1), "max_tokens"), (dict(slots=P + 2), "aligned"), (dict(table=P + 1), "aligned"),
    (dict(n_requests=0), "n_requests"), (dict(n_requests=8193), "n_requests"), (dict(page_size=0), "page_size"), (dict(page_size=24), "page_size"),
    (dict(page_size=2048), "page_size"), (dict(table_stride=0), "table_stride"), (dict(n_pages=0), "n_pages"),
    (dict(position_offset=-1), "32 bits"), (dict(position_offset=2**31 - 100), "32 bits"), (dict(n_pages=2**27), "32 bits"),
    (dict(table_stride=2**30), "32 bits"), (dict(lengths_out=2 * P), "own"), (dict(lengths=2 * P), "own"),
])
def test_block_tables_refusals(calls, change, word):
    lib, ctx, _ = calls
    a = dict(TABLES, ctx=ctx)
    a.update(change)
    refused(lib, call(lib.ml2_block_tables, _lib.BLOCK_TABLES, a), word)


ROPE = dict(ctx=None, dtype=0, query_out=P, query_out_stride=256, key_cache=P, value_cache=2 * P, cache_stride=256, cache_rows=64, query=2 * P,
            query_stride=256, key=3 * P, key_stride=256, value=4 * P, value_stride=256, query_weight=0, key_weight=0, positions=5 * P, slots=6 * P,
            n_tokens=3, n_heads=2, n_kv_heads=2, head_size=128, rotary_size=128, theta=10000.0, eps=1e-5)


@pytest.mark.parametrize("change,word", [
    (dict(ctx=0), "null"), (dict(key_cache=0), "null"), (dict(value_cache=0), "null"), (dict(query=0), "null"),
    (dict(key=0), "null"), (dict(value=0), "null"), (dict(query_out=0), "null"), (dict(positions=0), "null"), (dict(slots=0), "null"),
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(n_tokens=-1), "n_tokens"), (dict(n_heads=3), "multiple"), (dict(n_kv_heads=0), "multiple"),
    (dict(n_heads=0), "multiple"), (dict(head_size=72), "head_size"), (dict(head_size=272), "head_size"), (dict(head_size=0), "head_size"),
    (dict(rotary_size=8), "rotary_size"), (dict(rotary_size=144), "rotary_size"), (dict(rotary_size=-16), "rotary_size"),
    (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"), (dict(theta=float("inf")), "theta"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(query_weight=P), "together"), (dict(key_weight=P), "together"),
    (dict(query_out_stride=248), "shorter"), (dict(query_stride=0), "shorter"), (dict(key_stride=128), "shorter"), (dict(value_stride=255), "shorter"),
    (dict(cache_stride=128), "shorter"), (dict(cache_rows=0), "rows"), (dict(cache_rows=2**31), "rows"),
    (dict(query_stride=260), "aligned"), (dict(query=2 * P + 8), "aligned"), (dict(value_cache=P + 2), "aligned"),
    (dict(query_weight=P + 4, key_weight=P), "aligned"), (dict(slots=P + 2), "aligned"),
])
def test_qk_norm_rope_refusals(calls, change, word):
    lib, ctx, _ = calls
    a = dict(ROPE, ctx=ctx)
    a.update(change)
    refused(lib, call(lib.ml2_qk_norm_rope, _lib.QK_NORM_ROPE, a), word)


ATTN = dict(ctx=None, dtype=0, out=P, out_stride=256, lse=0, query=2 * P, query_stride=256, n_rows=4, prefix_key=P, prefix_value=2 * P,
            prefix_length=100, prefix_stride=256, key_cache=P, value_cache=2 * P, cache_stride=256, cache_rows=160, page_size=16, table=3 * P, table_stride=4, lengths=4 * P, query_start=5 * P, n_requests=4, max_length=64, n_heads=2, n_kv_heads=2,
            head_size=128, scale=0.1, workspace=6 * P, workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,word", [
    (dict(ctx=0), "null"), (dict(out=0), "null"), (dict(query=0), "null"),
    (dict(table=0), "null"), (dict(lengths=0), "null"), (dict(query_start=0), "null"), (dict(key_cache=0), "null"),
    (dict(prefix_value=0), "null"), (dict(dtype=7), "dtype"), (dict(n_rows=-1), "n_rows"), (dict(n_requests=0), "n_requests"),
    (dict(n_requests=8193), "n_requests"), (dict(n_heads=3), "multiple"), (dict(n_kv_heads=0), "multiple"), (dict(head_size=96), "head_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=0), "page_size"), (dict(table_stride=0), "table_stride"), (dict(max_length=-1), "max_length"),
    (dict(max_length=65), "max_length"), (dict(cache_rows=0), "rows"), (dict(cache_rows=2**31), "rows"), (dict(prefix_length=-1), "rows"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(out_stride=128), "shorter"),
    (dict(query_stride=128), "shorter"), (dict(cache_stride=128), "shorter"), (dict(prefix_stride=128), "shorter"),
    (dict(query=P + 8), "aligned"), (dict(out=P + 2), "aligned"), (dict(out_stride=260), "aligned"), (dict(key_cache=P + 8), "aligned"),
    (dict(prefix_stride=258), "aligned"), (dict(cache_stride=2**30), "further apart"), (dict(prefix_stride=2**31), "further apart"), (dict(workspace=P + 8), "aligned"), (dict(table=P + 2), "aligned"), (dict(lse=P + 1), "aligned"),
])
def test_prefix_attention_refusals(calls, change, word):
    lib, ctx, _ = calls
    a = dict(ATTN, ctx=ctx)
    a.update(change)
    refused(lib, call(lib.ml2_prefix_attention, _lib.PREFIX_ATTENTION, a), word)


@pytest.mark.parametrize("change,word", [
    (dict(ctx=0), "null"), (dict(bytes=0), "null"), (dict(n_rows=-1), "n_rows"), (dict(n_requests=0), "n_requests"), (dict(prefix=-1), "prefix"),
    (dict(max_length=-1), "max_length"), (dict(n_heads=3), "multiple"), (dict(head_size=32), "head_size"),
])
def test_prefix_attention_workspace_refusals(calls, change, word):
    lib, ctx, _ = calls
    n = ctypes.c_size_t()
    a = dict(ctx=ctx, n_rows=4, n_requests=4, prefix=100, max_length=64, n_heads=2, n_kv_heads=2, head_size=128, bytes=ctypes.addressof(n))
    a.update(change)
    kinds = [ctypes.c_void_p] + [ctypes.c_int] * 7 + [ctypes.c_void_p]
    refused(lib, lib.ml2_prefix_attention_workspace(*(k(v) for k, v in zip(kinds, a.values()))), word)


def test_missing_argument_structs_are_refused(calls):
    lib, ctx, _ = calls
    for function in (lib.ml2_block_tables, lib.ml2_qk_norm_rope, lib.ml2_prefix_attention):
        refused(lib, function(ctx, None), "null")
        refused(lib, function(None, None), "null")
