"""Edges of the batched-decoding operators' arguments, without a GPU."""
import ctypes

import pytest
import torch

import managedllama2_b200 as ml2
from managedllama2_b200 import _lib
from test_batch_ops_cpu import ATTN, P, ROPE, call, calls, refused  # noqa: F401  (calls is a fixture)


@pytest.mark.parametrize("scale", [3e38, -2.4e38])
def test_prefix_attention_refuses_a_scale_that_overflows_in_powers_of_two(calls, scale):  # noqa: F811
    lib, ctx, _ = calls
    refused(lib, call(lib.ml2_prefix_attention, _lib.PREFIX_ATTENTION, dict(ATTN, ctx=ctx, scale=scale)), "scale")


@pytest.mark.parametrize("name,arguments", [("ml2_block_tables_args", _lib.BLOCK_TABLES), ("ml2_qk_norm_rope_args", _lib.QK_NORM_ROPE),
                                            ("ml2_prefix_attention_args", _lib.PREFIX_ATTENTION)])
def test_packed_arguments_are_as_long_as_the_struct(name, arguments):
    """The library copies the whole struct, the bytes behind its last member among them."""
    kinds = {"p": ctypes.c_void_p, "l": ctypes.c_longlong, "i": ctypes.c_int, "f": ctypes.c_float}
    layout = type(name, (ctypes.Structure,), {"_fields_": [(n, kinds[k]) for n, k in zip(arguments.names, arguments.kinds)]})
    values = range(1, len(arguments.names) + 1)
    packed = arguments.pack(*values)
    assert len(packed) == ctypes.sizeof(layout)
    got = layout.from_buffer_copy(packed)
    assert [getattr(got, n) for n in arguments.names] == list(values)


def workspace(calls, **change):
    lib, ctx, _ = calls
    a = dict(n_rows=1, n_requests=1, prefix=0, max_length=0, n_heads=2, n_kv_heads=2, head_size=64)
    a.update(change)
    n = ctypes.c_size_t()
    rc = lib.ml2_prefix_attention_workspace(ctypes.c_void_p(ctx), *map(ctypes.c_int, a.values()), ctypes.byref(n))
    return rc, n.value


@pytest.mark.parametrize("name", ["prefix", "max_length"])
def test_prefix_attention_lengths_next_to_the_largest_int(calls, name):  # noqa: F811
    """Lengths are rounded up to whole tiles of 64 keys: 2^31 - 64 is the largest that can be."""
    lib, ctx, _ = calls
    for x in (2**31 - 63, 2**31 - 1):
        refused(lib, workspace(calls, **{name: x})[0], name)
    before = 0
    for x in (100, 2**20, 2**30, 2**31 - 64):
        rc, n = workspace(calls, **{name: x})
        assert rc == 0 and before <= n < 1 << 40
        before = n
    change = dict(prefix_length=2**31 - 1) if name == "prefix" else dict(max_length=2**31 - 1, table_stride=2**31 - 1, page_size=1)
    refused(lib, call(lib.ml2_prefix_attention, _lib.PREFIX_ATTENTION, dict(ATTN, ctx=ctx, **change)), name)


def test_qk_norm_rope_refuses_queries_over_themselves_with_another_stride(calls):  # noqa: F811
    """A row's result would lie over a row that another block has still to read."""
    lib, ctx, _ = calls
    for strides in ((256, 768), (768, 256)):
        a = dict(ROPE, ctx=ctx, query=P, query_out=P, query_stride=strides[0], query_out_stride=strides[1])
        refused(lib, call(lib.ml2_qk_norm_rope, _lib.QK_NORM_ROPE, a), "stride")


# ---- the modules' own checks, on CPU tensors: the call into the library is replaced ------------------------------------------------
@pytest.fixture()
def modules():
    lib = ml2.load()

    class Context:
        _lib, handle, device = lib, ctypes.c_void_p(0), -1  # the device number of CPU tensors
    cfg = ml2.Config(256, 0, 1, 2, 2, 0, 0)
    made = [ml2.BlockTables(Context, 16), ml2.QKNormRoPE(Context, cfg), ml2.PrefixAttention(Context, cfg, 16)]
    calls = []
    for m in made:
        m._call = lambda handle, packed: calls.append(packed) or 0
    return made + [calls]


def attention_arguments(**change):
    def half(*shape):
        return torch.zeros(*shape, dtype=torch.float16)

    def ints(*shape):
        return torch.zeros(*shape, dtype=torch.int32)
    a = dict(output=half(3, 256), query=half(3, 256), prefixKey=half(20, 256), prefixValue=half(20, 256), keyCache=half(64, 256),
             valueCache=half(64, 256), table=ints(2, 4), lengths=ints(2), queryStart=ints(3), workspace=half(4096), maxLength=40)
    a.update(change)
    return a


def test_prefix_attention_module_takes_prefix_key_and_value_together(modules):
    attend, calls = modules[2:]
    some, none = torch.zeros(20, 256, dtype=torch.float16), torch.zeros(0, 256, dtype=torch.float16)
    for both in ((some, some), (None, None), (none, none), (none, None), (None, none), (some[:1], some[:1])):
        attend.Forward(**attention_arguments(prefixKey=both[0], prefixValue=both[1]))
    assert len(calls) == 6
    for key, value in ((some, None), (None, some), (none, some), (some, none), (some, some[:5]), (some.view(-1), some),
                       (some, some.float()), (torch.zeros((), dtype=torch.float16), some)):
        with pytest.raises(ValueError, match="prefix"):
            attend.Forward(**attention_arguments(prefixKey=key, prefixValue=value))
    assert len(calls) == 6


@pytest.mark.parametrize("number", [2**31, -2**31 - 1, 2**70])
def test_modules_refuse_numbers_that_pass_32_bits(modules, number):
    tables, norm, attend, calls = modules
    ints = torch.zeros(64, dtype=torch.int32)
    with pytest.raises(ValueError, match="32 bits"):
        attend.Forward(**attention_arguments(maxLength=number))
    with pytest.raises(ValueError, match="32 bits"):
        tables.Forward(ints[:2], ints[:2], ints[:8].view(2, 4), ints, ints[:1], ints[:2], ints[:1], ints[:3], ints[:8], ints[:8], ints[:2], number)
    x = torch.zeros(2, 256, dtype=torch.float16)
    norm.rotarySize = number
    with pytest.raises(ValueError, match="32 bits"):
        norm.Forward(x, x, x, x, x, x, None, None, ints[:2], ints[:2])
    assert not calls
