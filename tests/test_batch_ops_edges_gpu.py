"""Edges of the batched-decoding operators: what a call may hold beyond the ordinary (long flat tails under a peak, scales of
zero, broken tables, request counts around a limit of the launch) and memory that a call must leave alone."""
import ctypes
import math
import os
import random
import subprocess
import sys
import threading

import pytest
import torch

import managedllama2_b200 as ml2
import test_batch_ops_gpu as base
from test_batch_ops_gpu import Batch, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ml2.CudaContext(0)
    c.set_wait_limit(2 * 10**9)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def clean(ctx):
    yield
    assert ctx.status() == (0, 0)


# ---- many small weights under one large one --------------------------------------------------------------------------------
# One key scores 0 powers of two and has values of 0, all others score -25.0625 and have values of 1: next to a weight of 1
# theirs are less than half of fp16's smallest number, but together they are the output, keys * 2^-25.0625 and a little less.
# A reference point at least 2^7 below the largest score leaves them a rounding of at most 2^-32 each. The rest is relative to
# the output: half a step of its own, 2^-11; 32-bit sums of keys / 8 weights (2^-24 each) and of keys / 16 products (2^-23).
FLAT, PEAK_ROOM = -25.0625, 7


def flat_tail(rows, columns):
    k, v = torch.zeros(rows, columns, device="cuda", dtype=torch.float16), torch.ones(rows, columns, device="cuda", dtype=torch.float16)
    k[1:, ::64] = FLAT
    v[0] = 0
    return k, v


def check_flat_tail(out, lse, keys):
    tail = (keys - 1) * 2.0 ** FLAT
    want = tail / (1 + tail)
    bound = keys * 2.0 ** (-25 - PEAK_ROOM) + want * (2.0 ** -11 + keys / 8 * 2.0 ** -24 + keys / 16 * 2.0 ** -23) + 2.0 ** -25
    worst = (out.double() - want).abs().max().item()
    assert worst <= bound, "off by %.3g, %.3g allowed" % (worst, bound)
    assert (lse.double() - math.log1p(tail)).abs().max().item() <= keys / 8 * 2.0 ** -24 + 2.0 ** -20


@pytest.mark.parametrize("rows", [1, 130])
def test_attention_long_flat_tail_in_blocks(ctx, rows):
    """As many key heads as SMs: one block walks through most of a head's keys."""
    heads, keys = 148, 65536
    pk, pv = flat_tail(keys, heads * 64)
    q = torch.zeros(rows, heads * 64, device="cuda", dtype=torch.float16)
    q[:, ::64] = 1
    own = torch.zeros(16, heads * 64, device="cuda", dtype=torch.float16)
    op = ml2.PrefixAttention(ctx, ml2.Config(heads * 64, 0, 1, heads, heads, 0, 0), 16)
    ws = torch.empty(op.WorkspaceBytes(rows, 1, keys, 0), dtype=torch.uint8, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(rows, heads, device="cuda")
    op.Forward(out, q, pk, pv, own, own, ints([[0]]), ints([0]), ints([0, rows]), ws, 0, lse, math.log(2.0))
    check_flat_tail(out, lse, keys)


def test_attention_long_flat_tail_in_own_pages(ctx):
    """As many requests and key heads as warps, all over the same pages: one warp walks through most of a request's keys."""
    heads, requests, keys, page = 4, 296, 65536, 64
    k, v = flat_tail(keys, heads * 64)
    q = torch.zeros(requests, heads * 64, device="cuda", dtype=torch.float16)
    q[:, ::64] = 1
    table = torch.arange(keys // page, device="cuda", dtype=torch.int32).repeat(requests, 1)
    op = ml2.PrefixAttention(ctx, ml2.Config(heads * 64, 0, 1, heads, heads, 0, 0), page)
    ws = torch.empty(op.WorkspaceBytes(requests, requests, 0, keys), dtype=torch.uint8, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(requests, heads, device="cuda")
    op.Forward(out, q, None, None, k, v, table, ints([keys] * requests), ints(list(range(requests + 1))), ws, keys, lse, math.log(2.0))
    check_flat_tail(out, lse, keys)


# ---- scores so large that neighbouring 32-bit numbers are far apart ------------------------------------------------------------
@pytest.mark.parametrize("prefix", [300, 1500])
@pytest.mark.parametrize("rows", [1, 3, 70, 200])
@pytest.mark.parametrize("dtype,size,scale", [("fp16", 60000.0, 1.0), ("fp16", 60000.0, None), ("fp16", 60000.0, -1.0), ("bf16", 1e18, 1.0), ("bf16", 1e18, -0.37),
                                              ("fp16", 2000.0, 1.0), ("fp16", 300.0, 0.7)])
def test_attention_huge_scores_give_the_key_that_has_the_largest(ctx, dtype, size, scale, rows, prefix):
    """The largest score is twice the next: its key has weight 1 and the others none, whichever tile they lie in."""
    b = Batch(29, dtype, 4, 2, 64, 16, prefix, [20] * rows, [1] * rows)
    b.q[:] = size
    sign = -1.0 if scale is not None and scale < 0 else 1.0
    b.pk[:] = (torch.rand(prefix, 1, device="cuda") * 0.45 * size * sign).to(b.t)
    b.pk[prefix // 2] = size * sign
    b.k[torch.cat(b.rows)] = sign * size / 2
    out, z = b.call(ctx, scale=scale)
    want = b.pv[prefix // 2].reshape(2, 1, 64).expand(2, 2, 64).reshape(1, -1)
    assert torch.equal(out, want.expand_as(out))
    # 64 products, then the scale: half a step each, and a step at the reference point
    score = 64 * float(torch.tensor(size, dtype=b.t)) ** 2 * (64 ** -0.5 if scale is None else abs(scale))
    assert ((z.double() - score).abs().max() <= 80 * 2.0 ** -24 * score).item()


# ---- scales next to zero -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("prefix", [300, 1500])  # by runs, by blocks
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-39, -1e-39])
def test_attention_scale_of_zero_and_below_the_normal_numbers(ctx, prefix, scale):
    """Products of size 10^37: a scale of zero makes every weight the same, one of 10^-39 nearly so."""
    b = Batch(13, "bf16", 2, 1, 64, 16, prefix, [20] * 70, [1] * 70, sigma=1.0)
    b.q[:] = (torch.sign(b.q) * 1e18).to(b.t)
    b.pk[:] = (torch.sign(b.pk) * 5e17).to(b.t)
    b.k[torch.cat(b.rows)] = (torch.sign(b.k[torch.cat(b.rows)]) * 5e17).to(b.t)
    b.check(ctx, scale=scale)


@pytest.mark.parametrize("prefix", [300, 1500])
def test_attention_scale_of_zero_times_infinity_is_nan(ctx, prefix):
    b = Batch(13, "bf16", 2, 2, 64, 16, prefix, [20] * 70, [1] * 70)
    b.q[:, 0] = 1.0
    b.pk[3, 0] = float("-inf")
    b.q[5, 70], b.q[6, 127] = float("inf"), float("nan")
    out, z = b.call(ctx, scale=0.0)
    assert bool(out[:, :64].isnan().all()) and bool(z[:, 0].isnan().all())
    fine = torch.ones(70, dtype=torch.bool, device="cuda")
    fine[5:7] = False
    assert bool(out[fine, 64:].isfinite().all()) and bool(out[5:7].isnan().all()) and bool(z[5:7].isnan().all())


# ---- block tables: pages that are none -----------------------------------------------------------------------------------------
def step_with(ctx, table, free, old, new, page=4, rows=16):
    op, n = ml2.BlockTables(ctx, page), len(old)
    got = dict(table=ints(table), free=ints(free), count=ints([sum(x != -9 for x in free)]), lengths=ints(old), start=ints([0] * (n + 1)),
               slots=ints([7] * rows), positions=ints([7] * rows), refused=ints([7] * n))
    op.Forward(got["lengths"], ints(new), got["table"], got["free"], got["count"], got["lengths"], got["count"], got["start"], got["slots"],
               got["positions"], got["refused"])
    return {k: v.tolist() for k, v in got.items()}


@pytest.mark.parametrize("bad", [-1, 8, 2**31 - 1, -2**31])
def test_block_tables_pages_given_back_that_are_none_stay_off_the_stack(ctx, bad):
    """Request 1 gives back three pages, the middle one of which is none; request 0 takes what is free, in order."""
    got = step_with(ctx, [[0, -1, -1], [1, bad, 2], [3, 4, -1]], [5] + [-9] * 7, [4, 12, 8], [12, 0, 4])
    with pytest.raises(ml2.Ml2Error, match="page of request 1"):
        ctx.status()
    # pushed on 5: 1 and 2 of request 1, 4 of request 2; taken: 4, then 2
    assert got["free"][:4] == [5, 1, 2, 4] and got["count"] == [2]
    assert got["table"][0] == [0, 4, 2] and got["lengths"] == [12, 0, 4] and got["refused"] == [0, 0, 0]
    assert got["slots"][:8] == [16, 17, 18, 19, 8, 9, 10, 11] and got["slots"][8:] == [-1] * 8


def test_block_tables_pages_that_are_none_do_not_count_as_free(ctx):
    """Two of three pages given back are none: the one that is left serves request 0 alone."""
    got = step_with(ctx, [[0, -1], [1, -1], [-1, 9]], [-9] * 8, [4, 4, 8], [5, 5, 0])
    with pytest.raises(ml2.Ml2Error, match="page of request 2"):
        ctx.status()
    assert got["refused"] == [2, 2, 0] and got["count"] == [0] and got["slots"] == [-1] * 16 and got["lengths"] == [4, 4, 0]
    got = step_with(ctx, [[0, -1], [1, -1], [-1, 6]], [-9] * 8, [4, 4, 8], [5, 5, 0])
    with pytest.raises(ml2.Ml2Error, match="page of request 2"):
        ctx.status()
    assert got["refused"] == [0, 2, 0] and got["count"] == [0] and got["slots"][:2] == [24, -1] and got["table"][0] == [0, 6]


def test_block_tables_pages_taken_that_are_none_are_entered_as_none(ctx):
    got = step_with(ctx, [[0, -1], [1, -1]], [2, 8] + [-9] * 6, [4, 4], [6, 5])
    with pytest.raises(ml2.Ml2Error, match="page of request 0"):
        ctx.status()
    assert got["table"] == [[0, -1], [1, 2]] and got["slots"][:3] == [-1, -1, 8] and got["count"] == [0]


@pytest.mark.parametrize("n", [1, 40, 1500])
def test_block_tables_many_broken_pages(ctx, n):
    """Every other page of requests that end is none; the rest lies on the stack in order of request and page."""
    rng = random.Random(n)
    width, page = 5, 4
    ids = list(range(n * width))
    rng.shuffle(ids)
    table = [[ids.pop() if (r + i) % 2 else -1 - i for i in range(width)] for r in range(n)]
    old, new = [width * page] * n, [rng.randint(0, width * page) for _ in range(n)]
    free = [-9] * (n * width)
    got = step_with(ctx, table, free, old, new, page)
    want = [table[r][i] for r in range(n) for i in range(-(-new[r] // page), width) if (r + i) % 2]
    broken = any((r + i) % 2 == 0 for r in range(n) for i in range(-(-new[r] // page), width))
    assert broken == (n > 1 or new[0] <= 16)
    if broken:
        with pytest.raises(ml2.Ml2Error, match="page of request"):
            ctx.status()
    assert got["free"][:len(want)] == want and got["count"] == [len(want)] and got["lengths"] == new


# ---- block tables: request counts around the launch's limit of shared memory ---------------------------------------------------
def tables_of_many_requests():
    c = ml2.CudaContext(0)
    for n in (3030, 3038, 3039, 3055, 3071, 3100):
        plain, dev = base.tables_setup(random.Random(n), n, 16, 2, 2 * n + 5)
        new = [min(x + 1, 32) for x in plain.old]
        base.tables_step(c, plain, dev, new, n, 0)
    assert c.status() == (0, 0)
    c.close()


def test_block_tables_around_the_default_shared_memory_of_a_launch():
    """In a process of its own: a larger call made before would have raised the limit."""
    run_alone("tables_of_many_requests")


def run_alone(name):
    """A function of this file in a process of its own."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = %r; import test_batch_ops_edges_gpu as t; t.%s()" % ([here, os.path.dirname(here)], name)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ---- memory that a call leaves alone -------------------------------------------------------------------------------------------
def guarded(shape, fill, dtype, before=64, behind=4096):
    """A tensor in the middle of a buffer that holds `fill` everywhere, and a check of what lies around it."""
    n = math.prod(shape)
    buffer = torch.full((before + n + behind,), fill, dtype=dtype, device="cuda")

    def untouched():
        return bool((buffer[:before] == fill).all()) and bool((buffer[before + n:] == fill).all())
    return buffer[before:before + n].view(shape), untouched


def guarded_call(ctx, b, scale=None, max_length=None):
    """A call whose workspace ends where it has to; nothing behind or before any output changes."""
    op = ml2.PrefixAttention(ctx, b.cfg, b.page)
    rows, most, width = b.q.shape[0], max(b.own) if max_length is None else max_length, b.heads * b.head
    need = op.WorkspaceBytes(rows, len(b.own), b.prefix, most)
    ws, ws_fine = guarded((need,), 0xA5, torch.uint8, behind=1 << 20)
    wide, out_fine = guarded((rows, width + 16), 7.0, b.t)
    z, z_fine = guarded((rows, b.heads), 7.0, torch.float32)
    op.Forward(wide[:, :width], b.q, b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, most, z, scale)
    assert ws_fine(), "written outside the workspace"
    assert out_fine() and bool((wide[:, width:] == 7.0).all()), "written outside the output"
    assert z_fine(), "written outside the log sums"
    return wide[:, :width], z


@pytest.mark.parametrize("heads,kv,head,prefix,requests,length,queries", [
    (1, 1, 64, 0, 1, 1, 1), (1, 1, 128, 5000, 1, 30, 1), (40, 40, 128, 4096, 1, 64, 1), (40, 40, 64, 1024, 17, 30, 1), (3, 1, 64, 1025, 129, 7, 1),
    (64, 1, 128, 1100, 3, 40, 2), (71, 1, 64, 1500, 5, 90, 20), (71, 1, 64, 300, 5, 90, 20), (200, 2, 64, 100, 2, 40, 9), (5, 5, 128, 0, 300, 20, 3),
    (8, 8, 64, 2000, 4, 700, 300), (8, 2, 128, 1600, 33, 60, 30), (148, 148, 64, 1024, 1, 1, 1), (1, 1, 64, 40000, 130, 3, 1), (12, 3, 64, 1, 1000, 4, 4)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_writes_nothing_around_its_outputs_and_workspace(ctx, heads, kv, head, prefix, requests, length, queries, dtype):
    b = Batch(prefix + heads, dtype, heads, kv, head, 16, prefix, *base.ragged(heads + requests, requests, length, queries), extra_rows=3)
    out, z = guarded_call(ctx, b)
    want, lse, tol, tol_lse = b.want()
    total = sum(b.count)
    assert bool(((out[:total].double() - want).abs() <= tol).all()) and bool(((z[:total].double() - lse).abs() <= tol_lse).all())
    assert bool((out[total:] == 7.0).all()) and bool((z[total:] == 7.0).all())
    # fewer query rows than the call has room for, as a replayed graph may meet them
    for k in (0, requests // 2):
        b.start[k + 1:] = b.start[k].item()
        out, z = guarded_call(ctx, b)
        rows = int(b.start[k])
        assert bool(((out[:rows].double() - want[:rows]).abs() <= tol[:rows]).all()) and bool((out[rows:] == 7.0).all()) and bool((z[rows:] == 7.0).all())


@pytest.mark.parametrize("prefix", [0, 30, 1200])
@pytest.mark.parametrize("start", [[0, 3, 1, 2], [1, 1, 2, 3], [5, 6, 7, 8], [0, 1, 2, 2**31 - 1], [-5, 0, 1, 2], [0, -1, -2, -3], [0, 3, 0, 3],
                                   [0, 2, 2, -2**31]])
def test_attention_query_rows_out_of_order_write_nothing_around(ctx, start, prefix):
    b = Batch(4, "fp16", 4, 2, 64, 16, prefix, [40, 40, 3], [1, 1, 1])
    b.start = ints(start)
    guarded_call(ctx, b)
    with pytest.raises(ml2.Ml2Error, match="length or the query rows of request"):
        ctx.status()


def test_attention_rows_claimed_by_many_requests_have_the_prefix_alone(ctx):
    """Every other request claims all 2048 rows, with 2^22 own tokens each: 2^32 tiles in all, where a call that is in order has
    2^27 at most. Nobody has own tokens then, and the call is reported."""
    requests, rows, page, prefix = 128, 2048, 1024, 30
    b = Batch(5, "fp16", 2, 2, 64, page, prefix, [1] * requests, [rows // requests] * requests)
    alone = Batch(5, "fp16", 2, 2, 64, page, prefix, [0] * requests, [rows // requests] * requests)
    alone.q, alone.pk, alone.pv = b.q, b.pk, b.pv
    want, lse, tol, tol_lse = alone.want()
    b.table = torch.zeros(requests, 4096, dtype=torch.int32, device="cuda")
    b.lengths = ints([4096 * page] * requests)
    b.start = ints([0, rows] * (requests // 2) + [rows])
    out, z = guarded_call(ctx, b, max_length=4096 * page)
    with pytest.raises(ml2.Ml2Error, match="length or the query rows of request"):
        ctx.status()
    assert bool(((out.double() - want).abs() <= tol).all()) and bool(((z.double() - lse).abs() <= tol_lse).all())


def test_tables_write_nothing_around_their_arrays(ctx):
    rng = random.Random(3)
    for n, page, width, rows in ((1, 16, 3, 1), (7, 4, 5, 60), (300, 16, 4, 1500), (1100, 8, 6, 9000), (40, 2, 700, 20000)):
        plain, dev = base.tables_setup(rng, n, page, width, n * width + 3)
        new = [rng.randint(0, width * page) for _ in range(n)]
        arrays = {k: guarded(v.shape, 77, torch.int32) for k, v in dev.items()}
        for k, v in dev.items():
            arrays[k][0].copy_(v)
        for k, m in (("start", n + 1), ("slots", rows), ("positions", rows), ("refused", n)):
            arrays[k] = guarded((m,), 77, torch.int32)
        a = {k: v[0] for k, v in arrays.items()}
        ml2.BlockTables(ctx, page).Forward(a["lengths"], ints(new), a["table"], a["free"], a["count"], a["lengths"], a["count"], a["start"],
                                           a["slots"], a["positions"], a["refused"], 5)
        refused, start, slots, positions = plain.step(new, width, rows, 5)
        assert a["refused"].tolist() == refused and a["start"].tolist() == start and a["slots"].tolist() == slots and a["positions"].tolist() == positions
        assert all(v[1]() for v in arrays.values()), [k for k, v in arrays.items() if not v[1]()]


# ---- a model on the same context -----------------------------------------------------------------------------------------------
def small_model(c):
    cfg = ml2.Config(256, 768, 2, 2, 2, 512, 64)
    tr = ml2.Transformer(cfg, ml2.synthetic_weights(c, cfg, seed=3, sigma=1.0), c)
    tr.set_tokens([7, 99, 300, 41])
    return tr


def busy(stream):
    """About 20 ms of nothing on a stream."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(40_000_000)


@pytest.mark.parametrize("own_stream", [False, True])
def test_operators_run_on_the_callers_stream_after_a_model_has_run(own_stream):
    """Their inputs come late, on the caller's stream: a launch on the stream of the model, which is idle, would miss them."""
    c = ml2.CudaContext(0)
    tr = small_model(c)
    stream = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
    if own_stream:
        c.set_stream(stream.cuda_stream)
    b = Batch(6, "fp16", 4, 2, 128, 16, 300, [20] * 5, [1] * 5)
    n, head = 5, 128
    kc, vc = torch.zeros(16, 2 * head, device="cuda").half(), torch.zeros(16, 2 * head, device="cuda").half()
    tables, norm, attend = ml2.BlockTables(c, 16), ml2.QKNormRoPE(c, b.cfg), ml2.PrefixAttention(c, b.cfg, 16)
    ws = torch.empty(attend.WorkspaceBytes(n, n, 300, 20), dtype=torch.uint8, device="cuda")
    late = dict(q=b.q.clone(), new=ints([3] * n), positions=ints(list(range(n))), slots=ints([9, 3, 5, 0, 1]))
    now = {k: torch.zeros_like(v) for k, v in late.items()}
    out, z, turned = torch.zeros(n, 4 * head, device="cuda").half(), torch.zeros(n, 4, device="cuda"), torch.zeros(n, 4 * head, device="cuda").half()
    t = dict(lengths=ints([0] * n), table=ints([[-1]] * n), free=ints(list(range(n))), count=ints([n]), start=ints([0] * (n + 1)),
             slots=ints([7] * 15), positions=ints([7] * 15), refused=ints([7] * n))

    def calls():
        tables.Forward(t["lengths"], now["new"], t["table"], t["free"], t["count"], t["lengths"], t["count"], t["start"], t["slots"], t["positions"],
                       t["refused"])
        norm.Forward(turned, kc, vc, now["q"], b.pk[:n], b.pv[:n], None, None, now["positions"], now["slots"])
        attend.Forward(out, now["q"], b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, 20, z)
    torch.cuda.synchronize()
    for first in ("tables", "norm", "attend"):  # each of them the first call after the model
        for v in now.values():
            v.zero_()
        t["lengths"].zero_()
        t["count"].fill_(n)
        torch.cuda.synchronize()
        tr.Forward(0, 1, False)
        tr.synchronize()
        busy(stream)
        with torch.cuda.stream(stream):
            for k, v in late.items():
                now[k].copy_(v)
            if first == "norm":
                norm.Forward(turned, kc, vc, now["q"], b.pk[:n], b.pv[:n], None, None, now["positions"], now["slots"])
            elif first == "attend":
                attend.Forward(out, now["q"], b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, 20, z)
            calls()
            got = out.clone(), z.clone(), kc.clone(), t["slots"].clone()
        stream.synchronize()
        want, lse, tol, tol_lse = b.want()
        assert bool(((got[0].double() - want).abs() <= tol).all()) and bool(((got[1].double() - lse).abs() <= tol_lse).all()), first
        assert bool((got[2][[9, 3, 5, 0, 1]] != 0).any(1).all()) and bool((got[2][[2, 4, 6, 7, 8]] == 0).all()), first
        assert got[3].tolist() == [16 * (n - 1 - r) + i for r in range(n) for i in range(3)], first
    assert c.status() == (0, 0)
    tr.close()
    c.close()


def test_operators_follow_what_a_model_has_queued():
    """The prompt is still under way when its rows are asked for as the prefix."""
    c = ml2.CudaContext(0)
    tr = small_model(c)
    ptr = ctypes.c_void_p()
    ml2._lib.check(tr.lib.ml2_model_stream(tr.handle, ctypes.byref(ptr)))
    rs = tr.runstate_ptrs()

    class Rows:
        def __init__(self, at):
            self.__cuda_array_interface__ = {"shape": (64, 256), "typestr": "<f2", "data": (at, False), "version": 2}
    b = Batch(12, "fp16", 2, 2, 128, 16, 4, [4, 30, 1], [1, 1, 1])
    b.pk, b.pv = (torch.as_tensor(Rows(p), device="cuda")[:4] for p in (rs.key_cache, rs.value_cache))
    b.pk.zero_()
    b.pv.zero_()
    b.call(c)
    torch.cuda.synchronize()
    busy(torch.cuda.ExternalStream(ptr.value))
    for pos in range(4):
        tr.Forward(pos, pos + 1, False)
    out, z = b.call(c)
    got, lse = out.clone(), z.clone()
    torch.cuda.synchronize()
    assert bool((b.pk != 0).any(1).all())
    want, want_lse, tol, tol_lse = b.want()
    assert bool(((got.double() - want).abs() <= tol).all()) and bool(((lse.double() - want_lse).abs() <= tol_lse).all())
    assert c.status() == (0, 0)
    tr.close()
    c.close()


def test_a_captured_call_after_a_model_has_run_lands_on_the_callers_stream():
    c = ml2.CudaContext(0)
    tr = small_model(c)
    b = Batch(6, "fp16", 4, 2, 128, 16, 1300, [20] * 5, [1] * 5)
    want, lse = b.call(c)
    op = ml2.PrefixAttention(c, b.cfg, 16)
    ws = torch.empty(op.WorkspaceBytes(5, 5, 1300, 20), dtype=torch.uint8, device="cuda")
    out, z = torch.zeros(5, 512, device="cuda").half(), torch.zeros(5, 4, device="cuda")
    s = torch.cuda.Stream()
    c.set_stream(s.cuda_stream)
    tr.Forward(0, 1, False)
    tr.synchronize()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        op.Forward(out, b.q, b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, 20, z)
    assert bool((out == 0).all())
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(z, lse) and c.status() == (0, 0)
    del g
    tr.close()
    c.close()


# ---- waits that run out ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,head,prefix,requests", [(64, 8, 128, 16384, 128), (40, 40, 128, 4096, 64), (8, 8, 64, 20000, 1), (37, 37, 64, 1100, 150)])
def test_attention_that_gives_up_waiting_is_reported_and_leaves_a_model_alone(heads, kv, head, prefix, requests):
    """With a limit of 1000 cycles waits for keys that come from memory run out (of a small prefix that is in the cache none
    need to). The call comes to its end, is reported by ``status``, writes nothing outside its outputs, and neither a model
    of the same context nor the next call suffers. One that is not reported is right."""
    c = ml2.CudaContext(0)
    tr = small_model(c)
    b = Batch(3, "fp16", heads, kv, head, 16, prefix, [20] * requests, [1] * requests)
    want, lse = b.call(c)
    reports = 0
    for _ in range(3):
        c.set_wait_limit(1000)
        out, z = guarded_call(c, b)
        c.synchronize()
        c.set_wait_limit(2 * 10**9)
        tr.Forward(0, 1, False)
        tr.synchronize()
        try:
            c.status()
        except ml2.Ml2Error as e:
            reports += 1
            assert "prefix_attention: a wait of block" in str(e)
        else:
            assert torch.equal(out, want) and torch.equal(z, lse)
        assert c.status() == (0, 0)
        out, z = b.call(c)
        assert torch.equal(out, want) and torch.equal(z, lse)
    assert reports or requests < 128 or prefix < 16384  # 220 tiles a block: it waits for every ring slot
    tr.close()
    c.close()


# ---- calls from several threads --------------------------------------------------------------------------------------------------
def first_calls_from_threads():
    cases = []
    for i in range(4):
        c, s = ml2.CudaContext(0), torch.cuda.Stream()
        b = Batch(40 + i, ("fp16", "bf16")[i & 1], 4, 2, (64, 128)[i >> 1], 16, 1100 + i, *base.ragged(i, 20, 60, 2))
        op = ml2.PrefixAttention(c, b.cfg, 16)
        ws = torch.empty(op.WorkspaceBytes(b.q.shape[0], 20, b.prefix, 60), dtype=torch.uint8, device="cuda")
        out = torch.zeros(b.q.shape[0], 4 * b.head, dtype=b.t, device="cuda")
        c.set_stream(s.cuda_stream)
        cases.append((c, s, b, op, ws, out))
    torch.cuda.synchronize()
    errors = []

    def calls(c, s, b, op, ws, out):
        try:
            for _ in range(50):
                op.Forward(out, b.q, b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, 60)
            c.synchronize()
            assert c.status() == (0, 0)
        except BaseException as e:
            errors.append(e)
    threads = [threading.Thread(target=calls, args=case) for case in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for c, s, b, op, ws, out in cases:
        want, _, tol, _ = b.want()
        assert bool(((out.double() - want).abs() <= tol).all())
        c.close()


def test_first_calls_of_a_process_from_threads_with_contexts_of_their_own():
    run_alone("first_calls_from_threads")


# ---- beside the operators of one sequence ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("pos", [0, 1, 17, 500, 2047, 4095])
@pytest.mark.parametrize("head", [64, 128])
def test_rotation_agrees_with_that_of_one_sequence(ctx, pos, head):
    """Keys of both meet in one softmax: a prefix that went through a model, own tokens through ``QKNormRoPE``. ``RoPERotation``
    (and the model's table, by the same expressions) takes the angle in 32 bits: a power and a quotient off by 4 steps of 2^-23
    and half of one, a product by another half, so the angle by 10 * 2^-24 of itself. Either result is rounded once to fp16."""
    heads = 4
    g = torch.Generator(device="cuda").manual_seed(pos + head)
    x = (torch.randn(2, heads * head, generator=g, device="cuda") * 1.5).half()
    cfg = ml2.Config(heads * head, 0, 1, heads, heads, 0, 0)
    kc, vc, out = (torch.zeros(1, heads * head, device="cuda").half() for _ in range(3))
    ml2.QKNormRoPE(ctx, cfg).Forward(out, kc, vc, x[:1], x[1:], x[1:], None, None, ints([pos]), ints([0]))
    q, k = x[:1].clone(), torch.zeros(pos + 1, heads * head, device="cuda").half()
    k[pos] = x[1]
    ml2.RoPERotation(ctx, cfg).Forward(q, k, heads, head, pos, 0, 10000.0)
    freq = torch.tensor([10000.0 ** (-2.0 * i / head) for i in range(head // 2)], dtype=torch.float64, device="cuda")
    for got, one, source in ((out[0], q[0], x[0]), (kc[0], k[pos], x[1])):
        want, slack = base.rope_want(source[None], None, heads, head, head, ints([pos]), 10000.0, 1e-5)
        y = source.double().reshape(heads, 2, head // 2).abs().sum(1, keepdim=True).expand(heads, 2, head // 2)
        bound = (2 * slack[0] + (y * (pos * freq * 10 * 2.0 ** -24)).reshape(-1)) * 1.001 + 2 * (2.0 ** -11 * want[0].abs() * 1.01 + 2.0 ** -25)
        assert bool(((got.double() - one.double()).abs() <= bound).all())


# ---- the largest and the odd calls -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("prefix", [0, 40, 1100])
def test_attention_of_as_many_requests_as_there_may_be(ctx, prefix):
    lengths, queries = base.ragged(3, 8192, 5, 2)
    lengths[5000], queries[5000] = 300, 7
    for r in range(0, 8192, 3):
        queries[r] = 0
    b = Batch(prefix, "bf16", 2, 1, 64, 16, prefix, lengths, queries, extra_rows=1)
    out, z = guarded_call(ctx, b)
    total = sum(queries)
    want, lse, tol, tol_lse = b.want()
    assert bool(((out[:total].double() - want).abs() <= tol).all()) and bool(((z[:total].double() - lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("pdl", [False, True])
def test_tables_of_many_rows_in_a_graph(ctx, pdl):
    """Two kernels, replayed with other lengths; each replay goes on from the last."""
    rng = random.Random(5)
    n, page, width, rows = 300, 16, 40, 20000
    plain, dev = base.tables_setup(rng, n, page, width, n * width)
    new = ints([0] * n)
    a = dict(start=ints([7] * (n + 1)), slots=ints([7] * rows), positions=ints([7] * rows), refused=ints([7] * n))
    op = ml2.BlockTables(ctx, page)

    def step():
        op.Forward(dev["lengths"], new, dev["table"], dev["free"], dev["count"], dev["lengths"], dev["count"], a["start"], a["slots"], a["positions"],
                   a["refused"], 9)
    new.copy_(dev["lengths"])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.set_stream(s.cuda_stream)
    ctx.set_pdl(pdl)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    finally:
        ctx.set_pdl(False)
        ctx.set_stream(0)
    for _ in range(4):
        want = [rng.choice([0, x, min(x + 1, width * page), rng.randint(0, width * page)]) for x in plain.old]
        new.copy_(ints(want))
        g.replay()
        refused, start, slots, positions = plain.step(want, width, rows, 9)
        torch.cuda.synchronize()
        assert a["refused"].tolist() == refused and a["start"].tolist() == start
        assert a["slots"].tolist() == slots and a["positions"].tolist() == positions and dev["lengths"].tolist() == plain.old
        assert dev["free"].tolist()[:len(plain.free)] == plain.free


@pytest.mark.parametrize("prefix,requests", [(300, 40), (1500, 40), (1500, 300)])
def test_attention_a_row_that_is_not_finite_spoils_itself_alone(ctx, prefix, requests):
    b = Batch(8, "fp16", 4, 2, 64, 16, prefix, [20] * requests, [1] * requests, extra_rows=2)
    clean_out, clean_lse = b.check(ctx)
    b.q[3, 70] = float("nan")
    b.q[17, 0] = float("inf")
    b.q[requests:] = float("nan")  # rows behind the last request
    b.pv[5, 1] = float("inf")      # one value of key head 0
    out, z = b.call(ctx)
    spoiled = torch.zeros(requests, 4, dtype=torch.bool, device="cuda")
    spoiled[3, 1] = spoiled[17, 0] = True
    assert torch.equal(z[:requests][~spoiled], clean_lse[:requests][~spoiled]) and bool(z[:requests][spoiled].isnan().all())
    rows, clean = out[:requests].reshape(requests, 4, 64), clean_out[:requests].reshape(requests, 4, 64)
    assert bool(rows[spoiled].isnan().all())
    same = (~spoiled)[:, :, None].expand(-1, -1, 64).clone()
    same[:, :2, 1] = False
    assert torch.equal(rows[same], clean[same])
    assert not bool(rows[:, :2, 1].isfinite().any())


def test_qk_norm_rope_positions_before_zero_turn_the_other_way(ctx):
    cfg = ml2.Config(2 * 96, 0, 1, 2, 1, 0, 0)
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k = (torch.randn(200, w, generator=g, device="cuda").bfloat16() for w in (192, 96))
    kc, vc = (torch.zeros(200, 96, device="cuda").bfloat16() for _ in range(2))
    positions, out = ints(list(range(-100, 99)) + [-2**31]), torch.zeros_like(q)
    ml2.QKNormRoPE(ctx, cfg, 32).Forward(out, kc, vc, q, k, k, None, None, positions, ints(list(range(200))))
    for got, x, heads in ((out, q, 2), (kc, k, 1)):
        want, slack = base.rope_want(x, None, heads, 96, 32, positions, 10000.0, 1e-5)
        base.near(got, want, slack, torch.bfloat16)


# ---- the bits of the weights -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bits", [("fp16", 22), ("bf16", 16)])
@pytest.mark.parametrize("prefix,rows,heads", [(0, 128, 1), (0, 300, 2), (300, 40, 2), (1023, 200, 1), (1500, 40, 2), (1100, 128, 1), (4200, 1, 2), (20000, 16, 4)])
@pytest.mark.parametrize("head", [64, 128])
def test_attention_small_difference_of_large_weights(ctx, dtype, bits, prefix, rows, heads, head):
    """Two keys have all of the weight, nearly the same, and opposite values: the output is half the difference of their scores,
    tanh(x / 2). Each weight, of at most 1, keeps `bits` bits; exponential, sum and quotient are off by 2^-21 together; the
    output by half a step. Rounded to 16 bits alone the weights were off by up to 2^-12 (fp16) and 2^-9 (bf16)."""
    own = 2 if prefix else 40
    b = Batch(1, dtype, heads, 1, head, 16, prefix, [own] * rows, [1] * rows)
    k, v = (b.pk, b.pv) if prefix else (b.k, b.v)
    places = (2, 9) if prefix else None  # in one tile: two warps, or blocks, would each have a weight of 1
    x = torch.arange(1, rows * heads + 1, device="cuda").reshape(rows, heads) / (64.0 * rows * heads)
    b.q.zero_()
    b.q.reshape(rows, heads, head)[:, :, 0] = x.to(b.t)
    x = b.q.reshape(rows, heads, head)[:, :, 0].double()
    b.q.reshape(rows, heads, head)[:, :, 1] = 1
    b.k[:], b.v[:] = 0, 0
    b.k[:, 1] = -100
    if prefix:
        k[:], v[:] = 0, 0
        k[:, 1] = -100
        k[places[0], 1], v[places[0]] = 0, 1
        k[places[1], :2], v[places[1]] = torch.tensor([-1.0, 0.0], device="cuda"), -1
    else:
        for r in range(rows):
            first, second = b.rows[r][3], b.rows[r][9]
            k[first, 1], v[first] = 0, 1
            k[second, :2], v[second] = torch.tensor([-1.0, 0.0], device="cuda"), -1
    out, z = b.call(ctx, scale=1.0)
    want = torch.tanh(x / 2)[:, :, None]
    off = (out.double().reshape(rows, heads, head) - want).abs()
    bound = base.step(b.t) * want * 1.01 + 2.0 ** -bits + 2.0 ** -21
    assert bool((off <= bound).all()), (off / bound).max().item()
    assert ((z.double() - torch.log1p(torch.exp(-x))).abs().max() <= 2.0 ** -20).item()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("prefix,rows", [(0, 3), (300, 40), (1500, 40), (4200, 1), (1500, 200)])
def test_attention_an_infinite_value_that_is_seen_is_infinite(ctx, dtype, prefix, rows):
    """Weights that are all the same, powers of two among them: none has a part that is zero."""
    b = Batch(2, dtype, 2, 2, 64, 16, prefix, [5] * rows, [1] * rows)
    b.q.zero_()
    v, at = (b.pv, prefix // 2) if prefix else (b.v, b.rows[0][2])
    v[at, 3], v[at, 70] = float("inf"), float("-inf")
    out, _ = b.call(ctx)
    seen = slice(None) if prefix else slice(0, 1)
    assert bool((out[seen, 3] == math.inf).all()) and bool((out[seen, 70] == -math.inf).all())
    out[seen, 3] = out[seen, 70] = 0
    assert bool(out.isfinite().all())


def test_a_model_goes_on_behind_the_operators_that_read_its_cache():
    """The next prompt overwrites the rows that a call on the caller's stream has still to read."""
    c = ml2.CudaContext(0)
    tr = small_model(c)
    rs = tr.runstate_ptrs()

    class Rows:
        def __init__(self, at):
            self.__cuda_array_interface__ = {"shape": (64, 256), "typestr": "<f2", "data": (at, False), "version": 2}
    b = Batch(12, "fp16", 2, 2, 128, 16, 4, [4, 30, 1], [1, 1, 1])
    b.pk, b.pv = (torch.as_tensor(Rows(p), device="cuda")[:4] for p in (rs.key_cache, rs.value_cache))
    for pos in range(4):
        tr.Forward(pos, pos + 1, False)
    want, lse = b.call(c)
    torch.cuda.synchronize()
    first = b.pk.clone()
    tr.set_tokens([411, 5, 17, 230])
    for _ in range(2):
        busy(torch.cuda.current_stream())
        out, z = b.call(c)  # behind 20 ms of nothing
        for pos in range(4):
            tr.Forward(pos, pos + 1, False)
        tr.synchronize()
        torch.cuda.synchronize()
        assert not torch.equal(b.pk, first)
        assert torch.equal(out, want) and torch.equal(z, lse)
        tr.set_tokens([7, 99, 300, 41])
        for pos in range(4):
            tr.Forward(pos, pos + 1, False)
        tr.synchronize()
        tr.set_tokens([411, 5, 17, 230])
    assert c.status() == (0, 0)
    tr.close()
    c.close()


def test_errors_of_operators_that_ran_before_a_model_are_reported():
    c = ml2.CudaContext(0)
    tr = small_model(c)
    b = Batch(4, "fp16", 2, 2, 64, 16, 30, [40, 40], [1, 1])
    b.table[1, 1] = 10**6
    busy(torch.cuda.current_stream())
    b.call(c)
    tr.Forward(0, 1, False)
    with pytest.raises(ml2.Ml2Error, match="page of request 1"):
        c.status()
    tr.synchronize()
    tr.close()
    c.close()


def check_guarded(ctx, b):
    out, z = guarded_call(ctx, b)
    total = sum(b.count)
    want, lse, tol, tol_lse = b.want()
    assert bool(((out[:total].double() - want).abs() <= tol).all()) and bool(((z[:total].double() - lse).abs() <= tol_lse).all())
    assert bool((out[total:] == 7.0).all()) and bool((z[total:] == 7.0).all())


@pytest.mark.parametrize("heads,kv,prefix,rows", [(65536, 1, 40, 2), (65536, 1, 1100, 2), (65536, 65536, 9, 1), (4096, 16, 1300, 3), (1, 1, 1000003, 3),
                                                  (2, 1, 1000003, 70)])
def test_attention_of_many_heads_and_of_a_prefix_of_a_million(ctx, heads, kv, prefix, rows):
    check_guarded(ctx, Batch(heads + prefix, "bf16", heads, kv, 64, 16, prefix, [20] * rows, [1] * rows, extra_rows=1))


@pytest.mark.parametrize("page", [1, 64, 1024])
def test_attention_of_long_requests(ctx, page):
    check_guarded(ctx, Batch(page, "fp16", 4, 2, 64, page, 50, [300001, 1, 70000], [3, 1, 40], extra_rows=1))


def test_tables_of_half_a_million_tokens_of_a_request(ctx):
    plain, dev = base.tables_setup(random.Random(3), 3, 1, 600000, 1800000)
    for new in ([600000, 0, 1], [5, 590001, 2], [0, 0, 600000]):
        base.tables_step(ctx, plain, dev, new, max(1, sum(max(0, b - a) for a, b in zip(plain.old, new)) + 3), 7)


def test_qk_norm_rope_of_many_tokens(ctx):
    tokens, cfg = 70001, ml2.Config(2 * 16, 0, 1, 2, 1, 0, 0)
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k = (torch.randn(tokens, w, generator=g, device="cuda").half() for w in (32, 16))
    w = (1 + torch.randn(16, generator=g, device="cuda") / 8).half()
    kc, vc = (torch.zeros(tokens + 5, 16, device="cuda").half() for _ in range(2))
    out, positions = torch.zeros_like(q), torch.arange(tokens, device="cuda", dtype=torch.int32) * 30000
    slots = torch.randperm(tokens + 5, generator=g, device="cuda")[:tokens].to(torch.int32)
    ml2.QKNormRoPE(ctx, cfg).Forward(out, kc, vc, q, k, k, w, w, positions, slots)
    for got, x, heads in ((out, q, 2), (kc[slots.long()], k, 1)):
        want, slack = base.rope_want(x, w, heads, 16, 16, positions, 10000.0, 1e-5)
        base.near(got, want, slack, torch.float16)
    assert torch.equal(vc[slots.long()], k)
