"""Block tables, query / key norm with rotation and cache write, and shared-prefix attention against plain
implementations in 64 bits (or in whole numbers), and the three of them together.

Tolerances. A store to 16 bits is off by at most half a step: u = 2^-11 (fp16) or 2^-8 (bf16) of the value, and 2^-25 where
fp16 is subnormal. 32-bit arithmetic adds the terms derived at each comparison.
"""
import math
import random

import pytest
import torch

import managedllama2_b200 as ml2

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def ctx():
    c = ml2.CudaContext(0)
    c.set_wait_limit(2 * 10**9)  # about a second: a wait that never ends is an error status, not ten seconds
    yield c
    c.close()


@pytest.fixture(autouse=True)
def clean(ctx):
    yield
    assert ctx.status() == (0, 0)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- block tables ------------------------------------------------------------------------------------------------------
class Tables:
    """The step as it is described, one request after another."""

    def __init__(self, old, table, free, page):
        self.old, self.table, self.free, self.page = list(old), [list(r) for r in table], list(free), page

    def pages(self, x):
        return -(-x // self.page)

    def step(self, new, width, max_tokens, offset):
        n, refused = len(new), [0] * len(new)
        for r in range(n):
            if new[r] < 0 or self.old[r] < 0 or self.pages(new[r]) > width or self.pages(self.old[r]) > width:
                refused[r] = 1
        for r in range(n):
            if not refused[r] and new[r] < self.old[r]:
                for i in range(self.pages(new[r]), self.pages(self.old[r])):
                    self.free.append(self.table[r][i])
        have = len(self.free)
        tokens = need = 0
        for r in range(n):
            if refused[r] or new[r] <= self.old[r]:
                continue
            tokens += new[r] - self.old[r]
            if tokens > max_tokens:
                refused[r] = 3
                continue
            k = self.pages(new[r]) - self.pages(self.old[r])
            need += k
            if k and need > have:
                refused[r] = 2
        start, slots, positions = [0], [], []
        for r in range(n):
            if not refused[r] and new[r] > self.old[r]:
                for i in range(self.pages(self.old[r]), self.pages(new[r])):
                    self.table[r][i] = self.free.pop()
                for j in range(self.old[r], new[r]):
                    slots.append(self.table[r][j // self.page] * self.page + j % self.page)
                    positions.append(offset + j)
            if not refused[r]:
                self.old[r] = new[r]
            start.append(len(slots))
        pad = max_tokens - len(slots)
        return refused, start, slots + [-1] * pad, positions + [0] * pad


def tables_setup(rng, n, page, width, total):
    """Random lengths and a table of shuffled pages; returns the plain form and the device arrays."""
    ids = list(range(total))
    rng.shuffle(ids)
    old, table = [], []
    for _ in range(n):
        x = rng.randint(0, width * page)
        k = -(-x // page)
        if k > len(ids):
            x, k = 0, 0
        old.append(x)
        table.append([ids.pop() for _ in range(k)] + [-1] * (width - k))
    plain = Tables(old, table, ids, page)
    dev = dict(lengths=ints(old), table=ints(table), free=ints(ids + [-1] * (total - len(ids))), count=ints([len(ids)]))
    return plain, dev


def tables_step(ctx, plain, dev, new, max_tokens, offset, in_place=True):
    n, width = dev["table"].shape
    out = dict(start=ints([7] * (n + 1)), slots=ints([7] * max_tokens), positions=ints([7] * max_tokens), refused=ints([7] * n))
    lengths = dev["lengths"] if in_place else torch.full_like(dev["lengths"], 7)
    count = dev["count"] if in_place else torch.full_like(dev["count"], 7)
    op = ml2.BlockTables(ctx, plain.page)
    for _ in range(1 if in_place else 2):  # out of place, a repeated call gives the same again
        op.Forward(dev["lengths"], ints(new), dev["table"], dev["free"], dev["count"], lengths, count, out["start"], out["slots"],
                   out["positions"], out["refused"], offset)
    refused, start, slots, positions = plain.step(new, width, max_tokens, offset)
    assert out["refused"].tolist() == refused
    assert out["start"].tolist() == start
    assert out["slots"].tolist() == slots
    assert out["positions"].tolist() == positions
    assert lengths.tolist() == plain.old
    assert count.item() == len(plain.free)
    assert dev["free"].tolist()[:len(plain.free)] == plain.free
    for r, x in enumerate(plain.old):
        k = plain.pages(x) if 0 <= x <= width * plain.page else 0
        assert dev["table"][r].tolist()[:k] == plain.table[r][:k]
    dev["lengths"], dev["count"] = lengths, count


@pytest.mark.parametrize("n,page,width", [(1, 1, 5), (1, 1024, 2), (3, 16, 4), (33, 2, 9), (255, 16, 8), (1025, 32, 3), (8192, 16, 2)])
@pytest.mark.parametrize("in_place", [True, False])
def test_block_tables_steps(ctx, n, page, width, in_place):
    """Three steps of growth by one, growth by many, ends, truncations and nothing at all, all of which fit."""
    rng = random.Random(n * 31 + page)
    plain, dev = tables_setup(rng, n, page, width, n * width + 5)
    for kind in range(3):
        new = []
        for x in plain.old:
            what = rng.randint(0, 4)
            new.append(min(x + 1, width * page) if what == 0 else rng.randint(x, width * page) if what == 1 else 0 if what == 2 else
                       rng.randint(0, x) if what == 3 else x)
        grown = sum(max(0, b - a) for a, b in zip(plain.old, new))
        tables_step(ctx, plain, dev, new, grown + (0, 1, 37)[kind], (0, 4032, 1)[kind], in_place)


@pytest.mark.parametrize("n", [1, 2, 40, 700, 1500])
@pytest.mark.parametrize("short", ["pages", "tokens", "both"])
def test_block_tables_refuses_what_does_not_fit(ctx, n, short):
    rng = random.Random(n + len(short))
    page, width = 4, 6
    plain, dev = tables_setup(rng, n, page, width, 3 * n + 2)
    new = [rng.choice([x + 1, rng.randint(x, width * page), rng.randint(0, x), x, -1, width * page + 1]) for x in plain.old]
    new = [b if a < width * page or b != a + 1 else a for a, b in zip(plain.old, new)]
    grown = sum(b - a for a, b in zip(plain.old, new) if b > a and b <= width * page)
    if short != "tokens":  # most of the free pages are lost to somebody else
        plain.free = plain.free[:len(plain.free) // 4]
        dev["count"] = ints([len(plain.free)])
    tables_step(ctx, plain, dev, new, grown if short == "pages" else grown // 2, 3)


def test_block_tables_nothing_free_and_no_rows(ctx):
    plain, dev = tables_setup(random.Random(1), 4, 8, 3, 12)
    plain.free, dev["count"] = [], ints([0])
    tables_step(ctx, plain, dev, [min(x + 1, 24) for x in plain.old], 0, 0)


def test_block_tables_reports_broken_state(ctx):
    """A count of free pages that cannot be, more pages given back than there are, a page that is none: clamped or left out,
    and reported."""
    op = ml2.BlockTables(ctx, 4)
    start, refused, slots, positions = ints([0] * 3), ints([0] * 2), ints([0] * 8), ints([0] * 8)
    lengths, count = ints([4, 4]), ints([99])
    op.Forward(lengths, ints([5, 4]), ints([[0, -1], [1, -1]]), ints([2, 3]), count, lengths, count, start, slots, positions, refused)
    # two pages of room: the count is taken as 2, and page 3 that comes off the stack is none of the cache's two
    assert slots.tolist() == [-1] * 8 and count.item() == 1
    with pytest.raises(ml2.Ml2Error, match="count of free pages was 99"):
        ctx.status()
    lengths, count, free = ints([4, 4]), ints([2]), ints([2, 3])
    op.Forward(lengths, ints([0, 0]), ints([[0, -1], [1, -1]]), free, count, lengths, count, start, slots, positions, refused)
    assert count.item() == 2 and free.tolist() == [2, 3] and lengths.tolist() == [0, 0]
    with pytest.raises(ml2.Ml2Error, match="2 pages given back overflow"):
        ctx.status()
    lengths, count = ints([1, 1]), ints([0])
    op.Forward(lengths, ints([2, 2]), ints([[7, -1], [1, -1]]), ints([2, 3]), count, lengths, count, start, slots, positions, refused)
    assert slots.tolist() == [-1, 5] + [-1] * 6
    with pytest.raises(ml2.Ml2Error, match="page of request 0"):
        ctx.status()


# ---- norm, rotation and cache write ------------------------------------------------------------------------------------
def rope_want(x, weight, heads, head, rotary, positions, theta, eps):
    """64-bit result and the bound of the 32-bit arithmetic: a value is a sum of two products of factors that are each right
    to a few units of 2^-24 (the norm's square root and sum, the unit of the angle, the products): 32 units of |a| + |b|."""
    y = x.double().reshape(x.shape[0], heads, head)
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    half = rotary // 2
    freq = torch.tensor([theta ** (-2.0 * i / rotary) for i in range(half)], dtype=torch.float64, device="cuda")
    angle = positions.double()[:, None, None] * freq
    a, b = y[..., :half], y[..., half:rotary]
    out = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), y[..., rotary:]], -1)
    size = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), y[..., rotary:].abs()], -1)
    # the angle: a position below 2^31 times a frequency, in 64 bits after `half` products: half * 2^-53 of it
    slack = 2.0 ** -24 * 32 + angle.abs().max().item() * half * 2.0 ** -53 if half else 2.0 ** -24 * 32
    return out.reshape(x.shape[0], -1), slack * size.reshape(x.shape[0], -1)


def near(got, want, slack, dtype):
    off = (got.double() - want).abs()
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    bound = step(dtype) * (want.abs() + slack) + slack + tiny
    assert bool((off <= bound).all()), "off by %.3g of the bound" % (off / bound.clamp(min=1e-300)).max().item()


ROPES = [  # tokens, heads, kv heads, head, rotary, norm, fused, largest position
    (1, 1, 1, 16, 16, True, False, 1), (1, 32, 32, 128, 128, False, False, 4096), (3, 5, 5, 128, 128, True, True, 2**31 - 1),
    (7, 6, 2, 48, 16, True, True, 100), (2, 4, 1, 64, 64, True, False, 131072), (5, 3, 3, 80, 80, True, True, 50000),
    (64, 15, 5, 96, 64, True, True, 32768), (9, 4, 4, 112, 96, False, True, 1 << 20), (4, 8, 8, 256, 256, True, False, 1 << 20),
    (6, 2, 2, 128, 0, True, False, 10), (6, 2, 2, 240, 0, False, True, 10), (777, 8, 2, 128, 128, True, True, 8192), (300, 96, 12, 64, 32, True, False, 500),
]


@pytest.mark.parametrize("tokens,heads,kv,head,rotary,norm,fused,far", ROPES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_qk_norm_rope(ctx, tokens, heads, kv, head, rotary, norm, fused, far, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens * head + rotary)
    t = TYPES[dtype]

    def normal(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 1.5).to(t)
    if fused:
        q, k, v = normal(tokens, (heads + 2 * kv) * head + 8).narrow(1, 8, (heads + 2 * kv) * head).split([heads * head, kv * head, kv * head], 1)
    else:
        q, k, v = normal(tokens, heads * head), normal(tokens, kv * head), normal(tokens, kv * head)
    qw, kw = ((1 + normal(head) / 4), (1 + normal(head) / 4)) if norm else (None, None)
    positions = torch.randint(0, far, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    positions[-1] = far
    rows = tokens + 11
    slots = torch.randperm(rows, generator=g, device="cuda")[:tokens].to(torch.int32)
    if tokens > 2:
        slots[tokens // 2] = -1  # padding in the middle
    both = normal(rows, 2 * kv * head)  # keys and values of a row beside one another
    kc, vc = both.split(kv * head, 1)
    k0, v0 = kc.clone(), vc.clone()
    cfg = ml2.Config(heads * head, 0, 1, heads, kv, 0, 0, 500000.0)
    out = normal(tokens, heads * head)
    q0 = out.clone()
    ml2.QKNormRoPE(ctx, cfg, rotary).Forward(out, kc, vc, q, k, v, qw, kw, positions, slots, eps=1e-6)
    live = slots >= 0
    at = slots[live].long()
    want, slack = rope_want(q, qw, heads, head, rotary, positions, 500000.0, 1e-6)
    near(out[live], want[live], slack[live], t)
    assert torch.equal(out[~live], q0[~live])
    want, slack = rope_want(k, kw, kv, head, rotary, positions, 500000.0, 1e-6)
    near(kc[at], want[live], slack[live], t)
    assert torch.equal(vc[at], v[live])
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(kc[rest], k0[rest]) and torch.equal(vc[rest], v0[rest])


def test_qk_norm_rope_in_place_and_special_values(ctx):
    """Queries over themselves; a head of zeros stays zero, one NaN or infinity spoils its own head alone."""
    cfg = ml2.Config(4 * 64, 0, 1, 4, 2, 0, 0)
    q, k, v = torch.randn(3, 256, device="cuda").half(), torch.randn(3, 128, device="cuda").half(), torch.randn(3, 128, device="cuda").half()
    q[0, :64] = 0
    q[1, 70] = float("nan")
    k[2, 3] = float("inf")
    v[0, 0] = float("nan")
    w = torch.ones(64, device="cuda").half()
    kc, vc = torch.zeros(4, 128, device="cuda").half(), torch.zeros(4, 128, device="cuda").half()
    pos, slots = ints([0, 5, 9]), ints([3, 1, 0])
    want, slack = rope_want(q, w, 4, 64, 64, pos, 10000.0, 1e-5)
    ml2.QKNormRoPE(ctx, cfg).Forward(q, kc, vc, q, k, v, w, w, pos, slots)
    assert bool((q[0, :64] == 0).all())
    fine = torch.ones(3, 256, dtype=torch.bool, device="cuda")
    fine[1, 64:128] = False
    assert bool(q[1, 64:128].isnan().all()) and bool(q[fine].isfinite().all())
    near(q[fine], want[fine], slack[fine], torch.float16)
    assert bool(kc[0, 64:].isfinite().all()) and not bool(kc[0, :64].isfinite().all()) and bool(vc[3, 0].isnan()) and bool(vc[3, 1:].isfinite().all())
    assert bool((kc[2] == 0).all())


def test_qk_norm_rope_slot_outside_the_cache_is_left_out_and_reported(ctx):
    cfg = ml2.Config(128, 0, 1, 1, 1, 0, 0)
    q = torch.randn(3, 128, device="cuda").half()
    out, kc, vc = torch.zeros_like(q), torch.zeros(5, 128, device="cuda").half(), torch.zeros(5, 128, device="cuda").half()
    ml2.QKNormRoPE(ctx, cfg).Forward(out, kc, vc, q, q, q, None, None, ints([1, 2, 3]), ints([4, 5, 2**31 - 1]))
    with pytest.raises(ml2.Ml2Error, match="slot of token"):
        ctx.status()
    assert torch.equal(vc[4], q[0]) and bool((vc[:4] == 0).all()) and bool((out[1:] == 0).all()) and bool((out[0] != 0).any())


# ---- shared-prefix attention -------------------------------------------------------------------------------------------
class Batch:
    """Random inputs; what no query may see holds NaN."""

    def __init__(self, seed, dtype, heads, kv, head, page, prefix, lengths, queries, sigma=2.0, extra_rows=0, extra_pages=2, poison=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = self.t = TYPES[dtype]
        self.heads, self.kv, self.head, self.page, self.prefix = heads, kv, head, page, prefix
        self.own, self.count = list(lengths), list(queries)
        n, total = len(lengths), sum(queries)

        def normal(rows, width, s=1.0):
            return (torch.randn(rows, width + 8, generator=g, device="cuda") * s).to(t)[:, 8:]  # strided rows
        self.q = normal(total + extra_rows, heads * head, sigma)
        self.pk, self.pv = normal(prefix, kv * head), normal(prefix, kv * head)
        held = [-(-x // page) for x in lengths]
        pages = sum(held) + extra_pages
        width = max(max(held), 1)
        ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).tolist()
        self.table = torch.full((n, width), -5, dtype=torch.int32, device="cuda")  # entries behind a request's pages are no pages
        both = normal(pages * page, 2 * kv * head)
        self.k, self.v = both.split(kv * head, 1)
        seen = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
        self.rows = []
        for r in range(n):
            mine = [ids.pop() for _ in range(held[r])]
            if mine:
                self.table[r, :held[r]] = ints(mine)
            j = torch.arange(lengths[r], device="cuda")
            at = (ints(mine).long()[j // page] * page + j % page) if mine else j
            self.rows.append(at)
            seen[at] = True
        if poison:
            both[~seen] = float("nan")
        self.lengths = ints(list(lengths))
        start = [0]
        for x in queries:
            start.append(start[-1] + x)
        self.start = ints(start)
        self.cfg = ml2.Config(heads * head, 0, 1, heads, kv, 0, 0)

    def want(self, scale=None):
        """(output, log sum, bound of the output, bound of the log sum) in 64 bits."""
        heads, kv, head = self.heads, self.kv, self.head
        scale = head ** -0.5 if scale is None else scale
        pk, pv = (x.double().reshape(-1, kv, head) for x in (self.pk, self.pv))
        out, lse, tol, tol_lse = [], [], [], []
        row = 0
        for r, (length, count) in enumerate(zip(self.own, self.count)):
            if not count:
                continue
            k = torch.cat([pk, self.k[self.rows[r]].double().reshape(-1, kv, head)]).permute(1, 0, 2)
            v = torch.cat([pv, self.v[self.rows[r]].double().reshape(-1, kv, head)]).permute(1, 0, 2)
            q = self.q[row:row + count].double().reshape(count, kv, heads // kv, head).permute(1, 2, 0, 3)
            seen = torch.cat([torch.ones(count, self.prefix, dtype=torch.bool, device="cuda"),
                              torch.arange(length, device="cuda") <= length - count + torch.arange(count, device="cuda")[:, None]], 1)
            s = (q @ k.mT[:, None]) * scale
            s = s.masked_fill(~seen, -math.inf)
            size = ((q.abs() @ k.abs().mT[:, None]) * abs(scale)).masked_fill(~seen, 0.0)
            m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full(s.shape[:-1] + (1,), -math.inf)
            e = torch.where(seen, torch.exp(s - m), 0.0)
            total = e.sum(-1, keepdim=True)
            p = torch.where(total > 0, e / total, 0.0)
            vv = v[:, None]
            o = p @ vv if bool(vv.isfinite().all()) else torch.stack([(p[..., i, :, None] * torch.where(seen[i][:, None], vv, 0.0)).sum(-2)
                                                                       for i in range(count)], -2)
            a = p @ torch.nan_to_num(vv).abs()
            # scores: `head` exact products added in fp32, each addition off by 2^-24 of the sum of sizes, then scaled: twice
            # that for scale and exponential; the weights carry it relatively, above and below the fraction bar
            es = 2.0 ** -24 * (head + 4) * (size.amax(-1, keepdim=True) if size.shape[-1] else size.new_zeros(size.shape[:-1] + (1,))) + 2.0 ** -20
            u = step(self.t)
            # weights below 2^-25 of the largest are lost in fp16: each at most 2^-25 of a weight of 1
            lost = 2.0 ** -25 * k.shape[1] * (torch.nan_to_num(vv).abs().amax() if vv.numel() else 0.0) if self.t is torch.float16 else 0.0
            bound = u * (o.abs() + a) * 1.01 + 4 * es * a + lost + (2.0 ** -25 if self.t is torch.float16 else 0.0)
            z = (m + torch.log(total))[..., 0]
            out.append(o.permute(2, 0, 1, 3).reshape(count, -1))
            tol.append(bound.permute(2, 0, 1, 3).reshape(count, -1))
            lse.append(z.permute(2, 0, 1).reshape(count, -1))
            tol_lse.append((2 * es[..., 0] + 2.0 ** -22 * z.abs()).permute(2, 0, 1).reshape(count, -1))
            row += count
        return [torch.cat(x) if x else torch.zeros(0, device="cuda") for x in (out, lse, tol, tol_lse)]

    def call(self, ctx, workspace=None, scale=None, lse=True, max_length=None):
        op = ml2.PrefixAttention(ctx, self.cfg, self.page)
        rows, most = self.q.shape[0], max(self.own) if max_length is None else max_length
        if workspace is None:
            workspace = torch.full((op.WorkspaceBytes(rows, len(self.own), self.prefix, most) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        out = torch.full((rows, self.heads * self.head + 16), 7.0, dtype=self.t, device="cuda")[:, :self.heads * self.head]
        z = torch.full((rows, self.heads), 7.0, device="cuda") if lse else None
        op.Forward(out, self.q, self.pk, self.pv, self.k, self.v, self.table, self.lengths, self.start, workspace, most, z, scale)
        return out, z

    def check(self, ctx, **kw):
        out, z = self.call(ctx, **kw)
        want, lse, tol, tol_lse = self.want(kw.get("scale"))
        total = sum(self.count)
        off = (out[:total].double() - want).abs()
        assert bool((off <= tol).all()), "output off by %.3g of its bound" % (off / tol).max().item()
        if z is not None:
            none = torch.isinf(lse)
            assert bool((z[:total][none] == -math.inf).all()) and bool((out[:total].reshape(total, self.heads, -1)[none] == 0).all())
            off = (z[:total].double() - lse).abs()[~none]
            assert bool((off <= tol_lse[~none]).all()), "log sum off by %.3g of its bound" % (off / tol_lse[~none]).max().item()
            assert bool((z[total:] == 7.0).all())
        assert bool((out[total:] == 7.0).all())  # rows behind the last request
        return out, z


def ragged(seed, n, most_length, most_queries):
    rng = random.Random(seed)
    lengths = [rng.randint(1, most_length) for _ in range(n)]
    return lengths, [rng.randint(1, min(x, most_queries)) for x in lengths]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (6, 2), (8, 1), (5, 5)])
@pytest.mark.parametrize("prefix", [0, 1, 63, 200])
def test_attention_single_tokens(ctx, dtype, head, heads, kv, prefix):
    lengths, _ = ragged(heads * 7 + prefix, 5, 90, 1)
    Batch(prefix + head, dtype, heads, kv, head, 16, prefix, lengths, [1] * 5).check(ctx)


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 511, 1025, 4032])
def test_attention_prefix_lengths(ctx, prefix):
    Batch(prefix, "fp16", 4, 2, 128, 16, prefix, [3, 20], [1, 1]).check(ctx)


@pytest.mark.parametrize("heads,kv,head,prefix,requests", [
    (40, 40, 128, 4032, 1), (40, 40, 128, 4032, 64), (5, 5, 128, 513, 3), (37, 37, 64, 640, 2), (16, 2, 128, 2048, 16), (16, 2, 128, 2049, 17),
    (24, 3, 64, 1111, 33), (8, 1, 64, 9000, 65), (64, 64, 64, 600, 130), (3, 1, 128, 700, 300), (12, 12, 128, 1500, 257),
    (5, 5, 128, 1025, 33), (37, 37, 64, 1100, 20), (64, 64, 64, 1088, 130), (3, 1, 128, 1300, 300), (40, 40, 128, 4096, 1), (8, 8, 64, 4200, 2),
    (1, 1, 128, 20000, 1), (2, 2, 64, 1024, 513)])
def test_attention_prefix_in_blocks(ctx, heads, kv, head, prefix, requests):
    """Runs of key tiles that begin and end anywhere in a head, blocks of up to 128, 129..256 and more rows; called twenty
    times over without waiting."""
    lengths, _ = ragged(prefix + requests, requests, 30, 1)
    b = Batch(prefix + heads, "fp16" if heads % 2 else "bf16", heads, kv, head, 16, prefix, lengths, [1] * requests, extra_rows=2)
    first, z = b.check(ctx)
    op = ml2.PrefixAttention(ctx, b.cfg, 16)
    ws = torch.full((op.WorkspaceBytes(b.q.shape[0], requests, prefix, max(lengths)),), 0xFF, dtype=torch.uint8, device="cuda")
    results = [b.call(ctx, workspace=ws) for _ in range(20)]
    for out, lse in results:
        assert torch.equal(out, first) and torch.equal(lse, z)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 32, 64, 128, 1024])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 129, 300, 1030])
def test_attention_pages_and_own_lengths(ctx, page, length):
    Batch(page + length, "bf16", 2, 2, 64, page, 40, [length, 1, max(1, length - 1)], [1, 1, 1]).check(ctx)


@pytest.mark.parametrize("requests", [1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 129, 200, 300])
def test_attention_batch_sizes(ctx, requests):
    lengths, _ = ragged(requests, requests, 40, 1)
    Batch(requests, "fp16", 2, 1, 128, 16, 300, lengths, [1] * requests).check(ctx)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1), (3, 1)])
@pytest.mark.parametrize("most", [2, 17, 70, 200])
def test_attention_several_queries(ctx, dtype, head, heads, kv, most):
    lengths, queries = ragged(most + heads, 4, 260, most)
    lengths[0], queries[0] = max(lengths[0], most), most
    lengths[1] = queries[1]  # a request whose tokens are all new
    Batch(most * head + kv, dtype, heads, kv, head, 32, 150, lengths, queries, extra_rows=5).check(ctx)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_requests_without_rows_tokens_or_pages(ctx, n):
    """Requests with nothing: no query rows, no own tokens, both; rows that see only the prefix; rows that see nothing."""
    for prefix in (0, 50):
        b = Batch(n + prefix, "fp16", 3, 3, 64, 16, prefix, [0, 5, 0, 33] * n, [0, 0, 1, 2] * n, extra_rows=3)
        b.check(ctx)
        # more query rows than own tokens: the first see only the prefix
        b = Batch(n, "bf16", 2, 1, 128, 16, prefix, [2, 0] * n, [5, 3] * n)
        b.check(ctx)
    Batch(3, "fp16", 1, 1, 64, 16, 0, [0] * n, [1] * n).check(ctx)
    b = Batch(3, "fp16", 1, 1, 64, 16, 10, [4] * n, [0] * n, extra_rows=2)
    out, z = b.call(ctx)
    assert bool((out == 7.0).all()) and bool((z == 7.0).all())


@pytest.mark.parametrize("sigma,scale", [(30.0, None), (0.0, None), (2.0, 0.0), (2.0, -0.3), (200.0, 1.0)])
def test_attention_peaked_and_flat_scores(ctx, sigma, scale):
    Batch(5, "fp16", 4, 2, 64, 16, 333, [70, 1, 20], [1, 1, 9], sigma=sigma).check(ctx, scale=scale)


@pytest.mark.parametrize("sigma,scale", [(30.0, None), (0.0, None), (2.0, 0.0), (2.0, -0.3), (200.0, 1.0)])
@pytest.mark.parametrize("requests", [17, 150])
def test_attention_peaked_and_flat_scores_in_blocks(ctx, sigma, scale, requests):
    """The reference point moves with a score that is much larger: first tiles of small scores, then larger and larger ones."""
    b = Batch(7, "fp16", 4, 2, 128, 16, 1500, [20] * requests, [1] * requests, sigma=sigma)
    b.check(ctx, scale=scale)
    b.pk *= (torch.arange(1500, device="cuda") / 300)[:, None].half()
    b.check(ctx, scale=scale)


@pytest.mark.parametrize("requests", [17, 150])
def test_attention_infinite_scores_in_blocks(ctx, requests):
    b = Batch(2, "bf16", 2, 2, 64, 16, 1100, [20] * requests, [1] * requests)
    b.q[:, 0], b.q[:, 64] = 1.0, 1.0
    clean, _ = b.call(ctx)
    b.pk[3, 0] = float("-inf")  # one key of head 0 has no weight
    out, z = b.call(ctx)
    want, lse, tol, tol_lse = b.want()
    assert bool(((out.double() - want).abs() <= torch.nan_to_num(tol, posinf=1.0)).all()) and bool(z.isfinite().all())
    assert torch.equal(out[:, 64:], clean[:, 64:])
    b.pk[:, 0] = float("-inf")  # none of the prefix has: the own tokens alone
    out, z = b.call(ctx)
    own = Batch(2, "bf16", 2, 2, 64, 16, 1100, [20] * requests, [1] * requests)
    own.q[:, 0], own.q[:, 64] = 1.0, 1.0
    own.pk, own.pv, own.prefix = own.pk[:0], own.pv[:0], 0
    want, lse, tol, tol_lse = own.want()
    assert bool(((out.double() - want).abs() <= tol)[:, :64].all()) and bool(((z.double() - lse).abs() <= tol_lse)[:, 0].all())
    b.pk[5, 64] = float("inf")  # and NaN for every row of head 1
    out, z = b.call(ctx)
    assert bool(out[:, 64:].isnan().all()) and bool(out[:, :64].isfinite().all())


def test_attention_without_log_sums_equals_with(ctx):
    b = Batch(9, "fp16", 4, 4, 128, 16, 500, [70, 3], [1, 2])
    assert torch.equal(b.call(ctx, lse=False)[0], b.call(ctx)[0])


@pytest.mark.parametrize("heads,kv,most", [(2, 2, 1), (2, 1, 20), (8, 1, 100)])
def test_attention_keeps_out_what_is_masked(ctx, heads, kv, most):
    """Tokens after a query's own place hold infinities and NaN, in keys and values: earlier queries do not see them."""
    lengths, queries = [150, 40], [most, min(most, 40)]
    b = Batch(most, "fp16", heads, kv, 128, 16, 70, lengths, queries)
    clean_out, clean_lse = b.check(ctx)
    for r in range(2):
        if queries[r] > 1:
            last = b.rows[r][lengths[r] - 1]
            b.k[last] = float("nan")
            b.v[last] = float("inf")
            b.v[last, :5] = float("nan")
    out, lse = b.call(ctx)
    first = torch.ones(sum(queries), dtype=torch.bool, device="cuda")
    if most > 1:
        first[[queries[0] - 1, sum(queries) - 1]] = False
        assert bool(out[~first].isnan().all())
    assert torch.equal(out[first], clean_out[first]) and torch.equal(lse[first], clean_lse[first])


def test_attention_infinite_scores_and_values(ctx):
    """A key that scores -inf has no weight; one that scores +inf or NaN gives NaN to its own rows; rows whose every score is
    -inf are empty."""
    b = Batch(2, "bf16", 2, 2, 64, 16, 40, [20, 20], [1, 1])
    b.q[:, 0], b.q[:, 64] = 1.0, 1.0
    b.pk[3, 0] = float("-inf")        # head 0 of every row
    b.k[b.rows[0][4], 64] = float("-inf")  # head 1 of row 0
    out, z = b.call(ctx)
    want, lse, tol, tol_lse = b.want()
    assert bool(((out.double() - want).abs() <= torch.nan_to_num(tol, posinf=1.0)).all())
    assert bool(z.isfinite().all())
    b.k[b.rows[1][4], 64] = float("inf")  # head 1 of row 1
    out2, z2 = b.call(ctx)
    assert bool(out2[1, 64:].isnan().all()) and torch.equal(out2[0], out[0]) and torch.equal(out2[1, :64], out[1, :64])
    b = Batch(2, "bf16", 2, 2, 64, 16, 40, [20, 20], [1, 1])
    b.q[:, 0] = 1.0
    b.pk[:, 0] = float("-inf")
    b.k[torch.cat(b.rows), 0] = float("-inf")
    out, z = b.call(ctx)
    assert bool((out[:, :64] == 0).all()) and bool((z[:, 0] == -math.inf).all()) and bool(z[:, 1].isfinite().all())
    b = Batch(3, "fp16", 2, 2, 64, 16, 40, [20, 20], [1, 1])
    b.v[b.rows[0][4], 3] = float("inf")
    out, z = b.call(ctx)
    assert out[0, 3].item() == math.inf and bool(out[0, 4:].isfinite().all()) and bool(out[1].isfinite().all())


def test_attention_bad_tables_are_left_out_and_reported(ctx):
    b = Batch(4, "fp16", 2, 2, 64, 16, 30, [40, 40], [1, 1])
    good, _ = b.call(ctx)
    b.table[1, 1] = 10**6
    out, _ = b.call(ctx)
    with pytest.raises(ml2.Ml2Error, match="page of request 1"):
        ctx.status()
    b.rows[1] = torch.cat([b.rows[1][:16], b.rows[1][32:]])
    b.own[1] = 24
    want, _, tol, _ = b.want()
    assert torch.equal(out[0], good[0]) and bool(((out.double() - want).abs() <= tol).all())
    b = Batch(4, "fp16", 2, 2, 64, 16, 30, [40, 40], [1, 1])
    b.call(ctx, max_length=39)
    with pytest.raises(ml2.Ml2Error, match="length or the query rows of request"):
        ctx.status()


@pytest.mark.parametrize("start", [[0, 3, 1, 2], [1, 1, 2, 3], [5, 6, 7, 8], [0, 1, 2, 2**31 - 1], [-5, 0, 1, 2], [0, -1, -2, -3]])
def test_attention_query_rows_out_of_order_stay_in_bounds(ctx, start):
    b = Batch(4, "fp16", 2, 2, 64, 16, 30, [40, 40, 3], [1, 1, 1])
    b.start = ints(start)
    out, z = b.call(ctx)
    with pytest.raises(ml2.Ml2Error, match="length or the query rows of request"):
        ctx.status()


@pytest.mark.parametrize("prefix", [30, 1200])
def test_attention_lengths_above_a_bound_of_zero_are_reported(ctx, prefix):
    """A call for no own tokens at all: a request that has some gets the prefix alone, and is reported."""
    b = Batch(4, "fp16", 34, 2, 64, 16, prefix, [0, 0, 0], [1, 1, 1])
    want, z = b.check(ctx)
    b.lengths = ints([0, 7, 0])
    out, z2 = b.call(ctx, max_length=0)
    with pytest.raises(ml2.Ml2Error, match="length or the query rows of request 1"):
        ctx.status()
    assert torch.equal(out, want) and torch.equal(z, z2)


def test_attention_same_result_twice_and_on_another_stream(ctx):
    b = Batch(6, "bf16", 8, 2, 128, 16, 1000, *ragged(6, 20, 100, 1))
    first, z = b.check(ctx)
    second, z2 = b.call(ctx)
    assert torch.equal(first, second) and torch.equal(z, z2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            third, z3 = b.call(ctx)
    finally:
        ctx.set_stream(0)
    s.synchronize()
    assert torch.equal(first, third) and torch.equal(z, z3)


def test_attention_cache_offsets_past_32_bits(ctx):
    """A cache of more than 2^31 elements, its pages at both ends."""
    page, kv, head = 1024, 8, 128
    pages = (2**31 // (kv * head * page)) + 3
    k = torch.zeros(pages * page, kv * head, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    b = Batch(8, "fp16", 8, 8, 128, 1024, 10, [1500, 9], [1, 1], poison=False)
    big = b.table.clone()
    for r, places in enumerate([[pages - 1, 0], [pages - 2]]):
        for i, page_id in enumerate(places):
            src = int(b.table[r, i])
            k[page_id * page:(page_id + 1) * page] = b.k[src * page:(src + 1) * page]
            v[page_id * page:(page_id + 1) * page] = b.v[src * page:(src + 1) * page]
            big[r, i] = page_id
    b2 = b.call(ctx)[0]
    b.k, b.v, b.table = k, v, big
    assert torch.equal(b.call(ctx)[0], b2)


def test_attention_workspace_too_small_is_refused(ctx):
    b = Batch(6, "bf16", 8, 2, 128, 16, 5000, [40] * 30, [1] * 30)
    need = ml2.PrefixAttention(ctx, b.cfg, 16).WorkspaceBytes(30, 30, 5000, 40)
    if need:
        with pytest.raises(ml2.Ml2Error, match="workspace"):
            b.call(ctx, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))


def test_modules_refuse_wrong_tensors(ctx):
    b = Batch(6, "bf16", 4, 2, 64, 16, 50, [40] * 3, [1] * 3)
    op = ml2.PrefixAttention(ctx, b.cfg, 16)
    ws, out = torch.empty(1 << 24, dtype=torch.uint8, device="cuda"), torch.empty(3, 256, dtype=b.t, device="cuda")
    good = dict(output=out, query=b.q, prefixKey=b.pk, prefixValue=b.pv, keyCache=b.k, valueCache=b.v, table=b.table, lengths=b.lengths,
                queryStart=b.start, workspace=ws, maxLength=40)
    op.Forward(**good)
    for change in (dict(query=b.q.float()), dict(query=b.q.half()), dict(output=out[:2]), dict(output=out.cpu()), dict(prefixValue=b.pv[:5]),
                   dict(valueCache=b.v.contiguous()), dict(table=b.table.long()), dict(table=b.table[:2]), dict(queryStart=b.start[:3]),
                   dict(lse=torch.empty(3, 4, device="cuda").half()), dict(lse=torch.empty(3, 3, device="cuda")), dict(workspace=ws.cpu()),
                   dict(keyCache=b.k.t()), dict(query=b.q[:, :128])):
        with pytest.raises(ValueError):
            op.Forward(**dict(good, **change))


# ---- together ----------------------------------------------------------------------------------------------------------
def decode_steps(ctx, graph, prefix):
    """Four samples behind one prompt, five steps: prompts of different length first, then one token each, one request that
    ends and one that begins; returns what the last step gave and the plain form of it."""
    heads, kv, head, page, width = 6, 2, 64, 16, 8
    cfg = ml2.Config(heads * head, 0, 1, heads, kv, 0, 0)
    g = torch.Generator(device="cuda").manual_seed(11)
    pk, pv = (torch.randn(prefix, kv * head, generator=g, device="cuda").half() for _ in range(2))
    weight = (1 + torch.randn(head, generator=g, device="cuda") / 8).half()
    pages, n, rows = 20, 4, 64
    kc, vc = (torch.full((pages * page, kv * head), float("nan"), device="cuda").half() for _ in range(2))
    table, free = torch.full((n, width), -1, dtype=torch.int32, device="cuda"), ints(list(range(pages)))
    lengths, count, new = ints([0] * n), ints([pages]), ints([0] * n)
    start, slots, positions, refused = ints([0] * (n + 1)), ints([0] * rows), ints([0] * rows), ints([0] * n)
    qkv = torch.zeros(rows, (heads + 2 * kv) * head, device="cuda").half()
    q, k, v = qkv.split([heads * head, kv * head, kv * head], 1)
    turned, out = torch.zeros(rows, heads * head, device="cuda").half(), torch.zeros(rows, heads * head, device="cuda").half()
    tables, norm, attend = ml2.BlockTables(ctx, page), ml2.QKNormRoPE(ctx, cfg), ml2.PrefixAttention(ctx, cfg, page)
    ws = torch.empty(attend.WorkspaceBytes(rows, n, prefix, width * page), dtype=torch.uint8, device="cuda")

    def step_():
        tables.Forward(lengths, new, table, free, count, lengths, count, start, slots, positions, refused, prefix)
        norm.Forward(turned, kc, vc, q, k, v, weight, weight, positions, slots)
        attend.Forward(out, turned, pk, pv, kc, vc, table, lengths, start, ws, width * page)

    replay = None
    if graph:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        ctx.set_stream(s.cuda_stream)
        with torch.cuda.stream(s):
            step_()  # nothing grows: every kernel is loaded
        s.synchronize()
        replay = torch.cuda.CUDAGraph()
        with torch.cuda.graph(replay, stream=s):
            step_()
        ctx.set_stream(0)
    history = [[] for _ in range(n)]
    old = [0] * n
    for want in ([5, 40, 1, 0], [6, 41, 2, 0], [7, 42, 0, 17], [8, 43, 0, 18], [9, 44, 3, 19]):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda").half())
        new.copy_(ints(want))
        if replay is not None:
            replay.replay()
        else:
            step_()
        row = 0
        for r in range(n):
            if want[r] < old[r]:
                history[r] = history[r][:want[r]]
            for j in range(old[r], want[r]):
                history[r].append((row, qkv[row].clone(), prefix + j))
                row += 1
        old = want
    torch.cuda.synchronize()
    assert refused.tolist() == [0] * n and lengths.tolist() == old and start.tolist()[-1] == row
    # plain: every request's keys and values from its history
    row, worst = 0, 0.0
    for r in range(n):
        x = torch.stack([h[1] for h in history[r]])
        pos = ints([h[2] for h in history[r]])
        fresh = {0: 1, 1: 1, 2: 3, 3: 1}[r]
        kk = rope_want(x[:, heads * head:(heads + kv) * head], weight, kv, head, head, pos, 10000.0, 1e-5)[0].half().double().reshape(-1, kv, head)
        vv = x[:, (heads + kv) * head:].double().reshape(-1, kv, head)
        qq = rope_want(x[-fresh:, :heads * head], weight, heads, head, head, pos[-fresh:], 10000.0, 1e-5)[0].half().double()
        kk = torch.cat([pk.double().reshape(-1, kv, head), kk]).permute(1, 0, 2)
        vv = torch.cat([pv.double().reshape(-1, kv, head), vv]).permute(1, 0, 2)
        qq = qq.reshape(fresh, kv, heads // kv, head).permute(1, 2, 0, 3)
        sc = (qq @ kk.mT[:, None]) * head ** -0.5
        last = sc.shape[-1] - fresh + torch.arange(fresh, device="cuda")[:, None]
        sc = sc.masked_fill(torch.arange(sc.shape[-1], device="cuda") > last, -math.inf)
        o = (torch.softmax(sc, -1) @ vv[:, None]).permute(2, 0, 1, 3).reshape(fresh, -1)
        # values of size 4 and below: the rounded weights and output 2^-11 each, a rotated key or query that fell on the other
        # side of a rounding moves a score by 2^-11 of one product of size 2 or so: 2^-11 * (4 + 4 + 4)
        worst = max(worst, (out[row:row + fresh].double() - o).abs().max().item())
        row += fresh
    assert worst <= 12 * 2.0 ** -11, worst
    return out[:row].clone()


@pytest.mark.parametrize("prefix", [0, 77, 1500])  # none, by runs, by blocks
def test_decode_steps_together_and_in_a_graph(ctx, prefix):
    eager = decode_steps(ctx, False, prefix)
    assert torch.equal(eager, decode_steps(ctx, True, prefix))
    ctx.set_pdl(True)  # programmatic launch edges between the calls too
    try:
        assert torch.equal(eager, decode_steps(ctx, False, prefix))
        assert torch.equal(eager, decode_steps(ctx, True, prefix))
    finally:
        ctx.set_pdl(False)


def test_samples_behind_a_prompt_in_a_transformers_own_cache(ctx):
    """The prompt goes through ``Transformer.Forward`` token by token; layer 0's rows of its key and value caches are then
    the shared prefix, in place."""
    cfg = ml2.Config(256, 768, 2, 2, 2, 512, 64)
    tr = ml2.Transformer(cfg, ml2.synthetic_weights(ctx, cfg, seed=3, sigma=1.0), ctx)
    prompt = [7, 99, 300, 5, 41, 17, 250, 8, 130]
    tr.set_tokens(prompt)
    for pos in range(len(prompt)):
        tr.Forward(pos, pos + 1, False)
    tr.synchronize()
    rs = tr.runstate_ptrs()

    class Rows:  # the library's own buffer as a tensor
        def __init__(self, ptr):
            self.__cuda_array_interface__ = {"shape": (cfg.seqLength, cfg.dim), "typestr": "<f2", "data": (ptr, False), "version": 2}
    k, v = (torch.as_tensor(Rows(p), device="cuda")[:len(prompt)] for p in (rs.key_cache, rs.value_cache))
    assert bool((k != 0).any()) and bool((v != 0).any())
    b = Batch(12, "fp16", 2, 2, 128, 16, len(prompt), [4, 30, 1], [1, 1, 1])
    b.pk, b.pv = k, v
    b.check(ctx)
    tr.close()


@pytest.mark.parametrize("prefix", [300, 2000])
def test_attention_over_its_own_queries(ctx, prefix):
    b = Batch(prefix, "bf16", 8, 2, 128, 16, prefix, [70, 3, 40], [1, 2, 9], extra_rows=1)
    want, z = b.call(ctx)
    q = b.q.clone()
    op = ml2.PrefixAttention(ctx, b.cfg, 16)
    ws = torch.empty(op.WorkspaceBytes(13, 3, prefix, 70), dtype=torch.uint8, device="cuda")
    op.Forward(q, q, b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, 70)
    assert torch.equal(q[:12], want[:12]) and torch.equal(q[12:], b.q[12:])


@pytest.mark.parametrize("head", [64, 128])
def test_calls_of_two_contexts_at_the_same_time(head):
    """Two contexts, each with its stream and workspace, the same kernels from both in flight together."""
    cases = []
    for i in range(2):
        c, s = ml2.CudaContext(0), torch.cuda.Stream()
        b = Batch(20 + i, "fp16", 8, 2, head, 16, 2000 + 100 * i, *ragged(i, 40, 120, 1))
        want, z = b.check(c)
        op = ml2.PrefixAttention(c, b.cfg, 16)
        ws = torch.empty(op.WorkspaceBytes(40, 40, b.prefix, 120), dtype=torch.uint8, device="cuda")
        outs = [(torch.zeros(40, 8 * head, dtype=b.t, device="cuda"), torch.zeros(40, 8, device="cuda")) for _ in range(10)]
        torch.cuda.synchronize()
        c.set_stream(s.cuda_stream)
        cases.append((c, s, b, op, ws, outs, want, z))
    for k in range(10):
        for c, s, b, op, ws, outs, want, z in cases:
            op.Forward(outs[k][0], b.q, b.pk, b.pv, b.k, b.v, b.table, b.lengths, b.start, ws, 120, outs[k][1])
    for c, s, b, op, ws, outs, want, z in cases:
        s.synchronize()
        for out, lse in outs:
            assert torch.equal(out, want) and torch.equal(lse, z)
        assert c.status() == (0, 0)
        c.close()

