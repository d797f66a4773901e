"""Cases and plain forms of the batched-decoding operators: block tables, query/key norm with rotation and cache write,
and attention of a batch that shares a prefix.

``own`` chooses what ``run`` does: False computes each operator from elementary torch operations, True makes the calls of
``managedllama2_b200`` (``BlockTables``, ``QKNormRoPE``, ``PrefixAttention``). Both work on what ``prepare`` gives.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ---------------------------------------------------------------------------------------------------------
def _tables(name, requests, tokens, grow, page, max_length, leave):
    """requests: rows of the table; tokens: new tokens of a request (1, or 1..tokens); grow: share of requests that grow by one
    token only; leave: share of requests that end and give their pages back."""
    return {"name": name, "op": "tables", "requests": requests, "tokens": tokens, "grow": grow, "page": page, "max_length": max_length,
            "leave": leave}


def _rope(name, tokens, heads, kv_heads, head_size, rotary, dtype, fused, norm, position, padding):
    """fused: query, key and value are columns of one tensor; position: positions are drawn below it; padding: rows behind the
    last token, which carry no slot."""
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_size": head_size,
            "rotary": rotary, "dtype": dtype, "fused": fused, "norm": norm, "position": position, "padding": padding}


def _attn(name, requests, queries, prefix, length, heads, kv_heads, head_size, page, dtype):
    """queries: new tokens of a request (1, or 1..queries); prefix: shared tokens; length: own tokens of a request, 1..length."""
    return {"name": name, "op": "attn", "requests": requests, "queries": queries, "prefix": prefix, "length": length,
            "heads": heads, "kv_heads": kv_heads, "head_size": head_size, "page": page, "dtype": dtype}


def listed():
    return [
        # one decode step of 64 samples: every request grows by one token, some into a new page
        _tables("tables_step_64", 64, 1, 1.0, 16, 4096, 0.0),
        # a full scheduler step: 512 requests, some decoding, some ending, the others bringing prompts of up to 1024 tokens
        _tables("tables_prompts_512", 512, 1024, 0.25, 32, 4096, 0.1),
        # the latency of one token of the 7B shape
        _rope("rope_1_7b", 1, 32, 32, 128, 128, "fp16", False, True, 4096, 0),
        # one decode step of 64 samples, 13B shape (that family has no head norms: rotation and cache write alone)
        _rope("rope_64_13b", 64, 40, 40, 128, 128, "fp16", False, False, 4096, 0),
        # a prompt of 4032 tokens, grouped heads, fused QKV product, far positions
        _rope("rope_prompt_gqa", 4032, 64, 8, 128, 128, "bf16", True, True, 131072, 0),
        # ragged: odd head counts, heads of 96 rotated in part, rows of padding behind the batch
        _rope("rope_ragged_96", 777, 15, 5, 96, 64, "bf16", True, True, 32768, 23),
        # a few samples of a short prompt on one of eight shards of the 13B shape: latency
        _attn("attn_4_short", 4, 1, 200, 40, 5, 5, 128, 16, "fp16"),
        # one sample behind a long prompt, 13B shape
        _attn("attn_1_13b", 1, 1, 4032, 64, 40, 40, 128, 16, "fp16"),
        # 64 samples of one 4032-token prompt, 13B shape
        _attn("attn_64_13b", 64, 1, 4032, 256, 40, 40, 128, 16, "fp16"),
        # 128 requests behind a long shared document, grouped heads: the largest
        _attn("attn_128_gqa_long", 128, 1, 16384, 512, 64, 8, 128, 32, "bf16"),
        # eight conversations bring their first messages (1..256 tokens each) behind a common system prompt, 7B shape
        _attn("attn_messages_7b", 8, 256, 2048, 512, 32, 32, 128, 64, "fp16"),
        # no shared part, small heads, grouped by four, ragged lengths
        _attn("attn_own_only_64", 48, 1, 0, 2048, 16, 4, 64, 16, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.25 / hi)))))


def draw(rng):
    op = rng.choice(["tables", "rope", "attn", "attn"])
    if op == "tables":
        c = _tables("", _log(rng, 1, 2048), rng.choice([1, _log(rng, 2, 1024)]), rng.uniform(0, 1), rng.choice([16, 32, 64, 128]),
                    _log(rng, 256, 8192), rng.uniform(0, 0.3))
        while c["requests"] * c["tokens"] > 512 * 1024:
            c["requests"] = (c["requests"] + 1) // 2
    elif op == "rope":
        kv, head = rng.choice([1, 2, 4, 5, 8, 20, 32, 40]), rng.choice([64, 80, 96, 128, 256])
        heads = kv * rng.choice([1, 2, 3, 4, 8] if kv <= 8 else [1])
        rotary = head if rng.random() < 0.7 else 16 * rng.randint(1, head // 16)
        c = _rope("", _log(rng, 1, 4096), heads, kv, head, rotary, rng.choice(["fp16", "bf16"]), rng.random() < 0.5, rng.random() < 0.7,
                  _log(rng, 16, 1 << 20), rng.choice([0, 0, rng.randint(1, 64)]))
        while c["tokens"] * (heads + 2 * kv) * head > 4032 * 80 * 128:
            c["tokens"] = (c["tokens"] + 1) // 2
    else:
        kv = rng.choice([1, 2, 4, 5, 8, 20, 32, 40])
        heads = kv * rng.choice([1, 2, 3, 4, 8] if kv <= 8 else [1])
        c = _attn("", _log(rng, 1, 256), rng.choice([1, 1, _log(rng, 2, 256)]), rng.choice([0, _log(rng, 1, 16384), _log(rng, 256, 16384)]),
                  _log(rng, 1, 2048), heads, kv, rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["fp16", "bf16"]))
        top = work(listed()[9])["flops"] / 2
        while True:  # no dearer than the largest listed one, and its padded plain form within memory
            n, q, own_len = c["requests"], c["queries"], c["length"]
            score = n * heads * q * (c["prefix"] + own_len)
            rows = n * own_len * kv * c["head_size"]
            if n == 1 or (score * 4 * c["head_size"] <= top and rows <= 1.2e8):
                break
            c["requests"] = (n + 1) // 2
        while c["queries"] > 1 and c["queries"] * heads * (c["prefix"] + c["length"]) * 4 * c["head_size"] > top:
            c["queries"] //= 2
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _pages(length, page):
    return -(-length // page)


def _lengths(case):
    """(own length, new tokens) of every request: the same for every seed of a case, so that work() can count them."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "tables":
        old, new = [], []
        for _ in range(case["requests"]):
            was = r.randint(0, case["max_length"])
            if r.random() < case["leave"]:
                new.append(0)
            elif case["tokens"] == 1 or r.random() < case["grow"]:
                was = min(was, case["max_length"] - 1)
                new.append(was + 1)
            else:
                was = 0
                new.append(min(r.randint(1, case["tokens"]), case["max_length"]))
            old.append(was)
        return old, new
    own_len = [r.randint(1, case["length"]) for _ in range(case["requests"])]
    return own_len, [1 if case["queries"] == 1 else min(n, r.randint(1, case["queries"])) for n in own_len]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def normal(*shape, sigma=1.0):
        t = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
        return (t * sigma if sigma != 1.0 else t).to(DTYPES[case["dtype"]])

    st = {"case": dict(case)}
    if case["op"] == "tables":
        old, new = _lengths(case)
        page, n = case["page"], case["requests"]
        width = _pages(case["max_length"], page)
        held = [_pages(x, page) for x in old]
        wanted = sum(max(0, _pages(b, page) - _pages(a, page)) for a, b in zip(old, new))
        total = sum(held) + wanted + 64
        ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        mask = torch.arange(width, device="cuda")[None, :] < ints(held)[:, None]
        table[mask] = ids[:sum(held)]
        free = torch.full((total,), -1, dtype=torch.int32, device="cuda")
        free[:total - sum(held)] = ids[sum(held):]
        grown = sum(max(0, b - a) for a, b in zip(old, new))
        rows = 8 * _pages(grown + 1, 8)  # the step's token buffer, a little longer than its tokens
        st.update(old=ints(old), new=ints(new), table=table, free=free, free_count=ints([total - sum(held)]), offset=int(torch.randint(0, 4096, (1,), generator=torch.Generator().manual_seed(seed))),
                  lengths=torch.zeros(n, dtype=torch.int32, device="cuda"), free_count_out=ints([0]),
                  start=torch.zeros(n + 1, dtype=torch.int32, device="cuda"), slots=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                  positions=torch.zeros(rows, dtype=torch.int32, device="cuda"), refused=torch.zeros(n, dtype=torch.int32, device="cuda"))
        return st
    heads, kv, head = case["heads"], case["kv_heads"], case["head_size"]
    if case["op"] == "rope":
        rows = case["tokens"] + case["padding"]
        if case["fused"]:
            qkv = normal(rows, (heads + 2 * kv) * head, sigma=1.5)
            q, k, v = qkv.split([heads * head, kv * head, kv * head], dim=1)
        else:
            q, k, v = normal(rows, heads * head, sigma=1.5), normal(rows, kv * head, sigma=1.5), normal(rows, kv * head)
        n_slots = 16 * _pages(case["tokens"] + case["tokens"] // 4 + 1, 16)
        slots = torch.randperm(n_slots, generator=gen, device="cuda")[:rows].to(torch.int32)
        if slots.numel() < rows:
            slots = torch.cat([slots, slots.new_full((rows - slots.numel(),), -1)])
        slots[case["tokens"]:] = -1
        weight = (lambda: 1.0 + normal(head, sigma=0.2)) if case["norm"] else (lambda: None)
        st.update(q=q, k=k, v=v, slots=slots, positions=torch.randint(0, case["position"], (rows,), generator=gen, device="cuda", dtype=torch.int32),
                  qw=weight(), kw=weight(), q_out=torch.zeros(rows, heads * head, dtype=q.dtype, device="cuda"),
                  k_cache=torch.zeros(n_slots, kv * head, dtype=q.dtype, device="cuda"),
                  v_cache=torch.zeros(n_slots, kv * head, dtype=q.dtype, device="cuda"))
        return st
    own_len, new = _lengths(case)
    page, n = case["page"], case["requests"]
    width = _pages(max(own_len), page)
    held = [_pages(x, page) for x in own_len]
    n_pages = sum(held) + 3
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < ints(held)[:, None]] = ids[:sum(held)]
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    st.update(q=normal(start[-1], heads * head, sigma=2.0), k_prefix=normal(case["prefix"], kv * head), v_prefix=normal(case["prefix"], kv * head),
              k_cache=normal(n_pages * page, kv * head), v_cache=normal(n_pages * page, kv * head), table=table, lengths=ints(own_len),
              start=ints(start), most_queries=max(new), most_length=max(own_len),
              out=torch.zeros(start[-1], heads * head, dtype=DTYPES[case["dtype"]], device="cuda"),
              lse=torch.zeros(start[-1], heads, dtype=torch.float32, device="cuda"))
    return st


# ---- the operators in plain form ---------------------------------------------------------------------------------------
def _plain_tables(st):
    page, free, table = st["case"]["page"], st["free"], st["table"]
    old, new, rows = st["old"].long(), st["new"].long(), st["slots"].numel()
    n, width, capacity = table.shape[0], table.shape[1], free.numel()
    had, want = (old + page - 1) // page, (new + page - 1) // page
    bad = (new < 0) | (want > width)
    # pages of requests that shrink go on the free stack, in order of request and page
    col = torch.arange(width, device=table.device)
    back = (col >= want[:, None]) & (col < had[:, None]) & ~bad[:, None]
    count = st["free_count"].long()
    at = torch.cumsum(back.reshape(-1).long(), 0) - 1 + count
    at = torch.where(back.reshape(-1), at, capacity)
    grown = torch.cat([free, free.new_zeros(1)])
    grown[at] = table.reshape(-1)
    free.copy_(grown[:capacity])
    have = count + back.sum()
    # who is served: inclusive sums of tokens, then of pages
    tokens = torch.where(bad, 0, (new - old).clamp(min=0))
    over = (tokens > 0) & (torch.cumsum(tokens, 0) > rows)
    need = torch.where(bad | over, 0, (want - had).clamp(min=0))
    end = torch.cumsum(need, 0)
    short = (need > 0) & (end > have)
    tokens, need = torch.where(over | short, 0, tokens), torch.where(short, 0, need)
    refused = torch.where(bad, 1, torch.where(over, 3, torch.where(short, 2, 0))).int()
    # new pages come off the top of the stack
    first = torch.cumsum(need, 0) - need
    k = col - had[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    top = (have - 1 - first[:, None] - k).clamp(0, capacity - 1)
    table.copy_(torch.where(fresh, free[top], table))
    start = torch.cat([tokens.new_zeros(1), torch.cumsum(tokens, 0)])
    row = torch.arange(rows, device=table.device)
    who = torch.searchsorted(start[1:], row, right=True).clamp(max=n - 1)
    place = old[who] + row - start[who]
    live = row < start[n]
    entry = table[who, (place // page).clamp(0, width - 1)]
    st["slots"].copy_(torch.where(live, entry * page + place % page, -1))
    st["positions"].copy_(torch.where(live, st["offset"] + place, 0))
    st["lengths"].copy_(torch.where(refused != 0, old, new))
    st["start"].copy_(start)
    st["free_count_out"].copy_(have - need.sum())
    st["refused"].copy_(refused)
    return _of_tables(st)


def _of_tables(st):
    return {"lengths": st["lengths"], "table": st["table"], "free": st["free"], "free_count": st["free_count_out"], "start": st["start"],
            "slots": st["slots"], "positions": st["positions"], "refused": st["refused"]}


def _plain_rope(st):
    c = st["case"]
    head, rotary, eps, theta = c["head_size"], c["rotary"], 1e-5, 10000.0
    half, rows = rotary // 2, c["tokens"] + c["padding"]
    live = st["slots"] >= 0
    power = torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 / rotary)
    angle = st["positions"].double()[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device="cuda"), power)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, weight):
        y = x.float().reshape(rows, -1, head)
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight.float()
        a, b = y[..., :half], y[..., half:rotary]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., rotary:]], -1).reshape(rows, -1).to(x.dtype)

    st["q_out"].copy_(torch.where(live[:, None], turn(st["q"], st["qw"]), st["q_out"]))
    at = st["slots"][:c["tokens"]].long()
    st["k_cache"][at] = turn(st["k"], st["kw"])[:c["tokens"]]
    st["v_cache"][at] = st["v"][:c["tokens"]]
    return {"q": st["q_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain_attn(st):
    c = st["case"]
    heads, kv, head, page = c["heads"], c["kv_heads"], c["head_size"], c["page"]
    group, scale, most, longest = heads // kv, c["head_size"] ** -0.5, st["most_queries"], st["most_length"]
    rows, n = st["q"].shape[0], c["requests"]
    q = st["q"].float().reshape(rows, kv, group, head) * scale
    # the shared prefix: one product for all rows
    kp = st["k_prefix"].float().reshape(-1, kv, head)
    vp = st["v_prefix"].float().reshape(-1, kv, head)
    sp = torch.bmm(q.permute(1, 0, 2, 3).reshape(kv, rows * group, head), kp.permute(1, 2, 0))
    # each request's own pages, padded to the longest
    place = torch.arange(longest, device="cuda")
    slot = st["table"].long()[:, place // page].clamp(min=0) * page + place % page
    ko = st["k_cache"][slot].float().reshape(n, longest, kv, head).permute(0, 2, 3, 1)
    vo = st["v_cache"][slot].float().reshape(n, longest, kv, head).permute(0, 2, 1, 3)
    start, length = st["start"].long(), st["lengths"].long()
    count = start[1:] - start[:-1]
    j = torch.arange(most, device="cuda")
    at = (start[:-1, None] + j).clamp(max=rows - 1)
    qo = q[at].permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, head)
    so = torch.matmul(qo, ko).reshape(n, kv, most, group, longest)
    seen = place <= (length - count)[:, None, None] + j[:, None]
    seen = (seen & (place < length[:, None, None]))[:, None, :, None, :]
    so = torch.where(seen, so, -math.inf).reshape(n, kv, most * group, longest)
    # joined softmax, with the rows of the padded part brought back in order
    real = (j < count[:, None]).reshape(-1)

    def back(t):
        return t.reshape(n, kv, most, group, -1).permute(0, 2, 1, 3, 4).reshape(n * most, kv, group, -1)[real]

    def ahead(t):
        return t.reshape(rows, kv, group, -1)[at].permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, -1)

    top = back(so.amax(-1, keepdim=True))
    if c["prefix"]:
        top = torch.maximum(top, sp.amax(-1).reshape(kv, rows, group, 1).permute(1, 0, 2, 3))
    po = torch.exp(so - ahead(top))
    pp = torch.exp(sp - top.permute(1, 0, 2, 3).reshape(kv, rows * group, 1))
    total = back(po.sum(-1, keepdim=True)) + pp.sum(-1).reshape(kv, rows, group, 1).permute(1, 0, 2, 3)
    out = back(torch.matmul(po, vo)) + torch.bmm(pp, vp.permute(1, 0, 2)).reshape(kv, rows, group, head).permute(1, 0, 2, 3)
    st["out"].copy_((out / total).reshape(rows, heads * head))
    st["lse"].copy_((top + torch.log(total)).reshape(rows, heads))
    return {"out": st["out"], "lse": st["lse"]}


# ---- the framework's calls ---------------------------------------------------------------------------------------------
_kept = {}  # what a program keeps for its whole life: the context, the operators and their workspace


def _operators(c):
    import managedllama2_b200 as ml2
    if "ctx" not in _kept:
        _kept["ctx"] = ml2.CudaContext(torch.cuda.current_device())
    key = tuple(sorted((k, v) for k, v in c.items() if k != "name"))
    if key not in _kept:
        ctx = _kept["ctx"]
        if c["op"] == "tables":
            _kept[key] = ml2.BlockTables(ctx, c["page"])
        else:
            config = ml2.Config(c["heads"] * c["head_size"], 0, 1, c["heads"], c["kv_heads"], 0, 0)
            if c["op"] == "rope":
                _kept[key] = ml2.QKNormRoPE(ctx, config, c["rotary"])
            else:
                _kept[key] = ml2.PrefixAttention(ctx, config, c["page"])
    return _kept[key]


def _call(st):
    c = st["case"]
    if "operator" not in st:  # looked up once for the inputs, as a program holds it: not at every pass
        st["operator"] = _operators(c)
    op = st["operator"]
    if c["op"] == "tables":
        op.Forward(st["old"], st["new"], st["table"], st["free"], st["free_count"], st["lengths"], st["free_count_out"], st["start"],
                   st["slots"], st["positions"], st["refused"], st["offset"])
        return _of_tables(st)
    if c["op"] == "rope":
        op.Forward(st["q_out"], st["k_cache"], st["v_cache"], st["q"], st["k"], st["v"], st["qw"], st["kw"], st["positions"], st["slots"])
        return {"q": st["q_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    need = op.WorkspaceBytes(st["q"].shape[0], c["requests"], c["prefix"], st["most_length"])
    if "workspace" not in _kept or _kept["workspace"].numel() < need:
        _kept["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    op.Forward(st["out"], st["q"], st["k_prefix"], st["v_prefix"], st["k_cache"], st["v_cache"], st["table"], st["lengths"], st["start"],
               _kept["workspace"], st["most_length"], st["lse"])
    return {"out": st["out"], "lse": st["lse"]}


def run(st):
    if own:
        return _call(st)
    return {"tables": _plain_tables, "rope": _plain_rope, "attn": _plain_attn}[st["case"]["op"]](st)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        old, new = _lengths(case)
        page = case["page"]
        grown = sum(max(0, b - a) for a, b in zip(old, new))
        moved = sum(abs(_pages(b, page) - _pages(a, page)) for a, b in zip(old, new))
        held = sum(1 for a, b in zip(old, new) if b > a and a % page)
        return {"bytes": 4 * (5 * case["requests"] + 2 * grown + 2 * moved + held + 3), "flops": 0}
    heads, kv, head = case["heads"], case["kv_heads"], case["head_size"]
    if case["op"] == "rope":
        values = case["tokens"] * (heads + 2 * kv) * head
        turned = case["tokens"] * (heads + kv)
        return {"bytes": 4 * values + 8 * case["tokens"], "flops": turned * (3 * case["rotary"] + (4 * head if case["norm"] else 0))}
    own_len, new = _lengths(case)
    rows = sum(new)
    seen = sum(n * L - n * (n - 1) // 2 for L, n in zip(own_len, new)) + rows * case["prefix"]
    table = sum(_pages(x, case["page"]) for x in own_len)
    return {"bytes": 4 * kv * head * (case["prefix"] + sum(own_len)) + 4 * rows * heads * head + 4 * rows * heads + 4 * (table + 2 * len(new) + 1),
            "flops": 4 * heads * head * seen}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    st = prepare(case, seed)
    heads, kv, head = case["heads"], case["kv_heads"], case["head_size"]
    if case["op"] == "rope":
        half = case["rotary"] // 2
        turns = torch.tensor([10000.0 ** (-2.0 * i / case["rotary"]) for i in range(half)], dtype=torch.float64, device="cuda")
        unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), st["positions"].double()[:, None] * turns)
        live = torch.nonzero(st["slots"] >= 0)[:, 0]

        def turn(x, weight, n):
            x = x.double().reshape(x.shape[0], n, head)
            if weight is not None:
                x = weight.double() * x / (x.pow(2).sum(-1, keepdim=True) / head + 1e-5).sqrt()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * unit[:, None, :]
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], dim=-1).flatten(1)

        q, k, v = st["q_out"].double(), st["k_cache"].double(), st["v_cache"].double()
        q[live] = turn(st["q"], st["qw"], heads)[live]
        k[st["slots"][live].long()] = turn(st["k"], st["kw"], kv)[live]
        v[st["slots"][live].long()] = st["v"].double()[live]
        return {"q": q, "k_cache": k, "v_cache": v}
    own_len, new = _lengths(case)
    kp = st["k_prefix"].double().view(-1, kv, head).transpose(0, 1)
    vp = st["v_prefix"].double().view(-1, kv, head).transpose(0, 1)
    out, lse, row = [], [], 0
    for r, (length, count) in enumerate(zip(own_len, new)):
        i = torch.arange(length, device="cuda")
        at = st["table"][r].long()[torch.div(i, case["page"], rounding_mode="floor")] * case["page"] + torch.remainder(i, case["page"])
        k = st["k_cache"][at].double().view(length, kv, head).transpose(0, 1)
        v = st["v_cache"][at].double().view(length, kv, head).transpose(0, 1)
        q = st["q"][row:row + count].double().view(count, kv, heads // kv, head).permute(1, 2, 0, 3) / math.sqrt(head)
        s = torch.cat([q @ kp.mT[:, None], (q @ k.mT[:, None]).masked_fill(i > length - count + torch.arange(count, device="cuda")[:, None], -math.inf)], -1)
        z = torch.logsumexp(s, -1)
        p = torch.exp(s - z[..., None])
        o = p[..., :case["prefix"]] @ vp[:, None] + p[..., case["prefix"]:] @ v[:, None]
        out.append(o.permute(2, 0, 1, 3).reshape(count, heads * head))
        lse.append(z.permute(2, 0, 1).reshape(count, heads))
        row += count
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
