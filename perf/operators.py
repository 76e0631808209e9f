"""The serving operators between a layer's q/k/v projections and its output
projection, as measured cases: the step's block tables and slot map, rotary
positions with the append to the paged cache, and attention over a paged cache
whose requests share a prefix.

`run` computes a case either in plain torch operations (`own` false) or
through the library's calls in vqlab_b200.attention (`own` true); `exact`
computes the same outputs from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# 40 query heads over 8 key/value heads of 128 are the 5120-wide layer whose
# projections (5120 x 5120 and 1024 x 5120) the benchmark runs; the others are
# generic head layouts.


def listed():
    return [
        # one decode step of a small batch: a few requests, one new token each
        {"name": "tables decode 8", "op": "tables", "requests": 8, "page": 16, "width": 128, "context": 1500,
         "new": 1, "released": 0.0, "offset": 0},
        # a decode step of a large ragged batch in which some requests have just finished
        {"name": "tables decode 1000", "op": "tables", "requests": 1000, "page": 32, "width": 512, "context": 12000,
         "new": 1, "released": 0.05, "offset": 4099},
        # admission of a batch of long prompts behind a shared prefix
        {"name": "tables prompts 300", "op": "tables", "requests": 300, "page": 64, "width": 1024, "context": 0,
         "new": 600, "released": 0.1, "offset": 16001},

        # one token of one request: the latency of the smallest call
        {"name": "rotary 1 token", "op": "rotary", "tokens": 1, "heads": 40, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": False, "dtype": "bf16", "page": 16, "position": 5000, "amplitude": 1.0, "skipped": 0.0},
        # a decode batch at far positions, part of the head rotated, pairs interleaved
        {"name": "rotary 129 far", "op": "rotary", "tokens": 129, "heads": 32, "kv_heads": 4, "dim": 128, "rot": 64,
         "interleaved": True, "dtype": "fp16", "page": 32, "position": 900000, "amplitude": 1.2, "skipped": 0.1},
        # a prompt of a long-context layer, all of the head rotated
        {"name": "rotary 16385 prompt", "op": "rotary", "tokens": 16385, "heads": 40, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "dtype": "bf16", "page": 64, "position": 0, "amplitude": 1.0,
         "skipped": 0.0},

        # interactive decode: a few requests with short contexts and no shared prefix
        {"name": "attention decode 4", "op": "attention", "requests": 4, "q_len": 1, "context": 700, "prefix": 0,
         "heads": 40, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # a batch decoding behind one long system prompt, short own contexts
        {"name": "attention shared 64", "op": "attention", "requests": 64, "q_len": 1, "context": 500,
         "prefix": 16421, "heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # the largest shared decode: many requests, a long prefix and long own contexts
        {"name": "attention shared 250", "op": "attention", "requests": 250, "q_len": 1, "context": 2000,
         "prefix": 32768, "heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # long ragged contexts with nothing shared, several drafted tokens a request, small heads
        {"name": "attention drafts 24", "op": "attention", "requests": 24, "q_len": 4, "context": 15000, "prefix": 0,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "dtype": "fp16"},
        # ragged prompts behind a shared prefix, a key/value head for each query head
        {"name": "attention prompts 6", "op": "attention", "requests": 6, "q_len": 900, "context": 900,
         "prefix": 2051, "heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "dtype": "fp16"},
        # a long chunk of one prompt, with as much already in its cache
        {"name": "attention prompt 4096", "op": "attention", "requests": 1, "q_len": 4096, "context": 8192,
         "prefix": 0, "heads": 40, "kv_heads": 8, "dim": 128, "page": 128, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "attention", "attention"])
    if op == "tables":
        requests, page = _log(rng, 1, 1000), rng.choice([16, 32, 64, 128])
        prompts = rng.random() < 0.4
        new = _log(rng, 2, min(8192, 180000 // requests)) if prompts else 1
        context = 0 if prompts and rng.random() < 0.5 else _log(rng, 1, 12000)
        width = -(-(context + new) // page) + rng.randint(0, 40)
        return {"op": op, "requests": requests, "page": page, "width": width, "context": context, "new": new,
                "released": rng.choice([0.0, 0.05, 0.2]), "offset": rng.choice([0, _log(rng, 1, 30000)])}
    if op == "rotary":
        dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _log(rng, 1, 12000), "heads": kv * rng.choice([1, 3, 4, 5]), "kv_heads": kv,
                "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4, dim - 4]),
                "interleaved": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16"]),
                "page": rng.choice([16, 32, 64, 128]), "position": _log(rng, 1, 1000000),
                "amplitude": rng.choice([1.0, round(rng.uniform(1.0, 1.5), 3)]),
                "skipped": rng.choice([0.0, 0.0, 0.2])}
    dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
    case = {"op": op, "heads": kv * rng.choice([1, 3, 4, 5, 8]), "kv_heads": kv, "dim": dim,
            "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"])}
    kind = rng.choice(["decode", "shared", "prompts"])
    if kind == "decode":
        requests = _log(rng, 1, 100)
        case.update(requests=requests, q_len=rng.choice([1, 1, 1, 2, 5]), context=_log(rng, 8, 16000), prefix=0)
    elif kind == "shared":
        requests = _log(rng, 2, 200)
        case.update(requests=requests, q_len=rng.choice([1, 1, 1, 3, 17]), context=_log(rng, 20, 1500),
                    prefix=_log(rng, 64, 24000))
    else:
        requests = _log(rng, 1, 6)
        q_len = _log(rng, 20, 1500)
        case.update(requests=requests, q_len=q_len, context=q_len + _log(rng, 1, 1000),
                    prefix=rng.choice([0, _log(rng, 64, 3000)]))
    # no drawn case costs more than the largest listed ones, in arithmetic or in the plain form's memory
    while (case["requests"] * case["q_len"] * case["heads"] * (case["prefix"] + case["context"]) > 3.0e8
           or case["requests"] * case["context"] * case["kv_heads"] * dim > 5.0e8):
        if case["requests"] > 1:
            case["requests"] = case["requests"] * 2 // 3
        else:
            case["context"] = max(case["q_len"], case["context"] // 2)
            case["prefix"] //= 2
    return case


# ---- inputs


def _lengths(case, seed):
    """Ragged lengths, made on the host: every request's context before the step, its new tokens (-1: finished).
    A case has one set of lengths, so that its outputs have one shape; the seed says which request has which."""
    n = case["requests"]
    rng, order = np.random.default_rng([n, case["context"], 17]), np.random.default_rng([seed, 17]).permutation(n)
    if case["op"] == "tables":
        context = rng.integers(0, case["context"] + 1, n)
        new = rng.integers(1, case["new"] + 1, n) if case["new"] > 1 else np.ones(n, np.int64)
        new = np.where(rng.random(n) < case["released"], -1, new)
        return context[order], new[order]
    queries = np.full(n, case["q_len"]) if case["q_len"] < 8 else rng.integers(1, case["q_len"] + 1, n)
    queries[0] = case["q_len"]
    spare = np.maximum(case["context"] - queries, 0)
    total = queries + rng.integers(0, spare + 1)
    total[0] = queries[0] + spare[0]
    return (total - queries)[order], queries[order]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng([seed, 5])
    cuda = lambda a, t=torch.int32: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    state = {"case": dict(case)}
    if case["op"] == "tables":
        page, width = case["page"], case["width"]
        context, new = _lengths(case, seed)
        held = -(-context // page)
        need = np.where(new < 0, 0, -(-(context + np.maximum(new, 0)) // page) - held)
        used, pages = int(held.sum()), int(held.sum() + need.sum()) + 7
        order = rng.permutation(pages)
        table = np.full((len(new), width), -1, np.int64)
        row = np.repeat(np.arange(len(new)), held)
        table[row, np.arange(used) - np.repeat(np.cumsum(held) - held, held)] = order[:used]
        ring = np.full(pages, -1, np.int64)
        head = int(rng.integers(0, 10 * pages))  # the ring has been round several times
        ring[(head + np.arange(pages - used)) % pages] = order[used:]
        state.update(context=cuda(context), new=cuda(new), table=cuda(table), ring=cuda(ring),
                     counters=torch.tensor([head, head + pages - used, 0, 0], dtype=torch.int64, device="cuda"),
                     max_tokens=int(np.maximum(new, 0).sum()) + 5)  # the last ones are padding
        return state
    dt, dim, page = DTYPES[case["dtype"]], case["dim"], case["page"]
    kv_heads = case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] == "rotary":
        tokens, rot = case["tokens"], case["rot"]
        pages = -(-tokens // page) + 2
        fused = normal(tokens, case["heads"] + 2 * kv_heads, dim)  # q, k and v of one fused projection
        slots = rng.permutation(pages * page)[:tokens]
        slots = np.where(rng.random(tokens) < case["skipped"], -1, slots)
        first = case["position"]
        positions = first + np.arange(tokens) if first == 0 else rng.integers(0, first + 1, tokens)
        # base 1e6, in turns per position as fixed point of 64 fraction bits
        turns = [int((1e6 ** (-2.0 * i / rot) / (2 * math.pi)) * 2.0 ** 64) for i in range(rot // 2)]
        state.update(q=fused[:, :case["heads"]], k=fused[:, case["heads"]:case["heads"] + kv_heads],
                     v=fused[:, case["heads"] + kv_heads:], positions=cuda(positions), slots=cuda(slots),
                     turns=torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64,
                                        device="cuda"),
                     k_cache=normal(pages, kv_heads, page, dim), v_cache=normal(pages, kv_heads, page, dim))
        return state
    context, queries = _lengths(case, seed)
    total = context + queries
    held, n = -(-total // page), len(total)
    shared = -(-case["prefix"] // page)
    pages = int(held.sum()) + shared + 3
    order = rng.permutation(pages)
    table = np.full((n, int(held.max())), -1, np.int64)
    row = np.repeat(np.arange(n), held)
    table[row, np.arange(int(held.sum())) - np.repeat(np.cumsum(held) - held, held)] = order[shared:shared + int(held.sum())]
    state.update(q=normal(int(queries.sum()), case["heads"], dim), k_cache=normal(pages, kv_heads, page, dim),
                 v_cache=normal(pages, kv_heads, page, dim), table=cuda(table), kv_lens=cuda(total),
                 cu_q=cuda(np.concatenate([[0], np.cumsum(queries)])),
                 prefix_pages=cuda(order[:shared]) if shared else None, prefix_len=case["prefix"],
                 max_q=int(queries.max()), max_kv=int(total.max()))
    return state


# ---- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "rotary": _own_rotary, "attention": _own_attention}[op](state)
    return {"tables": _plain_tables, "rotary": _plain_rotary, "attention": _plain_attention}[op](state)


def _own_tables(s):
    from vqlab_b200 import attention
    t = attention.paged_tables(s["context"], s["new"], s["table"], s["ring"], s["counters"],
                               page_size=s["case"]["page"], max_tokens=s["max_tokens"],
                               position_offset=s["case"]["offset"])
    return {"table": t.block_table, "kv_lens": t.kv_lens, "cu_q": t.cu_q, "slots": t.slots,
            "positions": t.positions, "requests": t.requests, "ring": t.free_pages, "state": t.state}


def _own_rotary(s):
    from vqlab_b200 import attention
    q = attention.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["turns"], s["k_cache"], s["v_cache"],
                                s["slots"], interleaved=s["case"]["interleaved"],
                                amplitude=s["case"]["amplitude"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    from vqlab_b200 import attention
    return {"out": attention.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"],
                                              s["cu_q"], max_q_len=s["max_q"], max_kv_len=s["max_kv"],
                                              prefix_pages=s["prefix_pages"], prefix_len=s["prefix_len"])}


def _plain_tables(s):
    page, table, ring, most = s["case"]["page"], s["table"], s["ring"], s["max_tokens"]
    context, new = s["context"].long(), s["new"].long()
    (n, width), size, dev = table.shape, ring.numel(), table.device
    head, tail = s["counters"][0], s["counters"][1]
    gone, fresh = new < 0, new.clamp(min=0)
    held = (context + page - 1) // page
    column = torch.arange(width, device=dev)[None]
    # pages given back go to the ring's tail, in the order of requests and pages
    back = torch.where(gone, held, 0)
    back_end = back.cumsum(0)
    at = tail + (back_end - back)[:, None] + column
    given = gone[:, None] & (column < held[:, None])
    wide = torch.cat([ring, ring.new_zeros(1)])
    ring_out = wide.scatter(0, torch.where(given, at % size, size).reshape(-1), table.reshape(-1))[:size]
    tail_out = tail + back_end[-1]
    # pages asked for, in the order of requests
    pages = (context + fresh + page - 1) // page
    fits = pages <= width
    need = torch.where(gone | ~fits, 0, pages - held)
    need_end = need.cumsum(0)
    taken = ~gone & fits & ((need == 0) | (need_end <= tail_out - head))
    first = need_end - need
    index = head + first[:, None] + column - held[:, None]
    added = taken[:, None] & (column >= held[:, None]) & (column < pages[:, None])
    kept = ~gone[:, None] & (column < held[:, None])
    table_out = torch.where(added, ring_out[index % size], torch.where(kept, table, -1))
    kv = torch.where(gone, 0, torch.where(taken, context + fresh, context))
    end = fresh.cumsum(0)
    cu = torch.cat([end.new_zeros(1), end])
    token = torch.arange(most, device=dev)
    real = token < end[-1]
    request = torch.searchsorted(end, token, right=True).clamp(max=n - 1)
    place = context[request] + token - cu[request]
    its_page = table_out[request, (place // page).clamp(max=width - 1)]
    slot = torch.where(real & taken[request], its_page * page + place % page, -1)
    given_out = torch.where(taken, need, 0).sum()
    refused = (~gone & ~taken).sum()
    counters = torch.stack([head + given_out, tail_out, refused, torch.zeros_like(head)])
    i32 = torch.int32
    return {"table": table_out.to(i32), "kv_lens": kv.to(i32), "cu_q": cu.to(i32), "slots": slot.to(i32),
            "positions": torch.where(real, place + s["case"]["offset"], 0).to(i32),
            "requests": torch.where(real, request, -1).to(i32), "ring": ring_out, "state": counters}


def _turn(x, cos, sin, rot, interleaved):
    x = x.float()
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1)


def _plain_rotary(s):
    case, dt = s["case"], s["q"].dtype
    # the turns past the point, exact in 64-bit integers that wrap, then 32-bit arithmetic
    phase = s["positions"].long()[:, None] * s["turns"][None]
    angle = (phase >> 32).float() * (2 * math.pi / 2.0 ** 32)
    cos, sin = torch.cos(angle)[:, None] * case["amplitude"], torch.sin(angle)[:, None] * case["amplitude"]
    q = _turn(s["q"], cos, sin, case["rot"], case["interleaved"]).to(dt)
    k = _turn(s["k"], cos, sin, case["rot"], case["interleaved"]).to(dt)
    stored = s["slots"] >= 0
    slot = s["slots"][stored].long()
    where = (slot // case["page"], slice(None), slot % case["page"])
    s["k_cache"][where] = k[stored]
    s["v_cache"][where] = s["v"][stored]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _paged(cache, pages, tokens):
    """[..., tokens, kv_heads, dim] in 32 bits of the pages [..., n]."""
    x = cache[pages.clamp(min=0).long()].float().transpose(-3, -2)
    return x.flatten(-4, -3)[..., :tokens, :, :]


def _plain_attention(s):
    q, cu, kv_lens = s["q"], s["cu_q"].long(), s["kv_lens"].long()
    (tokens, heads, dim), dev = q.shape, q.device
    kv_heads, most, longest = s["k_cache"].shape[1], s["max_q"], s["max_kv"]
    group, n = heads // kv_heads, kv_lens.numel()
    queries = cu[1:] - cu[:-1]
    i = torch.arange(most, device=dev)
    real = i[None] < queries[:, None]
    source = (cu[:-1, None] + i[None]).clamp(max=tokens - 1)
    x = q.float()[source].view(n, most, kv_heads, group, dim)
    k, v = (_paged(c, s["table"], longest) for c in (s["k_cache"], s["v_cache"]))
    scores = torch.einsum("rqhgd,rkhd->rhgqk", x, k)
    j = torch.arange(longest, device=dev)
    seen = j[None, None] <= (kv_lens - queries)[:, None, None] + i[None, :, None]
    seen = seen & (j[None, None] < kv_lens[:, None, None])
    scores = scores.mul_(dim ** -0.5).masked_fill_(~seen[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    if s["prefix_len"]:
        pk, pv = (_paged(c, s["prefix_pages"], s["prefix_len"]) for c in (s["k_cache"], s["v_cache"]))
        far = torch.einsum("rqhgd,khd->rhgqk", x, pk).mul_(dim ** -0.5)
        top = torch.maximum(top, far.amax(-1, keepdim=True))
    top = torch.where(torch.isinf(top), 0.0, top)
    scores = scores.sub_(top).exp_()
    total = scores.sum(-1)
    # a place that holds no token of the request is not multiplied, whatever it holds
    v = torch.where((j[None] < kv_lens[:, None])[..., None, None], v, 0.0)
    out = torch.einsum("rhgqk,rkhd->rqhgd", scores, v)
    if s["prefix_len"]:
        far = far.sub_(top).exp_()
        total = total + far.sum(-1)
        out = out + torch.einsum("rhgqk,khd->rqhgd", far, pv)
    total = total.permute(0, 3, 1, 2)[..., None]
    out = torch.where(total > 0, out / total, 0.0)
    return {"out": out.reshape(n, most, heads, dim)[real].to(q.dtype)}


# ---- what a pass cannot do without


def work(case):
    if case["op"] == "tables":
        context, new = _lengths(case, 1)
        n, tokens = case["requests"], int(np.maximum(new, 0).sum()) + 5
        ring = int((-(-context // case["page"])).sum() + tokens // case["page"])
        return {"bytes": 4 * (2 * n * case["width"] + 2 * ring + 4 * n + 3 * tokens) + 64, "flops": 0}
    dim = case["dim"]
    if case["op"] == "rotary":
        heads = case["heads"] + 2 * case["kv_heads"]
        return {"bytes": case["tokens"] * (4 * heads * dim + 8) + 4 * case["rot"],
                "flops": 3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]}
    context, queries = _lengths(case, 1)
    tokens = int(queries.sum())
    pairs = int((queries * (context + case["prefix"]) + queries * (queries + 1) // 2).sum())
    keys = int((context + queries).sum()) + case["prefix"]
    return {"bytes": 4 * tokens * case["heads"] * dim + 4 * keys * case["kv_heads"] * dim + 4 * (keys // case["page"]),
            "flops": 4 * pairs * case["heads"] * dim}


# ---- the definitions in 64 bits


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rotary":
        rot, page = case["rot"], case["page"]
        turns = [int(t) % (1 << 64) for t in s["turns"].tolist()]
        phase = np.array([[(p * t % (1 << 64)) / 2.0 ** 64 for t in turns] for p in s["positions"].tolist()])
        z = torch.from_numpy(case["amplitude"] * np.exp(2j * np.pi * phase)).cuda()[:, None]

        def turned(x):
            x = x.double()
            first, second = ((slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else
                             (slice(0, rot // 2), slice(rot // 2, rot)))
            w = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
            x[..., first], x[..., second] = w.real, w.imag
            return x

        out = {"q": turned(s["q"])}
        for name, new in (("k_cache", turned(s["k"])), ("v_cache", s["v"].double())):
            flat = s[name].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
            keep = (s["slots"] >= 0).nonzero()[:, 0]
            flat[s["slots"][keep].long()] = new[keep]
            out[name] = flat.view(-1, page, case["kv_heads"], case["dim"]).transpose(1, 2).contiguous()
        return out
    q, cu, lens = s["q"].double(), s["cu_q"].tolist(), s["kv_lens"].tolist()
    group, page, prefix = case["heads"] // case["kv_heads"], case["page"], case["prefix"]
    out = torch.empty_like(q)

    def rows(cache, pages, count, head):
        return cache[pages.long(), head].double().reshape(-1, case["dim"])[:count]

    shared = [[rows(c, s["prefix_pages"], prefix, h) for c in (s["k_cache"], s["v_cache"])] if prefix else None
              for h in range(case["kv_heads"])]
    for r, length in enumerate(lens):
        a, b = cu[r], cu[r + 1]
        own_pages = s["table"][r, :-(-length // page)]
        for h in range(case["kv_heads"]):
            k, v = (rows(c, own_pages, length, h) for c in (s["k_cache"], s["v_cache"]))
            if prefix:
                k, v = torch.cat([shared[h][0], k]), torch.cat([shared[h][1], v])
            x = q[a:b, h * group:(h + 1) * group].reshape(-1, case["dim"])
            weights = x @ k.T / math.sqrt(case["dim"])
            if b - a > 1:
                last = prefix + length - (b - a) + torch.arange(b - a, device="cuda").repeat_interleave(group)
                weights.masked_fill_(torch.arange(k.shape[0], device="cuda")[None] > last[:, None], -torch.inf)
            weights = torch.softmax(weights, -1)
            out[a:b, h * group:(h + 1) * group] = (weights @ v).view(b - a, group, case["dim"])
    return {"out": out}
