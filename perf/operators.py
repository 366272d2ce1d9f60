"""Timed cases of the paged operators: many requests that share one key / value cache held in 4 bits, in pages.

  plan    page tables and slot maps of one step, built on the device from the requests' lengths (kv_plan)
  store   a step's keys and values quantized into their slots (kv_store), and read back as the values kept (kv_load)
  attend  attention of each request's newest tokens over its pages (kv_attend)
  prompt  attention of packed prompts of different lengths over keys and values in 16 bits (attend_packed)

A page holds `page` tokens of every key / value head.  A row of a head is kept in groups of 32 values: with m the value of
largest magnitude (the first of equal ones), d = m / -8 rounded to f16 and q = floor(x / d + 8.5) within 0 .. 15, the value
kept is (q - 8) * d.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32

# heads of a llama decoder of 8B, 1B and 70B parameters
HEADS_8B = dict(heads=32, kv_heads=8, dim=128)
HEADS_1B = dict(heads=32, kv_heads=4, dim=64)
HEADS_70B = dict(heads=64, kv_heads=8, dim=128)


def listed():
    return [
        # serving: sixteen conversations, a token each; nothing but latency
        dict(name="plan 16 x 1", kind="plan", requests=16, shortest=120, longest=600, ended=0, prompts=0, prompt=0, page=16),
        # serving: a thousand requests, a tenth of them over, an eighth new with long prompts
        dict(name="plan 1000 mixed", kind="plan", requests=1000, shortest=30, longest=4000, ended=100, prompts=125, prompt=1500, page=16),
        # the new token of sixteen conversations
        dict(name="store 16 x 1 8b bf16", kind="store", type="bf16", requests=16, cached=333, fresh=1, page=16, kv_heads=8, dim=128),
        # a handful of questions, f32 activations, a size that fits no tile
        dict(name="store 5 x 77 1b f32", kind="store", type="f32", requests=5, cached=40, fresh=77, page=16, kv_heads=4, dim=64),
        # long documents
        dict(name="store 8 x 4095 8b f16", kind="store", type="f16", requests=8, cached=0, fresh=4095, page=64, kv_heads=8, dim=128),
        # one short conversation with a small model: latency
        dict(name="attend 1 x 333 1b f16", kind="attend", type="f16", requests=1, shortest=333, longest=333, tokens=1, page=16, **HEADS_1B),
        # sixteen conversations of different lengths, as the batch decode case has them
        dict(name="attend 16 x 120-600 8b bf16", kind="attend", type="bf16", requests=16, shortest=120, longest=600, tokens=1, page=16, **HEADS_8B),
        # one reader of a very long document, three guessed tokens checked beside the newest
        dict(name="attend 1 x 100001 8b f16", kind="attend", type="f16", requests=1, shortest=100001, longest=100001, tokens=4, page=64, **HEADS_8B),
        # a full server: 64 long conversations
        dict(name="attend 64 x 1000-8000 70b bf16", kind="attend", type="bf16", requests=64, shortest=1000, longest=8000, tokens=1, page=16, **HEADS_70B),
        # one ordinary question to a small model
        dict(name="prompt 1 x 333 1b f16", kind="prompt", type="f16", requests=1, shortest=333, longest=333, before=0, **HEADS_1B),
        # a step of mixed questions, each behind what its conversation holds already
        dict(name="prompt 13 x 17-600 8b bf16", kind="prompt", type="bf16", requests=13, shortest=17, longest=600, before=257, **HEADS_8B),
        # two long documents
        dict(name="prompt 2 x 4100-8190 8b bf16", kind="prompt", type="bf16", requests=2, shortest=4100, longest=8190, before=0, **HEADS_8B),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: plans of 1 to 2000 requests; stores of 1 to 32,000 tokens; attention of 1 to 64 requests and 1 to 8 new
    tokens each over 10 to 100,000 cached ones; 1 to 32 packed prompts of 1 to 8,000 tokens behind 0 to 2,000 earlier ones.
    Head sizes 32 to 128, 1 to 16 key / value heads, 1 to 16 query heads to each."""
    kind = rng.choice(["plan", "store", "attend", "attend", "prompt", "prompt"])
    page = rng.choice([16, 16, 32, 64, 128])
    dim = rng.choice([32, 64, 64, 96, 128, 128, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    if kind == "plan":
        n = _log(rng, 1, 2000)
        ended = rng.randint(0, n // 4)
        prompts = rng.randint(0, n - ended)
        prompt = _log(rng, 1, 4000)
        while prompts * prompt > 180000:
            prompt = max(1, prompt // 2)
        shortest = _log(rng, 1, 500)
        longest = shortest + _log(rng, 1, 4000)
        return dict(kind="plan", requests=n, shortest=shortest, longest=longest, ended=ended, prompts=prompts, prompt=prompt, page=page)
    if kind == "store":
        n = rng.randint(1, 24)
        fresh = _log(rng, 1, 8000)
        t = rng.choice(list(TYPES))
        while n * fresh * kv * dim > 32760 * (512 if t == "f32" else 1024):
            fresh = max(1, fresh // 2)
        return dict(kind="store", type=t, requests=n, cached=rng.choice([0, rng.randint(1, 500)]), fresh=fresh, page=page,
                    kv_heads=kv, dim=dim)
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    heads = dict(heads=kv * group, kv_heads=kv, dim=dim)
    if kind == "attend":
        n, tokens = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 4, 8])
        shortest = _log(rng, 10, 4000)
        longest = shortest + rng.choice([0, _log(rng, 1, 96000)])
        while n * (shortest + longest) // 2 * kv * dim * max(1, tokens * group // 8) > 64 * 4500 * 1024:
            longest = max(1, longest // 2)
            shortest = min(shortest, longest)
        return dict(kind="attend", type=rng.choice(["f16", "bf16"]), requests=n, shortest=shortest, longest=longest, tokens=min(tokens, shortest),
                    page=page, **heads)
    n = rng.randint(1, 32)
    shortest = _log(rng, 1, 2000)
    longest = shortest + rng.choice([0, _log(rng, 1, 6000)])
    before = rng.choice([0, 0, rng.randint(1, 2000)])
    while n * kv * group * dim * longest * (longest / 2 + before) > 32 * 128 * 1.2e8 or n * kv * group * longest > 32 * 12290:
        if longest > 1:
            longest //= 2
            shortest = min(shortest, longest)
        else:
            n = max(1, n // 2)
    return dict(kind="prompt", type=rng.choice(["f16", "bf16"]), requests=n, shortest=shortest, longest=longest, before=before, **heads)


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _spread(n, lo, hi):
    """n lengths from lo to hi, in no order."""
    return [lo + (hi - lo) * ((7 * i) % n) // max(1, n - 1) if n % 7 else lo + (hi - lo) * ((5 * i) % n) // max(1, n - 1) for i in range(n)]


def _ints(v, t=torch.int32):
    return torch.tensor(v, dtype=t, device="cuda")


def _cumulated(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _pages(n, page):
    return (n + page - 1) // page


def _tables(g, lengths, page, spare=3):
    """Page tables of requests of these lengths, pages in a random order; the count of pages of the cache."""
    counts = [_pages(n, page) for n in lengths]
    total = sum(counts) + spare
    width = max(1, max(counts))
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, total


def _slots(table, begin, end, page):
    """Slot of each token begin[b] .. end[b]-1 of each request, packed."""
    out = []
    for b, (lo, hi) in enumerate(zip(begin, end)):
        p = torch.arange(lo, hi, device="cuda")
        out.append(table[b, p // page].long() * page + p % page)
    return torch.cat(out)


def _activations(g, rows, heads, dim, t, outliers):
    """Keys have channels that are larger than others in every row, queries and values do not."""
    x = torch.randn((rows, heads, dim), generator=g, device="cuda")
    if outliers:
        gain = 1.0 + 3.0 * (torch.rand((heads, dim), generator=g, device="cuda") < 0.05).float()
        for i in range(0, rows, 65536):
            x[i:i + 65536] *= gain
    return x.to(t)


def _plan_lengths(c):
    """(tokens cached, tokens that the step brings; -1: the request is over)"""
    n = c["requests"]
    cached = _spread(n, c["shortest"], c["longest"])
    fresh = [1] * n
    for i in range(c["ended"]):
        fresh[i * n // max(1, c["ended"])] = -1
    left = c["prompts"]
    for i in range(n - 1, -1, -1):
        if left and fresh[i] == 1:
            cached[i], fresh[i] = (0 if i % 3 else cached[i] // 2), max(1, c["prompt"] * (1 + i % 5) // 5)
            left -= 1
    return cached, fresh


def _plan_inputs(c, seed):
    g = _generator(seed)
    cached, fresh = _plan_lengths(c)
    page, n = c["page"], c["requests"]
    have = [_pages(x, page) for x in cached]
    want = [_pages(x + max(f, 0), page) for x, f in zip(cached, fresh)]
    need = sum(w - h for w, h, f in zip(want, have, fresh) if f >= 0)
    # nine tenths of the pages that are wanted are free beside what the ended requests give back: the last requests wait
    back = sum(h for h, f in zip(have, fresh) if f < 0)
    free = max(1, need * 9 // 10 - back if c["prompts"] > 8 else need)
    pages = sum(have) + free + 5000  # the others are held by requests that are not in this step
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n, max(want) + 1), -1, dtype=torch.int32, device="cuda")
    at = _cumulated(have)
    for b in range(n):
        table[b, :have[b]] = ids[at[b]:at[b + 1]]
    stack = torch.zeros(pages, dtype=torch.int32, device="cuda")
    stack[:free] = ids[at[-1]:at[-1] + free]
    tokens = sum(max(f, 0) for f in fresh)
    return dict(cached=_ints(cached), fresh=_ints(fresh), table=table, stack=stack, free=_ints([free]), capacity=(tokens + 63) // 64 * 64)


def _store_inputs(c, seed):
    g = _generator(seed)
    n, t = c["requests"], TYPES[c["type"]]
    cached = [(c["cached"] * (i + 1)) // n for i in range(n)]
    fresh = [max(1, c["fresh"] - 3 * i) if c["fresh"] > 1 else 1 for i in range(n)]
    lengths = [a + b for a, b in zip(cached, fresh)]
    table, pages = _tables(g, lengths, c["page"])
    begin = _cumulated(fresh)
    slots = _slots(table, cached, lengths, c["page"])
    # a step of fixed size has a few rows behind the last request that belong to none
    slots = torch.cat([slots, torch.full((2,), -1, dtype=torch.int64, device="cuda")])
    rows = begin[-1] + 2
    k = _activations(g, rows, c["kv_heads"], c["dim"], t, True)
    v = _activations(g, rows, c["kv_heads"], c["dim"], t, False)
    return dict(k=k, v=v, slots=slots, table=table, pages=pages, first=_ints(cached), lengths=_ints(lengths), begin=_ints(begin), rows=rows)


def _attend_inputs(c, seed):
    g = _generator(seed)
    t = TYPES[c["type"]]
    lengths = _spread(c["requests"], c["shortest"], c["longest"])
    table, pages = _tables(g, lengths, c["page"])
    total = sum(lengths)
    k = _activations(g, total, c["kv_heads"], c["dim"], torch.float16, True)
    v = _activations(g, total, c["kv_heads"], c["dim"], torch.float16, False)
    q = _activations(g, c["requests"] * c["tokens"], c["heads"], c["dim"], t, False)
    return dict(q=q, k=k, v=v, table=table, pages=pages, lengths=lengths, slots=_slots(table, [0] * c["requests"], lengths, c["page"]))


def _prompt_lengths(c):
    queries = _spread(c["requests"], c["shortest"], c["longest"])
    keys = [n + (c["before"] * (i % 4)) // 3 for i, n in enumerate(queries)]
    return queries, keys


def _prompt_inputs(c, seed):
    g = _generator(seed)
    t = TYPES[c["type"]]
    queries, keys = _prompt_lengths(c)
    q = _activations(g, sum(queries), c["heads"], c["dim"], t, False)
    k = _activations(g, sum(keys), c["kv_heads"], c["dim"], t, True)
    v = _activations(g, sum(keys), c["kv_heads"], c["dim"], t, False)
    return dict(q=q, k=k, v=v, query_begin=_cumulated(queries), key_begin=_cumulated(keys))


# ---------------------------------------------------------------- states
_backends = []


def _backend():
    """One context for all states, as a program keeps it."""
    import emel_cpp_b200 as eb
    if not _backends:
        _backends.append(eb.Backend(0))
    return _backends[0]


def prepare(case, seed):
    c = case
    s = {"plan": _prepare_plan, "store": _prepare_store, "attend": _prepare_attend, "prompt": _prepare_prompt}[c["kind"]](c, seed)
    s["case"] = c
    torch.cuda.synchronize()
    return s


def _prepare_plan(c, seed):
    s = _plan_inputs(c, seed)
    if own:
        from emel_cpp_b200 import paged
        n, cap = c["requests"], s["capacity"]
        out = dict(lengths=torch.zeros(n, dtype=torch.int32, device="cuda"), query_begin=torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
                   key_begin=torch.zeros(n + 1, dtype=torch.int32, device="cuda"), slots=torch.zeros(cap, dtype=torch.int64, device="cuda"),
                   positions=torch.zeros(cap, dtype=torch.int32, device="cuda"), free=torch.zeros(1, dtype=torch.int32, device="cuda"),
                   shortage=torch.zeros(1, dtype=torch.int32, device="cuda"))
        s["backend"], s["out"] = _backend(), out
        s["request"] = paged.plan_request(
            cached=s["cached"], fresh=s["fresh"], table=s["table"], table_width=s["table"].shape[1], free_pages=s["stack"], pages=s["stack"].numel(),
            free_count=s["free"], free_left=out["free"], lengths=out["lengths"], query_begin=out["query_begin"], key_begin=out["key_begin"],
            slots=out["slots"], positions=out["positions"], shortage=out["shortage"], requests=n, page_tokens=c["page"], token_capacity=cap)
        out.update(table=s["table"], stack=s["stack"])
    return s


def _own_pages(c, count):
    from emel_cpp_b200 import paged
    data = torch.zeros(count * paged.page_bytes(c["dim"], c["kv_heads"], c["page"]), dtype=torch.uint8, device="cuda")
    return data, paged.pages(data, count, c["page"], c["kv_heads"], c["dim"])


def _prepare_store(c, seed):
    s = _store_inputs(c, seed)
    if own:
        from emel_cpp_b200 import paged
        s["backend"] = _backend()
        s["data"], cache = _own_pages(c, s["pages"])
        s["out"] = (torch.zeros_like(s["k"]), torch.zeros_like(s["v"]))
        s["request"] = paged.store_request(cache, s["k"], s["v"], c["type"], s["slots"], s["rows"])
        s["load"] = paged.load_request(cache, *s["out"], c["type"], s["table"], s["table"].shape[1], s["lengths"], s["begin"], c["requests"], s["rows"],
                                       first=s["first"])
    return s


def _prepare_attend(c, seed):
    s = _attend_inputs(c, seed)
    if own:
        from emel_cpp_b200 import paged
        s["backend"] = _backend()
        s["data"], cache = _own_pages(c, s["pages"])
        torch.cuda.synchronize()
        _do(s["backend"].kv_store(paged.store_request(cache, s["k"], s["v"], "f16", s["slots"], s["slots"].numel())), s["backend"])
        s["backend"].sync()
        s["out"] = torch.zeros_like(s["q"])
        s["lengths_dev"] = _ints(s["lengths"])
        begin = None
        if c["tokens"] > 1:
            begin = s["begin"] = _ints([c["tokens"] * i for i in range(c["requests"] + 1)])
        s["request"] = paged.attend_request(cache, s["q"], s["out"], c["type"], s["table"], s["table"].shape[1], s["lengths_dev"], c["requests"],
                                            c["heads"], c["requests"] * c["tokens"], query_begin=begin, max_queries=c["tokens"],
                                            scale=c["dim"] ** -0.5)
    else:
        s["quants"] = []
        for x in (s["k"], s["v"]):
            q = torch.empty((s["pages"] * c["page"], c["kv_heads"], c["dim"]), dtype=torch.uint8, device="cuda")
            d = torch.empty((s["pages"] * c["page"], c["kv_heads"], c["dim"] // GROUP), dtype=torch.float16, device="cuda")
            for i in range(0, x.shape[0], 32768):
                part, at = x[i:i + 32768], s["slots"][i:i + 32768]
                pq, pd = _quantize(part)
                q[at], d[at] = pq.view(part.shape), pd
            s["quants"].append((q, d))
    del s["k"], s["v"]
    return s


def _prepare_prompt(c, seed):
    s = _prompt_inputs(c, seed)
    if own:
        from emel_cpp_b200 import paged
        s["backend"] = _backend()
        s["out"] = torch.zeros_like(s["q"])
        s["begins"] = (_ints(s["query_begin"]), _ints(s["key_begin"]))
        s["request"] = paged.packed_request(s["q"], s["k"], s["v"], s["out"], c["type"], *s["begins"], c["requests"], c["heads"], c["kv_heads"], c["dim"],
                                            s["query_begin"][-1], s["key_begin"][-1], max_queries=max(_prompt_lengths(c)[0]), causal=True,
                                            scale=c["dim"] ** -0.5)
    return s


# ---------------------------------------------------------------- one pass
def _do(ok, backend):
    if not ok:
        raise RuntimeError(f"refused with error mask {backend.last_error}")


def run(state):
    kind = state["case"]["kind"]
    if own:
        be = state["backend"]
        if kind == "plan":
            _do(be.kv_plan(state["request"]), be)
        elif kind == "store":
            _do(be.kv_store(state["request"]), be)
            _do(be.kv_load(state["load"]), be)
        elif kind == "attend":
            _do(be.kv_attend(state["request"]), be)
        else:
            _do(be.attend_packed(state["request"]), be)
        return state["out"]
    return {"plan": _run_plan, "store": _run_store, "attend": _run_attend, "prompt": _run_prompt}[kind](state)


def _before(x):
    """Sums of what stands before each place, and behind the last."""
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=x.device), x.long().cumsum(0)])


def _run_plan(s):
    page, cap = s["case"]["page"], s["capacity"]
    cached, fresh, table, stack = s["cached"].long(), s["fresh"].long(), s["table"].clone(), s["stack"].clone()
    n = cached.numel()
    over = fresh < 0
    new = fresh.clamp(min=0)
    have = (cached + page - 1) // page
    need = torch.where(over, 0, (cached + new + page - 1) // page - have)
    # the ended requests' pages go on top of the stack, in order; new pages come from its top
    columns = torch.arange(table.shape[1], device="cuda")
    back = table[over.unsqueeze(1) & (columns < have.unsqueeze(1))]
    free = s["free"].long()
    top = free + back.numel()
    upto = need.cumsum(0)
    granted = ~over & ((need == 0) | (upto <= top))
    grant = torch.where(granted, new, 0)
    all_free = torch.cat([stack[:int(free)], back])
    takes = torch.where(granted, need, 0)
    owner = torch.repeat_interleave(torch.arange(n, device="cuda"), takes)
    nth = torch.arange(owner.numel(), device="cuda")
    table[owner, have[owner] + nth - _before(takes)[owner]] = all_free[top - 1 - nth]
    left = top - takes.sum()
    held = torch.arange(back.numel(), device="cuda")
    kept = held[free + held < left]
    stack[free + kept] = back[kept]
    lengths = torch.where(over, 0, cached + grant)
    query_begin = _before(new)
    token = torch.arange(cap, device="cuda")
    request = torch.searchsorted(query_begin[1:].contiguous(), token, right=True).clamp(max=n - 1)
    live = token < query_begin[-1]
    position = torch.where(live, cached[request] + token - query_begin[request], 0)
    place = table[request, (position // page).clamp(max=table.shape[1] - 1)].long() * page + position % page
    slots = torch.where(live & granted[request], place, -1)
    return dict(lengths=lengths.int(), query_begin=query_begin.int(), key_begin=_before(lengths).int(), slots=slots, positions=position.int(),
                free=left.int(), shortage=(upto[-1:] - top).clamp(min=0).int(), table=table, stack=stack)


def _quantize(x):
    """Quants 0 .. 15 and f16 scales of each group of 32 values; quotients in 64 bits, where none falls on a border that it does not meet."""
    g = x.double().view(*x.shape[:-1], -1, GROUP)
    top = g.gather(-1, g.abs().argmax(-1, keepdim=True))
    d = (top / -8.0).clamp(-65504.0, 65504.0).half().double()
    q = torch.where(d == 0, 8.0, (g / torch.where(d == 0, 1.0, d) + 8.5).floor().clamp(0, 15))
    return q.to(torch.uint8), d.half().squeeze(-1)


def _values(q, d):
    return (q.float().view(*d.shape, GROUP) - 8.0) * d.float().unsqueeze(-1)


def _run_store(s):
    out = []
    for x in (s["k"], s["v"]):
        y = torch.zeros_like(x)
        for i in range(0, s["rows"] - 2, 8192):
            part = x[i:min(i + 8192, s["rows"] - 2)]
            y[i:i + part.shape[0]] = _values(*_quantize(part)).view(part.shape).to(x.dtype)
        out.append(y)
    return tuple(out)


def _attention(q, k, v, scale):
    """q {n, heads, dim}, k and v {L, kv_heads, dim} in f32; query i sees the first L - n + i + 1 keys."""
    n, heads, dim = q.shape
    length, kv = k.shape[0], k.shape[1]
    group = heads // kv
    out = torch.empty_like(q)
    step = max(1, int(3e8) // (group * length))
    for h in range(kv):
        keys, values = k[:, h].t().contiguous(), v[:, h].contiguous()
        for i in range(0, n, step):
            rows = q[i:i + step, h * group:(h + 1) * group]
            score = (rows.reshape(-1, dim) @ keys).view(rows.shape[0], group, length) * scale
            sees = torch.arange(i, i + rows.shape[0], device=q.device) + length - n
            score.masked_fill_((torch.arange(length, device=q.device) > sees.unsqueeze(1)).unsqueeze(1), -math.inf)
            top = score.amax(-1, keepdim=True)
            weight = (score - torch.where(top == -math.inf, 0.0, top)).exp_()
            total = weight.sum(-1, keepdim=True)
            mixed = (weight.view(-1, length) @ values).view(rows.shape)
            out[i:i + step, h * group:(h + 1) * group] = mixed / torch.where(total == 0, 1.0, total)
    return out


def _run_attend(s):
    c = s["case"]
    n, page = c["tokens"], c["page"]
    out = torch.empty_like(s["q"])
    for b, length in enumerate(s["lengths"]):
        p = torch.arange(length, device="cuda")
        at = s["table"][b, p // page].long() * page + p % page
        k, v = (_values(q[at], d[at]).view(length, c["kv_heads"], c["dim"]) for q, d in s["quants"])
        out[b * n:(b + 1) * n] = _attention(s["q"][b * n:(b + 1) * n].float(), k, v, c["dim"] ** -0.5).to(out.dtype)
    return out


def _run_prompt(s):
    out = torch.empty_like(s["q"])
    qb, kb = s["query_begin"], s["key_begin"]
    for b in range(s["case"]["requests"]):
        q, k, v = s["q"][qb[b]:qb[b + 1]], s["k"][kb[b]:kb[b + 1]], s["v"][kb[b]:kb[b + 1]]
        out[qb[b]:qb[b + 1]] = _attention(q.float(), k.float(), v.float(), s["case"]["dim"] ** -0.5).to(out.dtype)
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "plan":
        cached, fresh = _plan_lengths(c)
        tokens = sum(max(f, 0) for f in fresh)
        moved = sum(_pages(a + max(f, 0), c["page"]) - _pages(a, c["page"]) if f >= 0 else _pages(a, c["page"]) for a, f in zip(cached, fresh))
        # lengths in and out, both running sums, each page's id where it comes from and goes to, slot and position of each token
        return {"bytes": 20 * c["requests"] + 8 * moved + 12 * tokens, "flops": 0}
    if c["kind"] == "store":
        tokens = c["requests"] * c["fresh"] if c["fresh"] == 1 else sum(max(1, c["fresh"] - 3 * i) for i in range(c["requests"]))
        size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]]
        values = 2 * tokens * c["kv_heads"] * c["dim"]
        return {"bytes": values * (2 * size + 2 * 18 / 32) + 8 * tokens, "flops": 4 * values}
    if c["kind"] == "attend":
        lengths = _spread(c["requests"], c["shortest"], c["longest"])
        n = c["tokens"]
        seen = sum(sum(x - n + i + 1 for i in range(n)) for x in lengths)
        values = 2 * sum(lengths) * c["kv_heads"] * c["dim"]
        return {"bytes": values * 18 / 32 + 4 * c["requests"] * n * c["heads"] * c["dim"], "flops": 4 * seen * c["heads"] * c["dim"]}
    queries, keys = _prompt_lengths(c)
    seen = sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(queries, keys))
    return {"bytes": 4 * (sum(queries) * c["heads"] + sum(keys) * c["kv_heads"]) * c["dim"], "flops": 4 * seen * c["heads"] * c["dim"]}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _kept(x):
    """What the cache keeps of rows x, one threshold at a time: q is the count of borders (j - 8.5) d, j = 1 .. 15, that x has reached."""
    rows = x.double().reshape(-1, GROUP)
    size = rows.abs()
    first = (size == size.max(1, keepdim=True).values).int().argmax(1)
    d = (rows[torch.arange(rows.shape[0], device=x.device), first] / -8).half().double().clamp(-65504, 65504).unsqueeze(1)
    q = torch.zeros_like(rows)
    for j in range(1, 16):
        q += ((rows - (j - 8.5) * d) * d.sign() >= 0).double()
    return torch.where(d == 0, torch.zeros_like(rows), (q - 8) * d).view(x.shape)


def _softmax_mix(q, k, v, ahead, scale):
    """One head: rows of q, which see `ahead` + 1, `ahead` + 2, ... keys."""
    score = torch.mm(q, k.t()) * scale
    hidden = torch.ones_like(score, dtype=torch.bool).triu_(ahead + 1)
    score[hidden] = -math.inf
    return torch.mm(torch.softmax(score, 1), v)


def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return None
    if c["kind"] == "store":
        s = _store_inputs(c, seed)
        out = []
        for x in (s["k"], s["v"]):
            y = torch.cat([_kept(x[i:i + 4096]) for i in range(0, x.shape[0], 4096)])
            y[-2:] = 0
            out.append(y)
        return tuple(out)
    scale = c["dim"] ** -0.5
    group = c["heads"] // c["kv_heads"]
    if c["kind"] == "attend":
        s = _attend_inputs(c, seed)
        queries, keys = [c["tokens"]] * c["requests"], s["lengths"]
    else:
        s = _prompt_inputs(c, seed)
        queries, keys = _prompt_lengths(c)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    qa, ka = 0, 0
    for n, length in zip(queries, keys):
        for h in range(c["kv_heads"]):
            k, v = s["k"][ka:ka + length, h], s["v"][ka:ka + length, h]
            k, v = (_kept(k), _kept(v)) if c["kind"] == "attend" else (k.double(), v.double())
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                for j in range(h * group, (h + 1) * group):
                    out[qa + i:qa + i + m, j] = _softmax_mix(s["q"][qa + i:qa + i + m, j].double(), k, v, length - n + i, scale)
        qa, ka = qa + n, ka + length
    return out
