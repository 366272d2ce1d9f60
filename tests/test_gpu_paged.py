"""The paged operators on the GPU against plain 64-bit arithmetic (tests/paged_plain.py)."""
import numpy as np
import pytest
import torch

import emel_cpp_b200 as eb
from emel_cpp_b200 import paged
from tests import paged_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = eb.Backend(0)
    yield b
    b.close()


def dev(x, t=torch.int32):
    return torch.tensor(x, dtype=t, device="cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def done(be, ok):
    assert ok, be.last_error
    assert be.sync(), be.last_error


# ---------------------------------------------------------------- plan
class Step:
    """Arrays of a plan of n requests."""

    def __init__(self, n, width, pages, page, capacity, in_place=False, stride=None):
        z = lambda k, t=torch.int32: torch.full((k,), -77, dtype=t, device="cuda")  # noqa: E731
        self.n, self.width, self.page, self.capacity = n, width, page, capacity
        self.cached, self.fresh = z(n), z(n)
        self.table = torch.full((n, stride or width), -1, dtype=torch.int32, device="cuda")
        self.stack, self.count = z(pages), z(1)
        self.lengths, self.left = (self.cached, self.count) if in_place else (z(n), z(1))
        self.query_begin, self.key_begin = z(n + 1), z(n + 1)
        self.slots, self.positions, self.shortage = z(capacity, torch.int64), z(capacity), z(1)

    def request(self):
        return paged.plan_request(cached=self.cached, fresh=self.fresh, table=self.table, table_width=self.width, free_pages=self.stack,
                                  pages=self.stack.numel(), free_count=self.count, free_left=self.left, lengths=self.lengths,
                                  query_begin=self.query_begin, key_begin=self.key_begin, slots=self.slots, positions=self.positions,
                                  shortage=self.shortage, requests=self.n, page_tokens=self.page, token_capacity=self.capacity)

    def check(self, want):
        for name, got in (("table", self.table[:, :self.width]), ("free_pages", self.stack), ("lengths", self.lengths),
                          ("query_begin", self.query_begin), ("key_begin", self.key_begin), ("slots", self.slots), ("positions", self.positions)):
            w = want[name][:, :self.width] if name == "table" else want[name]
            assert np.array_equal(got.cpu().numpy(), np.asarray(w)), name
        assert int(self.left) == want["free_left"] and int(self.shortage) == want["shortage"]


def random_step(rng, s, page, free, cached=None):
    n = s.n
    room = s.width * page
    cached = rng.integers(0, room // 2 + 1, n) if cached is None else cached
    fresh = np.where(rng.random(n) < 0.2, -1, np.where(rng.random(n) < 0.5, 1, rng.integers(0, room // 2 + 1, n)))
    return cached.astype(np.int64), fresh.astype(np.int64)


@pytest.mark.parametrize("n,width,page,free,stride", [
    (1, 1, 16, 1, None), (1, 3, 16, 0, None), (5, 4, 16, 3, None), (16, 40, 16, 1000, None), (33, 9, 32, 40, 11), (255, 6, 16, 100, None),
    (256, 3, 256, 150, None), (257, 12, 64, 500, None), (1000, 30, 16, 9000, None), (1025, 7, 128, 10, 9), (3000, 5, 16, 4000, None), (8192, 2, 16, 100, None),
])
def test_plan_matches_lists(be, n, width, page, free, stride):
    rng = np.random.default_rng(n + free)
    for case in range(3):
        probe = Step(n, width, 1, page, 1)
        cached, fresh = random_step(rng, probe, page, free)
        if case == 1:
            fresh[:] = 1
            cached = np.minimum(cached, width * page - 1)
        if case == 2 and n > 1:
            fresh[: n // 2] = -1
        held = int(sum(-(-c // page) for c in cached))
        pages = held + free + 5
        capacity = max(1, int(np.maximum(fresh, 0).sum()) + (0, 7, 64)[case])
        s = Step(n, width, pages, page, capacity, stride=stride)
        ids = rng.permutation(pages).astype(np.int32)
        table = np.full((n, s.table.shape[1]), -1, np.int32)
        at = 0
        for b in range(n):
            k = -(-int(cached[b]) // page)
            table[b, :k] = ids[at:at + k]
            at += k
        stack = np.full(pages, -77, np.int32)
        stack[:free] = ids[at:at + free]
        s.cached.copy_(dev(cached.tolist()))
        s.fresh.copy_(dev(fresh.tolist()))
        s.table.copy_(torch.from_numpy(table))
        s.stack.copy_(torch.from_numpy(stack))
        s.count.fill_(free)
        torch.cuda.synchronize()
        want = plain.plan(cached, fresh, table, stack, free, page, capacity)
        for _ in range(2):                       # again on the same state: the same
            done(be, be.kv_plan(s.request()))
            s.check(want)


def test_plan_in_place_replayed(be):
    """A captured step, replayed: lengths and the stack's size go on from where the replay before left them."""
    n, page, width, pages, cap = 9, 16, 8, 40, 64
    rng = np.random.default_rng(4)
    s = Step(n, width, pages, page, cap, in_place=True)
    cached, count = np.zeros(n, np.int64), pages
    table, stack = np.full((n, width), -1, np.int32), rng.permutation(pages).astype(np.int32)
    s.cached.zero_()
    s.table.fill_(-1)
    s.stack.copy_(torch.from_numpy(stack))
    s.count.fill_(count)
    torch.cuda.synchronize()
    assert be.graph_begin()
    assert be.kv_plan(s.request())
    graph = be.graph_end()
    for step in range(12):
        fresh = np.where((step > 3) & (rng.random(n) < 0.15), -1, np.minimum(rng.integers(0, 8, n), width * page - cached))
        s.fresh.copy_(dev(fresh.tolist()))
        torch.cuda.synchronize()
        assert be.graph_launch(graph) and be.sync()
        want = plain.plan(cached, fresh, table, stack, count, page, cap)
        s.check(want)
        cached, count, table, stack = np.asarray(want["lengths"]), want["free_left"], want["table"], want["free_pages"]
    be.graph_destroy(graph)


def test_plan_in_place_of_many_rows(be):
    """Steps in place that several CTAs make: lengths and the stack's size wait for the last read of the ones before."""
    n, page, width, pages, cap = 700, 16, 30, 12000, 20000
    rng = np.random.default_rng(8)
    for lengths_too in (True, False):
        s = Step(n, width, pages, page, cap, in_place=True)
        if not lengths_too:
            s.lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
        cached, count = np.zeros(n, np.int64), pages
        table, stack = np.full((n, width), -1, np.int32), rng.permutation(pages).astype(np.int32)
        s.cached.zero_()
        s.table.fill_(-1)
        s.stack.copy_(torch.from_numpy(stack))
        s.count.fill_(count)
        for step in range(6):
            fresh = np.where((step > 1) & (rng.random(n) < 0.2), -1, np.minimum(rng.integers(0, 56, n), width * page - cached))
            s.fresh.copy_(dev(fresh.tolist()))
            if not lengths_too:
                s.cached.copy_(dev(cached.tolist()))
            torch.cuda.synchronize()
            done(be, be.kv_plan(s.request()))
            want = plain.plan(cached, fresh, table, stack, count, page, cap)
            s.check(want)
            cached, count, table, stack = np.asarray(want["lengths"]), want["free_left"], want["table"], want["free_pages"]


@pytest.mark.parametrize("what", ["negative", "fresh", "long", "capacity", "count", "page"])
def test_plan_reports_values_out_of_range(be, what):
    s = Step(4, 4, 30, 16, 20)
    s.cached.copy_(dev([5, 16, 0, 40]))
    s.fresh.copy_(dev([1, 1, 3, 2]))
    s.table.copy_(torch.arange(16, dtype=torch.int32).view(4, 4))
    s.stack.copy_(torch.arange(30, dtype=torch.int32))
    s.count.fill_(10)
    if what == "negative":
        s.cached[1] = -3
    elif what == "fresh":
        s.fresh[1] = -2
    elif what == "long":
        s.cached[1] = 64
    elif what == "capacity":
        s.fresh[1] = 18
    elif what == "count":
        s.count.fill_(31)
    else:
        s.stack.fill_(30)
    torch.cuda.synchronize()
    assert be.kv_plan(s.request())
    assert not be.sync() and be.last_error == eb.INVALID_REQUEST
    assert be.sync()
    slots = s.slots.cpu().numpy()
    assert slots.max() < 30 * 16
    if what not in ("count", "page"):
        assert slots[0] == 5                                    # the sound request before it has its slot
        assert what == "fresh" or slots[{"capacity": 19}.get(what, 1)] == -1     # rows 0, 1 .. 18, 19 ..: the third is cut off


# ---------------------------------------------------------------- store and load
class Cache:
    def __init__(self, pages, page, heads, dim, fill=0):
        self.data = torch.full((pages * paged.page_bytes(dim, heads, page),), fill, dtype=torch.uint8, device="cuda")
        self.count, self.page, self.heads, self.dim = pages, page, heads, dim
        self.pages = paged.pages(self.data, pages, page, heads, dim)


def tables(rng, lengths, page, spare=4, extra=1):
    counts = [-(-n // page) for n in lengths]
    ids = rng.permutation(sum(counts) + spare).astype(np.int32)
    table = np.full((len(lengths), max(1, max(counts)) + extra), -1, np.int32)
    at = 0
    for b, k in enumerate(counts):
        table[b, :k] = ids[at:at + k]
        at += k
    return table, sum(counts) + spare


def slots_of(table, first, lengths, page):
    return np.concatenate([np.array([int(table[b, p // page]) * page + p % page for p in range(lo, hi)], np.int64)
                           for b, (lo, hi) in enumerate(zip(first, lengths))])


def placed(x, layout, t):
    """The same values in another arrangement of memory."""
    rows, heads, dim = x.shape
    x = x.to(t)
    if layout == "heads":                                      # [heads][rows][dim]
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if layout == "odd":                                        # rows at odd addresses
        buf = torch.zeros(rows * (heads * (dim + 3) + 1) + 1, dtype=t, device="cuda")
        y = buf[1:].as_strided((rows, heads, dim), (heads * (dim + 3) + 1, dim + 3, 1))
        y.copy_(x)
        return y
    if layout == "part":                                       # columns of a wider row
        buf = torch.full((rows, 3 * heads, dim), -5.0, dtype=t, device="cuda")
        y = buf[:, heads:2 * heads]
        y.copy_(x)
        return y
    return x.contiguous()


@pytest.mark.parametrize("dim,heads,page,t,layout", [
    (32, 1, 16, "f32", "dense"), (32, 3, 32, "bf16", "odd"), (64, 4, 16, "f16", "dense"), (64, 2, 64, "f32", "heads"), (96, 2, 16, "bf16", "dense"),
    (96, 5, 128, "f32", "odd"), (128, 8, 16, "bf16", "dense"), (128, 2, 256, "f16", "part"), (128, 1, 16, "f32", "part"), (64, 8, 16, "bf16", "heads"),
])
def test_store_and_load(be, dim, heads, page, t, layout):
    rng = np.random.default_rng(dim + heads)
    first = [0, 5, 16, 31, 0, 100, 7]
    lengths = [1, 6, 49, 33, 17, 100, 160]
    table, pages = tables(rng, lengths, page)
    slots = slots_of(table, first, lengths, page)
    slots = np.concatenate([slots[:40], [-1], slots[40:], [-1, -9]])
    g = gen(dim * heads)
    x = [torch.randn((len(slots), heads, dim), generator=g, device="cuda") * torch.exp(2 * torch.randn((len(slots), heads, 1), generator=g, device="cuda"))
         for _ in range(2)]
    k, v = (placed(y, layout, plain.TORCH[t]) for y in x)
    c = Cache(pages, page, heads, dim)
    torch.cuda.synchronize()
    done(be, be.kv_store(paged.store_request(c.pages, k, v, t, dev(slots.tolist(), torch.int64), len(slots))))
    live = torch.from_numpy(slots >= 0).cuda()
    begin = np.concatenate([[0], np.cumsum([b - a for a, b in zip(first, lengths)])])
    rows = int(begin[-1])
    for out_t in ("f32", "bf16", "f16"):
        for out_layout in ("dense", layout):
            got = [placed(torch.full((rows + 3, heads, dim), 7.0, device="cuda"), out_layout, plain.TORCH[out_t]) for _ in range(2)]
            torch.cuda.synchronize()
            keep = [dev(first), dev(lengths), dev(begin.tolist()), torch.from_numpy(table).cuda()]
            torch.cuda.synchronize()
            done(be, be.kv_load(paged.load_request(c.pages, *got, out_t, keep[3], table.shape[1], keep[1], keep[2], len(lengths), rows + 3, first=keep[0])))
            for y, z in zip((k, v), got):
                want = plain.kept(y)[live].to(plain.TORCH[out_t])
                assert torch.equal(z[:rows], want)
                assert (z[rows:] == 7.0).all()                # behind the last request: as it was
    # without `first`: from the request's beginning; rows that no length reaches stay
    got = [torch.full((20, heads, dim), 7.0, device="cuda") for _ in range(2)]
    two, b2, t2 = dev([1]), dev([3, 20]), torch.from_numpy(table).cuda()
    torch.cuda.synchronize()
    done(be, be.kv_load(paged.load_request(c.pages, *got, "f32", t2, table.shape[1], two, b2, 1, 20)))
    assert torch.equal(got[0][3], plain.kept(k)[0].float()) and (got[0][:3] == 7.0).all() and (got[0][4:] == 7.0).all()


@pytest.mark.parametrize("n,with_first,short", [(1500, True, 0), (1500, False, 0), (40, True, 100), (33, False, 7), (1, True, 0)])
def test_load_many_requests(be, n, with_first, short):
    """Requests of every length from none up, behind rows of no request, into fewer rows than they have (`short`)."""
    rng, g = np.random.default_rng(n + short), gen(n)
    lengths = rng.integers(0, 50, n)
    lengths[0] = 21
    first = np.minimum(rng.integers(0, 40, n), lengths) if with_first else np.zeros(n, np.int64)
    c, table, k, v = filled(be, rng, g, lengths.tolist(), 16, 2, 64)
    begin = 5 + np.concatenate([[0], np.cumsum(lengths - first)])
    rows = int(begin[-1]) - short
    got = [torch.full((int(begin[-1]) + 2, 2, 64), 7.0, device="cuda") for _ in range(2)]
    keep = [dev(lengths.tolist()), dev(begin.tolist()), dev(first.tolist()) if with_first else None]
    torch.cuda.synchronize()
    done(be, be.kv_load(paged.load_request(c.pages, *got, "f32", table, table.shape[1], keep[0], keep[1], n, rows, first=keep[2])))
    at = np.concatenate([[0], np.cumsum(lengths)])
    pick = dev(np.concatenate([np.arange(at[b] + first[b], at[b + 1]) for b in range(n)]).tolist(), torch.int64)
    for y, z in zip((k, v), got):
        want = y[pick].reshape(-1, 2, 64).float()
        assert torch.equal(z[5:rows], want[:rows - 5]) and (z[:5] == 7.0).all() and (z[rows:] == 7.0).all()


@pytest.mark.parametrize("heads,dim,lengths,layout", [(8, 32, [9000, 3001, 7], "dense"), (7, 64, [6000, 5, 8000], "part"), (3, 96, [26000], "heads")])
def test_store_and_load_many_rows(be, heads, dim, lengths, layout):
    """So many rows that a CTA takes several heads, and not all CTAs the same number."""
    rng, g = np.random.default_rng(heads), gen(heads)
    table, pages = tables(rng, lengths, 32)
    slots = slots_of(table, [0] * len(lengths), lengths, 32)
    n = len(slots)
    slots[5], slots[n - 3] = -1, -4
    k, v = (placed(torch.randn((n, heads, dim), generator=g, device="cuda"), layout, torch.bfloat16) for _ in range(2))
    c = Cache(pages, 32, heads, dim)
    got = [torch.full((n, heads, dim), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    keep = [dev(slots.tolist(), torch.int64), torch.from_numpy(table).cuda(), dev(lengths), dev(np.concatenate([[0], np.cumsum(lengths)]).tolist())]
    torch.cuda.synchronize()
    done(be, be.kv_store(paged.store_request(c.pages, k, v, "bf16", keep[0], n)))
    done(be, be.kv_load(paged.load_request(c.pages, *got, "f16", keep[1], table.shape[1], keep[2], keep[3], len(lengths), n)))
    live = keep[0] >= 0
    for y, z in zip((k, v), got):
        assert torch.equal(z[live], plain.kept(y)[live].half())


def test_load_reports_beginnings_out_of_order(be):
    c = Cache(8, 16, 2, 64)
    table, lengths = dev([[0], [1], [2]]), dev([10, 10, 10])
    for begin in ([0, 20, 10, 30], [-5, 5, 10, 20], [0, 10, 20, 15]):
        out = [torch.full((40, 2, 64), 7.0, device="cuda") for _ in range(2)]
        begins = dev(begin)
        torch.cuda.synchronize()
        assert be.kv_load(paged.load_request(c.pages, *out, "f32", table, 1, lengths, begins, 3, 30))
        assert not be.sync() and be.last_error == eb.INVALID_REQUEST
        assert be.sync() and (out[0][30:] == 7.0).all() and (out[1][30:] == 7.0).all()


def test_store_of_special_values(be):
    """Ties, borders, both signs at the largest magnitude, zeros, tiny and huge values, infinities, NaN."""
    g = gen(3)
    rows = []
    for d in (1.0, -1.0, 0.3330078125, 2.0 ** -20, 2.0 ** -24, 1000.0, -65504.0):
        steps = torch.arange(-8, 8, device="cuda").float().repeat(2)
        rows += [steps * d, (steps + 0.5).clamp(-8, 7.5) * d, torch.cat([steps[:1] * d, torch.nextafter((steps[1:] + 0.5).clamp(-7.5, 7.5) * d, torch.zeros(31, device="cuda"))])]
    z = torch.zeros(32, device="cuda")
    rows += [z, -z, z + 1e-30, z + 3e-8, z + 1e30, z - 3e38]
    pair = z.clone()
    pair[3], pair[20] = 2.0, -2.0
    rows += [pair, -pair]
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = torch.randn(32, generator=g, device="cuda")
        y[11] = bad
        rows.append(y)
    rows.append(z + float("nan"))
    x = torch.stack(rows).view(-1, 1, 32).contiguous()
    n = x.shape[0]
    for t in ("f32", "f16", "bf16"):
        k = x.to(plain.TORCH[t])
        v = k.flip(0).contiguous()
        c = Cache(4, 16, 1, 32)
        slots, table, got = dev(range(n), torch.int64), dev([[0, 1, 2, 3]]), [torch.zeros(n, 1, 32, device="cuda") for _ in range(2)]
        lens, begin = dev([n]), dev([0, n])
        torch.cuda.synchronize()
        done(be, be.kv_store(paged.store_request(c.pages, k, v, t, slots, n)))
        done(be, be.kv_load(paged.load_request(c.pages, *got, "f32", table, 4, lens, begin, 1, n)))
        for y, z2 in zip((k, v), got):
            assert torch.equal(z2, plain.kept(y).float())
            assert torch.isfinite(z2).all()


def test_store_and_load_report_values_out_of_range(be):
    c = Cache(3, 16, 2, 64)
    before = c.data.clone()
    x = torch.ones(4, 2, 64, device="cuda")
    slots = dev([48, 1 << 40, -1, 1000], torch.int64)
    torch.cuda.synchronize()
    assert be.kv_store(paged.store_request(c.pages, x, x.clone(), "f32", slots, 4))
    assert not be.sync() and be.last_error == eb.INVALID_REQUEST
    assert be.sync() and torch.equal(c.data, before)
    for table, length, begin, first in (([[3]], 16, [0, 4], None), ([[-1]], 16, [0, 4], None), ([[0]], 40, [0, 40], None), ([[0]], 16, [0, 4], [-2])):
        rows = max(begin)
        out = [torch.full((rows, 2, 64), 7.0, device="cuda") for _ in range(2)]
        keep = [dev(table), dev([length]), dev(begin), dev(first) if first else None]
        torch.cuda.synchronize()
        assert be.kv_load(paged.load_request(c.pages, *out, "f32", keep[0], 1, keep[1], keep[2], 1, rows, first=keep[3]))
        assert not be.sync() and be.last_error == eb.INVALID_REQUEST
        assert (out[0][16:] == 7.0).all()
        assert be.sync()


def test_host_memory_is_refused(be):
    x = np.zeros((4, 2, 64), np.float32)
    c = Cache(3, 16, 2, 64)
    slots = dev([0, 1, 2, 3], torch.int64)
    torch.cuda.synchronize()
    assert not be.kv_store(paged.store_request(c.pages, x, x.copy(), "f32", slots, 4, k_strides=(128, 64), v_strides=(128, 64)))
    assert be.last_error == eb.INVALID_REQUEST
    y = torch.zeros(4, 2, 64, device="cuda")
    host_slots = np.arange(4)
    assert not be.kv_store(paged.store_request(c.pages, y, y.clone(), "f32", host_slots, 4))
    assert be.sync()


# ---------------------------------------------------------------- attention over the pages
def filled(be, rng, g, lengths, page, heads, dim, gain=(1.0, 1.0), extra=1):
    """A cache whose unwritten bytes make infinite and NaN scales, with requests of these lengths; (cache, table, kept k, kept v)."""
    table, pages = tables(rng, lengths, page, extra=extra)
    c = Cache(pages, page, heads, dim, fill=0xff)
    total = max(1, sum(lengths))
    k = torch.randn((total, heads, dim), generator=g, device="cuda") * gain[0]
    v = torch.randn((total, heads, dim), generator=g, device="cuda") * gain[1]
    if sum(lengths):
        slots = dev(slots_of(table, [0] * len(lengths), lengths, page).tolist(), torch.int64)
        torch.cuda.synchronize()
        done(be, be.kv_store(paged.store_request(c.pages, k, v, "f32", slots, total)))
    return c, torch.from_numpy(table).cuda(), plain.kept(k), plain.kept(v)


def attend_bound(q, k, v, out, size, total, t, scale):
    """How far a result may be off, from the roundings that are made.  Weights times value scales: two roundings to f16 each (f32:
    one of the 22 bits of two f16 operands); scores: an f32 sum of 32 products (base + q) |query| less (base + 8) times the queries, which
    is kept to 22 bits, times a scale; bases 1024, 64, 256 and 16 in turn for pairs of dims, with f32 queries all 64; f32 accumulation over
    the tokens; ex2 to 2^-22; products below f16's normal range; the result's own rounding."""
    length = k.shape[0]
    if length == 0 or q.shape[0] == 0:
        return torch.zeros_like(out)
    heads, kv = q.shape[1], k.shape[1]
    group = heads // kv
    top = k.abs().view(length, kv, -1, 32).amax((0, 3)).repeat_interleave(group, 0) / 7      # at least the scale
    base = torch.tensor([64.0] * 8 if t == "f32" else [1024.0] * 2 + [64.0] * 2 + [256.0] * 2 + [16.0] * 2, dtype=torch.float64, device=q.device).repeat(4)
    off = 34 * 2.0 ** -23 * (2 * base + 23) + 2.0 ** -22 * (base + 8)
    score = scale * ((q.abs().view(*q.shape[:2], -1, 32) * off).sum(-1) * top).sum(-1, keepdim=True)
    rel = (2.0 ** -20 if t == "f32" else 2.0 ** -10) + 2 * score + (length / 16 + 20) * 2.0 ** -23 + 2.0 ** -21
    tiny = length * 2.0 ** -22 * v.abs().max() / total
    return rel * size + tiny + plain.HALF_STEP[t] * out.abs() + 1e-30


def check_attend(be, lengths, rows, heads, kv, dim, page, t, seed, gain=(1.0, 1.0), layout="dense", begin=True, before=0, after=0, q_gain=1.0):
    """Requests with `rows` query rows each; q_gain: a number, or one for each head."""
    rng, g = np.random.default_rng(seed), gen(seed)
    c, table, k, v = filled(be, rng, g, lengths, page, kv, dim, gain)
    total = before + sum(rows) + after
    q_gain = torch.as_tensor(q_gain, device="cuda").reshape(1, -1, 1)
    q = placed(torch.randn((max(total, 1), heads, dim), generator=g, device="cuda") * 1.5 * q_gain, layout, plain.TORCH[t])
    out = placed(torch.full((max(total, 1), heads, dim), 7.0, device="cuda"), layout, plain.TORCH[t])
    qb = np.concatenate([[before], before + np.cumsum(rows)])
    keep = [dev(lengths), dev(qb.tolist())]
    scale = dim ** -0.5
    req = paged.attend_request(c.pages, q, out, t, table, table.shape[1], keep[0], len(lengths), heads, q.shape[0],
                               query_begin=keep[1] if begin else None, max_queries=max(max(rows), 1), scale=scale)
    torch.cuda.synchronize()
    done(be, be.kv_attend(req))
    got = out.double()
    first = out.clone()
    at = 0
    for b, (length, n) in enumerate(zip(lengths, rows)):
        qr = q[qb[b]:qb[b + 1]].double()
        want, size, tot = plain.attention(qr, k[at:at + length], v[at:at + length], scale)
        bound = attend_bound(qr, k[at:at + length], v[at:at + length], want, size, tot, t, scale)
        err = (got[qb[b]:qb[b + 1]] - want).abs()
        assert torch.isfinite(err).all() and (err <= bound).all(), (b, length, n, float((err / bound).max()) if n else 0)
        at += length
    assert (got[:before] == 7.0).all() and (got[qb[-1]:] == 7.0).all()
    done(be, be.kv_attend(req))
    assert torch.equal(first, out)                              # the same bits again
    return req


@pytest.mark.parametrize("heads,kv,dim,page,t", [
    (8, 8, 64, 16, "f16"), (8, 2, 64, 16, "bf16"), (32, 8, 128, 16, "bf16"), (32, 4, 64, 32, "f16"), (10, 2, 96, 64, "f16"), (7, 1, 32, 16, "bf16"),
    (64, 8, 128, 128, "f16"), (16, 1, 128, 16, "bf16"), (33, 3, 32, 256, "f16"), (64, 1, 96, 16, "bf16"), (8, 2, 128, 16, "f32"), (24, 1, 64, 16, "f32"),
    (3, 3, 96, 16, "f32"), (16, 2, 32, 16, "f32"),
])
def test_attend_one_token(be, heads, kv, dim, page, t):
    lengths = [1, 2, 15, 16, 17, 31, 33, 100, 0, 64, 257, 600]
    check_attend(be, lengths, [1] * len(lengths), heads, kv, dim, page, t, heads + dim, begin=False, after=2)


@pytest.mark.parametrize("heads,kv,dim,t", [(8, 2, 64, "bf16"), (32, 8, 128, "f16"), (5, 1, 96, "f16"), (16, 1, 128, "bf16"), (4, 4, 32, "f32"), (8, 1, 128, "f32")])
def test_attend_several_tokens(be, heads, kv, dim, t):
    """Ragged rows: none, one, some; more rows than tokens leaves rows that see nothing."""
    check_attend(be, [5, 40, 0, 33, 200, 2, 1, 17], [1, 4, 3, 0, 8, 5, 0, 17], heads, kv, dim, 16, t, heads + dim, before=3, after=2)


@pytest.mark.parametrize("lengths,heads,kv,dim,t", [
    ([20001], 32, 8, 128, "f16"), ([70000], 8, 1, 64, "bf16"), ([30000, 3, 500, 9000], 16, 4, 128, "bf16"), ([12000, 12000], 4, 2, 96, "f16"),
    ([9000], 8, 1, 128, "f32"),
])
def test_attend_long(be, lengths, heads, kv, dim, t):
    check_attend(be, lengths, [1] * len(lengths), heads, kv, dim, 64, t, len(lengths))
    check_attend(be, lengths, [3] * len(lengths), heads, kv, dim, 16, t, len(lengths) + 9)


@pytest.mark.parametrize("n,lo,hi,heads,kv,dim", [(64, 1, 300, 32, 8, 128), (300, 1, 40, 8, 2, 64), (600, 1, 20, 4, 1, 32), (1000, 5, 6, 16, 2, 64)])
def test_attend_many_requests(be, n, lo, hi, heads, kv, dim):
    lengths = np.random.default_rng(n).integers(lo, hi, n).tolist()
    check_attend(be, lengths, [1] * n, heads, kv, dim, 16, "bf16", n, begin=False)


@pytest.mark.parametrize("gain", [(1.0, 1e-5), (1.0, 3e4), (30.0, 1.0), (1e-4, 1.0)])
@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_attend_magnitudes(be, gain, t):
    check_attend(be, [700, 31], [1, 1], 8, 2, 128, 16, t, 5, gain=gain)


@pytest.mark.parametrize("t,q_gain,k_gain", [
    ("bf16", 1e6, 2e-6), ("f32", 1e6, 2e-6), ("bf16", 1e-6, 1e5), ("f32", 1e-6, 1e5), ("f16", 5e3, 2e-4), ("f16", 1e-4, 1e4),
    ("bf16", [1e5, 1e3, 1e4, 1e2, 1e3, 1e3, 1e5, 1e2], 1e-3), ("f32", [1e-5, 1e-3, 1e-4, 1e-2, 1e-3, 1e-3, 1e-5, 1e-2], 1.0),
])
def test_attend_query_magnitudes(be, t, q_gain, k_gain):
    """Queries far outside of f16's range."""
    check_attend(be, [700, 31, 64], [1, 3, 1], 8, 2, 64, 16, t, 6, gain=(k_gain, 1.0), q_gain=q_gain)


@pytest.mark.parametrize("layout", ["heads", "part", "odd"])
@pytest.mark.parametrize("t", ["f16", "f32"])
def test_attend_layouts(be, layout, t):
    check_attend(be, [50, 3, 18], [2, 1, 3], 8, 2, 64, 16, t, 8, layout=layout)


def test_attend_captured_and_replayed(be):
    """A captured call reads lengths, tables and queries anew at each replay."""
    rng, g = np.random.default_rng(2), gen(2)
    lengths = [900, 40, 333]
    c, table, k, v = filled(be, rng, g, lengths, 16, 2, 64)
    q, out, lens = torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda"), torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda"), dev(lengths)
    req = paged.attend_request(c.pages, q, out, "f16", table, table.shape[1], lens, 3, 8, 3)
    torch.cuda.synchronize()
    assert be.graph_begin() and be.kv_attend(req)
    graph = be.graph_end()
    for now in ([900, 40, 333], [1, 0, 17], [450, 39, 2], [899, 1, 320]):
        q.copy_(torch.randn(3, 8, 64, generator=g, device="cuda"))
        lens.copy_(dev(now))
        torch.cuda.synchronize()
        assert be.graph_launch(graph) and be.sync()
        for b, length in enumerate(now):
            at = sum(lengths[:b])
            want, size, tot = plain.attention(q[b:b + 1], k[at:at + length], v[at:at + length], 0.125)
            bound = attend_bound(q[b:b + 1].double(), k[at:at + length], v[at:at + length], want, size, tot, "f16", 0.125)
            assert ((out[b:b + 1].double() - want).abs() <= bound).all()
    be.graph_destroy(graph)


def test_attend_reports_values_out_of_range(be):
    rng, g = np.random.default_rng(6), gen(6)
    c, table, k, v = filled(be, rng, g, [40, 40, 40], 16, 2, 64)
    good = table.clone()
    q = torch.randn(6, 4, 64, generator=g, device="cuda").half()

    def run(lengths, begin, table, most=2):
        out = torch.full_like(q, 7.0)
        keep = [dev(lengths), dev(begin)]
        torch.cuda.synchronize()
        assert be.kv_attend(paged.attend_request(c.pages, q, out, "f16", table, table.shape[1], keep[0], 3, 4, 6, query_begin=keep[1], max_queries=most))
        ok = be.sync()
        assert ok or be.last_error == eb.INVALID_REQUEST
        assert be.sync()
        return ok, out

    ok, sound = run([40, 40, 40], [0, 2, 4, 6], good)
    assert ok
    for lengths, begin, change in (([40, -1, 40], [0, 2, 4, 6], None), ([40, 1 << 30, 40], [0, 2, 4, 6], None), ([40, 40, 40], [0, 2, 4, 6], c.count),
                                   ([40, 40, 40], [0, 2, 4, 6], -1), ([40, 40, 40], [0, 2, 5, 6], None), ([40, 40, 40], [0, 2, 1, 6], None),
                                   ([40, 40, 40], [0, 2, 1 << 30, 6], None)):
        bad = good.clone()
        if change is not None:
            bad[1, 1] = change
        ok, out = run(lengths, begin, bad)
        assert not ok
        assert torch.equal(out[:2], sound[:2])                  # the request before it is whole
    ok, out = run([40, 40, 40], [0, 2, 4, 6], good, most=1)
    assert not ok and (out == 7.0).all()


# ---------------------------------------------------------------- packed prompts
def packed_bound(q, k, v, out, size, t, scale):
    """Weights rounded to the type; scores an f32 sum of dim products; f32 accumulation over the keys; ex2; the result's rounding."""
    length, dim = k.shape[0], q.shape[2]
    if length == 0 or q.shape[0] == 0:
        return torch.zeros_like(out)
    group = q.shape[1] // k.shape[1]
    score = scale * torch.einsum("nhd,hd->nh", q.double().abs(), k.double().abs().amax(0).repeat_interleave(group, 0)).unsqueeze(-1) * (dim + 2) * 2.0 ** -23
    rel = plain.HALF_STEP[t] + 2 * score + (length / 16 + 20) * 2.0 ** -23 + 2.0 ** -20
    return rel * size + plain.HALF_STEP[t] * out.abs() + 1e-6 * size.max() * (t == "f16") + 1e-30


def check_packed(be, queries, keys, heads, kv, dim, t, seed, causal=True, layout="dense", gap=0, gain=1.0):
    """`gap` rows of NaN behind each request's keys, rows of no request before and behind the queries."""
    g = gen(seed)
    T = plain.TORCH[t]
    qb = np.concatenate([[2], 2 + np.cumsum(queries)])
    kb = np.concatenate([[0], np.cumsum(keys)])
    q = placed(torch.randn((int(qb[-1]) + 3, heads, dim), generator=g, device="cuda") * 1.5 * gain, layout, T)
    k, v = (placed(torch.randn((int(kb[-1]) + gap, kv, dim), generator=g, device="cuda"), layout, T) for _ in range(2))
    if gap:
        k[int(kb[-1]):], v[int(kb[-1]):] = float("nan"), float("inf")
    out = placed(torch.full((q.shape[0], heads, dim), 7.0, device="cuda"), layout, T)
    keep = [dev(qb.tolist()), dev(kb.tolist())]
    scale = dim ** -0.5
    req = paged.packed_request(q, k, v, out, t, keep[0], keep[1], len(queries), heads, kv, dim, q.shape[0], int(kb[-1]), causal=causal, scale=scale,
                               max_queries=max(max(queries), 1))
    torch.cuda.synchronize()
    done(be, be.attend_packed(req))
    got = out.double()
    first = out.clone()
    for b, (n, length) in enumerate(zip(queries, keys)):
        qr, kr, vr = q[qb[b]:qb[b + 1]], k[kb[b]:kb[b + 1]], v[kb[b]:kb[b + 1]]
        want, size, _ = plain.attention(qr, kr, vr, scale, causal)
        bound = packed_bound(qr, kr, vr, want, size, t, scale)
        err = (got[qb[b]:qb[b + 1]] - want).abs()
        assert torch.isfinite(err).all() and (err <= bound).all(), (b, n, length, float((err / bound).max()) if n else 0)
    assert (got[:2] == 7.0).all() and (got[qb[-1]:] == 7.0).all()
    done(be, be.attend_packed(req))
    assert torch.equal(first, out)


@pytest.mark.parametrize("heads,kv,dim,t", [
    (8, 8, 64, "f16"), (8, 2, 64, "bf16"), (32, 8, 128, "bf16"), (16, 4, 128, "f16"), (10, 2, 96, "f16"), (7, 1, 32, "bf16"), (3, 3, 8, "f16"),
    (12, 4, 72, "bf16"), (128, 1, 64, "f16"), (5, 1, 120, "bf16"), (6, 2, 16, "f16"), (64, 8, 128, "bf16"),
])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(be, heads, kv, dim, t, causal):
    check_packed(be, [1, 2, 15, 64, 65, 0, 130, 33], [1, 2, 15, 64, 65, 7, 130, 33], heads, kv, dim, t, heads + dim, causal, gap=3)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (4, 4, 128), (6, 1, 40)])
def test_packed_behind_earlier_tokens(be, heads, kv, dim, causal):
    """Fewer queries than keys, and more: rows that see nothing; requests without keys or queries."""
    check_packed(be, [1, 40, 129, 10, 5, 0, 256, 3], [300, 41, 500, 4, 0, 50, 257, 1], heads, kv, dim, "bf16", heads + dim, causal, gap=2)


@pytest.mark.parametrize("queries,heads,kv,dim,t", [([1000], 8, 2, 128, "bf16"), ([2049, 700], 4, 1, 64, "f16"), ([1537], 3, 3, 128, "f16"),
                                                    ([513, 1, 2, 1024], 8, 8, 96, "bf16")])
def test_packed_long(be, queries, heads, kv, dim, t):
    check_packed(be, queries, [n + 100 for n in queries], heads, kv, dim, t, len(queries), gap=5)


@pytest.mark.parametrize("layout", ["heads", "part"])
def test_packed_layouts(be, layout):
    check_packed(be, [50, 3, 200], [60, 3, 200], 8, 2, 64, "bf16", 8, layout=layout)


def test_packed_large_scores(be):
    """Scores far apart: the running maximum moves, weights vanish."""
    check_packed(be, [300], [300], 4, 2, 64, "f16", 3, gain=40.0)


def test_packed_many_requests(be):
    lengths = np.random.default_rng(1).integers(0, 40, 500).tolist()
    check_packed(be, lengths, lengths, 4, 2, 64, "bf16", 9)


@pytest.mark.parametrize("heads,kv,dim,t", [(8, 2, 128, "bf16"), (3, 3, 64, "f16"), (16, 1, 40, "f16")])
def test_packed_hidden_values_have_no_influence(be, heads, kv, dim, t):
    """Keys and values that are not finite reach the rows that see them, in their heads and dims, and no other."""
    lengths, g = [400, 70, 1], gen(heads)
    n, dt = sum(lengths), plain.TORCH[t]
    q = torch.randn(n, heads, dim, generator=g, device="cuda").to(dt)
    k, v = (torch.randn(n, kv, dim, generator=g, device="cuda").to(dt) for _ in range(2))
    begin = dev([0, 400, 470, 471])

    def run():
        out = torch.full_like(q, 7.0)
        torch.cuda.synchronize()
        assert be.attend_packed(paged.packed_request(q, k, v, out, t, begin, begin, 3, heads, kv, dim, n, n, max_queries=400))
        assert be.sync()
        return out

    clean, inf, group, last = run(), float("inf"), heads // kv, kv - 1
    v[150, last, 5], v[320, 0, dim - 1] = float("nan"), -inf
    v[440, 0, 33], v[460, 0, 33], v[469, last, 0] = inf, -inf, float("nan")
    k[468, 0, 2] = float("nan")
    want = clean.clone()
    want[150:400, last * group:, 5] = float("nan")
    want[320:400, :group, dim - 1] = -inf
    want[440:470, :group, 33] = inf
    want[460:470, :group, 33] = float("nan")
    want[469, last * group:, 0] = float("nan")
    want[468:470, :group] = float("nan")
    got = run()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=3.0), want.nan_to_num(nan=3.0))


def test_packed_reports_values_out_of_range(be):
    g = gen(7)
    q, k, v = (torch.randn(60, 4, 64, generator=g, device="cuda").half() for _ in range(3))

    def run(begin, key_begin, most=30):
        out = torch.full_like(q, 7.0)
        keep = [dev(begin), dev(key_begin)]
        torch.cuda.synchronize()
        assert be.attend_packed(paged.packed_request(q, k, v, out, "f16", keep[0], keep[1], 3, 4, 4, 64, 60, 60, max_queries=most))
        ok = be.sync()
        assert ok or be.last_error == eb.INVALID_REQUEST
        assert be.sync()
        return ok, out

    ok, sound = run([0, 20, 40, 60], [0, 20, 40, 60])
    assert ok
    for begin, key_begin in (([0, 20, 40, 60], [0, 20, 61, 60]), ([0, 20, 40, 60], [0, 20, 10, 60]), ([0, 20, 40, 61], [0, 20, 40, 60]),
                             ([0, 20, 55, 60], [0, 20, 40, 60])):
        ok, out = run(begin, key_begin)
        assert not ok and torch.equal(out[:20], sound[:20])


# ---------------------------------------------------------------- together
def test_serving_steps(be):
    """Prompts, then tokens one by one: plan, store, attend; the prompts' attention over what the cache keeps equals the packed one
    over what it loads."""
    g = gen(11)
    heads, kv, dim, page, n, width, pages, cap = 8, 2, 64, 16, 5, 12, 50, 160
    s = Step(n, width, pages, page, cap, in_place=True)
    s.cached.zero_()
    s.table.fill_(-1)
    s.stack.copy_(torch.arange(pages, dtype=torch.int32))
    s.count.fill_(pages)
    c = Cache(pages, page, kv, dim, fill=0xff)
    keys, values = [torch.zeros(0, kv, dim, device="cuda") for _ in range(n)], [torch.zeros(0, kv, dim, device="cuda") for _ in range(n)]
    lengths = [0] * n
    for step in range(8):
        fresh = [30, 17, 64, 1, 40] if step == 0 else [1, 1, -1 if step == 3 else 1, 2 if step % 2 else 1, 1]
        s.fresh.copy_(dev(fresh))
        rows = [max(f, 0) for f in fresh]
        total = sum(rows)
        k, v = (torch.randn(cap, kv, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
        q = torch.randn(cap, heads, dim, generator=g, device="cuda").bfloat16()
        out = torch.full_like(q, 7.0)
        torch.cuda.synchronize()
        assert be.kv_plan(s.request())
        assert be.kv_store(paged.store_request(c.pages, k, v, "bf16", s.slots, cap))
        assert be.kv_attend(paged.attend_request(c.pages, q, out, "bf16", s.table, width, s.lengths, n, heads, cap, query_begin=s.query_begin, max_queries=64))
        assert be.sync(), be.last_error
        at = 0
        for b, f in enumerate(fresh):
            if f < 0:
                keys[b], values[b] = keys[b][:0], values[b][:0]
                continue
            keys[b], values[b] = (torch.cat([x[b], y[at:at + f].float()]) for x, y in ((keys, k), (values, v)))
            kk, vv = plain.kept(keys[b]), plain.kept(values[b])
            qr = q[at:at + f].double()
            want, size, tot = plain.attention(qr, kk, vv, dim ** -0.5)
            bound = attend_bound(qr, kk, vv, want, size, tot, "bf16", dim ** -0.5)
            assert ((out[at:at + f].double() - want).abs() <= bound).all()
            at += f
        assert (out[total:] == 7.0).all()
        lengths = [x.shape[0] for x in keys]
        assert s.lengths.cpu().tolist() == lengths
        # the same rows over keys and values loaded back
        all_keys = sum(lengths)
        lk, lv = (torch.zeros(all_keys, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        out2 = torch.full_like(q, 7.0)
        torch.cuda.synchronize()
        assert be.kv_load(paged.load_request(c.pages, lk, lv, "bf16", s.table, width, s.lengths, s.key_begin, n, all_keys))
        assert be.attend_packed(paged.packed_request(q, lk, lv, out2, "bf16", s.query_begin, s.key_begin, n, heads, kv, dim, cap, all_keys))
        assert be.sync(), be.last_error
        qa = 0
        for b, (f, ka) in enumerate(zip(rows, np.concatenate([[0], np.cumsum(lengths)]))):
            kk, vv = lk[ka:ka + lengths[b]], lv[ka:ka + lengths[b]]
            want, size, _ = plain.attention(q[qa:qa + f], kk, vv, dim ** -0.5)
            bound = packed_bound(q[qa:qa + f], kk, vv, want, size, "bf16", dim ** -0.5)
            assert ((out2[qa:qa + f].double() - want).abs() <= bound).all()
            qa += f


def test_step_captured_and_replayed(be):
    """A whole step as one graph (plan in place, store, attention over the pages, rows back, packed attention), replayed with other
    lengths and rows; beside it the same calls without a graph, on another context."""
    g = gen(12)
    heads, kv, dim, page, n, width, pages, cap, most = 8, 2, 64, 16, 3, 12, 40, 96, 400
    other = eb.Backend(0)

    def side(b):
        s = Step(n, width, pages, page, cap, in_place=True)
        s.cached.zero_()
        s.table.fill_(-1)
        s.stack.copy_(torch.arange(pages, dtype=torch.int32))
        s.count.fill_(pages)
        c = Cache(pages, page, kv, dim)
        x = dict(s=s, c=c, b=b, lk=torch.zeros(most, kv, dim, dtype=torch.float16, device="cuda"), lv=torch.zeros(most, kv, dim, dtype=torch.float16, device="cuda"))
        x.update(k=torch.zeros(cap, kv, dim, dtype=torch.float16, device="cuda"), v=torch.zeros(cap, kv, dim, dtype=torch.float16, device="cuda"))
        x.update({name: torch.zeros(cap, heads, dim, dtype=torch.float16, device="cuda") for name in ("q", "out", "out2")})
        x["calls"] = [
            (b.kv_plan, s.request()), (b.kv_store, paged.store_request(c.pages, x["k"], x["v"], "f16", s.slots, cap)),
            (b.kv_attend, paged.attend_request(c.pages, x["q"], x["out"], "f16", s.table, width, s.lengths, n, heads, cap, query_begin=s.query_begin, max_queries=64)),
            (b.kv_load, paged.load_request(c.pages, x["lk"], x["lv"], "f16", s.table, width, s.lengths, s.key_begin, n, most)),
            (b.attend_packed, paged.packed_request(x["q"], x["lk"], x["lv"], x["out2"], "f16", s.query_begin, s.key_begin, n, heads, kv, dim, cap, most)),
        ]
        return x

    left, right = side(be), side(other)
    torch.cuda.synchronize()
    assert be.graph_begin()
    for call, request in left["calls"]:
        assert call(request)
    graph = be.graph_end()
    for fresh in ([33, 5, 0], [1, 60, 30], [1, 1, 1], [-1, 2, 3], [7, 1, -1], [64, 0, 17]):
        for name in ("k", "v", "q"):
            left[name].copy_(torch.randn(left[name].shape, generator=g, device="cuda"))
            right[name].copy_(left[name])
        for x in (left, right):
            x["s"].fresh.copy_(dev(fresh))
        torch.cuda.synchronize()
        assert be.graph_launch(graph)
        for call, request in right["calls"]:                    # at the same time, on a stream of its own
            assert call(request)
        assert be.sync() and other.sync()
        for name in ("out", "out2", "lk", "lv"):
            assert torch.equal(left[name], right[name])
        assert torch.equal(left["s"].table, right["s"].table) and torch.equal(left["c"].data, right["c"].data)
        rows = sum(max(f, 0) for f in fresh)
        # keys and values are rounded once more for the one (scores off by this), weights and results to f16 for both
        score = dim ** -0.5 * 2.0 ** -11 * left["q"].float().abs().sum(-1).max() * left["lk"].float().abs().max()
        assert (left["out"][:rows].float() - left["out2"][:rows].float()).abs().max() < (2 * score + 2.0 ** -8) * left["lv"].float().abs().max()
    be.graph_destroy(graph)
    other.close()


def test_contexts_at_once(be):
    """Calls of two contexts without a wait between them; each result as by itself."""
    g, other = gen(13), eb.Backend(0)
    rng = np.random.default_rng(13)
    c, table, k, v = filled(be, rng, g, [900, 5000, 64, 3], 16, 2, 128)
    lens, begin = dev([900, 5000, 64, 3]), dev([0, 700, 1500, 1501])
    q = torch.randn(4, 16, 128, generator=g, device="cuda").bfloat16()
    pq, pk, pv = (torch.randn(1501, h, 128, generator=g, device="cuda").bfloat16() for h in (8, 2, 2))
    outs = [(torch.zeros_like(q), torch.zeros_like(pq)) for _ in range(5)]
    torch.cuda.synchronize()

    def both(b, out):
        assert b.kv_attend(paged.attend_request(c.pages, q, out[0], "bf16", table, table.shape[1], lens, 4, 16, 4))
        assert b.attend_packed(paged.packed_request(pq, pk, pv, out[1], "bf16", begin, begin, 3, 8, 2, 128, 1501, 1501))

    both(be, outs[0])
    assert be.sync()
    for i in range(20):
        both((be, other)[i % 2], outs[1 + i % 4])
    assert be.sync() and other.sync()
    for out in outs[1:]:
        assert torch.equal(out[0], outs[0][0]) and torch.equal(out[1], outs[0][1])
    other.close()


@pytest.mark.parametrize("lengths,first", [([10, -1, 10], None), ([10, 10, -7], [0, 0, 0]), ([10, 0, 10], [0, -1, 0]), ([-1, 10, 10], [3, 0, 0])])
def test_load_reports_negative_lengths(be, lengths, first):
    """Of requests with rows and without; the others' tokens come back all the same."""
    rng, g = np.random.default_rng(3), gen(3)
    c, table, k, v = filled(be, rng, g, [10, 10, 10], 16, 2, 64)
    for begin in ([0, 10, 20, 30], [0, 10, 10, 20], [5, 5, 5, 5]):
        out = [torch.full((30, 2, 64), 7.0, device="cuda") for _ in range(2)]
        keep = [dev(lengths), dev(begin), dev(first) if first else None]
        torch.cuda.synchronize()
        assert be.kv_load(paged.load_request(c.pages, *out, "f32", table, table.shape[1], keep[0], keep[1], 3, 30, first=keep[2]))
        assert not be.sync() and be.last_error == eb.INVALID_REQUEST
        assert be.sync()
        for b in range(3):
            rows = begin[b + 1] - begin[b]
            sound = lengths[b] == 10 and (not first or first[b] == 0)
            for got, kept in ((out[0], k), (out[1], v)):
                at = got[begin[b]:begin[b + 1]]
                assert torch.equal(at, kept[10 * b:10 * b + rows].float()) if sound else (at == 7.0).all()


@pytest.mark.parametrize("n", [4, 1500])
@pytest.mark.parametrize("where", ["given back", "taken at once", "stack", "unused"])
def test_plan_reports_pages_out_of_range(be, n, where):
    """-1 or a number too large in the row of a request that ends, or on the stack, in the step that meets it; not where none does."""
    page, width = 16, 4
    pages = 4 * n + 8
    for bad in (-1, pages, 1 << 30):
        s = Step(n, width, pages, page, n + 64)
        cached, fresh = np.full(n, 40), np.ones(n, np.int64)
        table = np.arange(4 * n, dtype=np.int32).reshape(n, 4)
        stack = np.full(pages, -77, np.int32)
        stack[:8] = np.arange(4 * n, 4 * n + 8)
        fresh[n // 2] = -1
        if where == "given back":
            table[n // 2, 0] = bad
        elif where == "taken at once":                        # the last given back is the first taken
            table[n // 2, 2] = bad
            fresh[0] = 9
        elif where == "stack":
            stack[7] = bad
            fresh[0], fresh[n // 2] = 9, 1
        else:
            table[n // 2, 3], stack[8] = bad, bad              # behind what the request holds, above the stack's top
        s.cached.copy_(dev(cached.tolist()))
        s.fresh.copy_(dev(fresh.tolist()))
        s.table.copy_(torch.from_numpy(table))
        s.stack.copy_(torch.from_numpy(stack))
        s.count.fill_(8)
        torch.cuda.synchronize()
        assert be.kv_plan(s.request())
        ok = be.sync()
        assert ok == (where == "unused") and (ok or be.last_error == eb.INVALID_REQUEST)
        assert be.sync()
        want = plain.plan(cached, fresh, table, stack, 8, page, n + 64)
        if where in ("taken at once", "stack"):
            want["slots"][want["slots"] // page == bad] = -1
            want["slots"][want["slots"] < 0] = -1
        s.check(want)                                           # passed on as it stands
