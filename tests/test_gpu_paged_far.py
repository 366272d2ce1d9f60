"""The paged operators over many tokens, where sums grow long, work is shared among many and a lost token would hardly show:
equal values, planted keys, and errors held to what the roundings make on average."""
import numpy as np
import pytest
import torch

import emel_cpp_b200 as eb
from emel_cpp_b200 import paged
from tests import paged_plain as plain
from tests.test_gpu_paged import Cache, dev, done, filled, gen, slots_of, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = eb.Backend(0)
    yield b
    b.close()


def exact(q, k, v, scale, causal=True):
    """(result, root of the sum of (weight * value)^2) in 64 bits, a head at a time."""
    n, heads, _ = q.shape
    length, kv = k.shape[:2]
    out, root = (torch.empty(n, heads, v.shape[2], dtype=torch.float64, device=q.device) for _ in range(2))
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(length, device=q.device)[None]
    for h in range(heads):
        g = h // (heads // kv)
        s = q[:, h].double() @ k[:, g].double().T * scale
        if causal:
            s = s.masked_fill(j > length - n + i, -np.inf)
        p = torch.softmax(s, -1)
        out[:, h] = p @ v[:, g].double()
        root[:, h] = (p * p @ (v[:, g].double() ** 2)).sqrt()
    return out, root


def rms(x):
    return float(x.double().square().mean().sqrt())


def check_rms(got, want, root, weight_step, t, score=0.0):
    """Roundings of weights are independent of one another: together about weight_step * root; the result has one more.  Twice that, and
    what errors of the scores make (`score`, relative to root: they are independent, too).  Below 2^-14 f16 results have a fixed step,
    2^-24, of which a rounding is off by half."""
    err, bound = rms(got.double() - want), 2 * ((weight_step + score) * rms(root) + plain.HALF_STEP[t] * rms(want)) + 2.0 ** -25 * (t == "f16")
    assert np.isfinite(err) and err <= bound, (err, bound)


# ---------------------------------------------------------------- packed prompts
@pytest.mark.parametrize("keys,dim,t,lift", [((1 << 20) + 3, 8, "f16", 0.5), (1 << 20, 128, "f16", 0.0), (1 << 22, 8, "bf16", 0.3), (1 << 25, 8, "f16", 0.5)])
def test_packed_equal_values_of_many_keys(be, keys, dim, t, lift):
    """All keys alike but the first, whose score is 2^lift above: sums of equal numbers, where every rounding goes the same way.  The
    tensor cores cut a sum's 17 addends (16 products, O) off at a unit of 2^-23 of O or less, O grows over 512 such products; a weight and a
    result have a rounding each, the sums f32 ones: of 64 weights, 64 tiles, the rest."""
    dt = plain.TORCH[t]
    q, k = torch.zeros(1, 1, dim, device="cuda", dtype=dt), torch.zeros(keys, 1, dim, device="cuda", dtype=dt)
    q[..., 0], k[0, 0, 0] = 1, lift
    v = torch.empty(keys, 1, dim, device="cuda", dtype=dt).copy_(torch.linspace(-3, 2, dim, device="cuda").to(dt))
    out, begin = torch.zeros_like(q), [dev([0, 1]), dev([0, keys])]
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, t, *begin, 1, 1, 1, dim, 1, keys, causal=False, scale=float(np.log(2)))))
    want = v[0].double()
    rel = 2 * plain.HALF_STEP[t] + 256 * 17 * 2.0 ** -23 + (64 + 64 + keys / 8192) * 2.0 ** -24 + 2.0 ** -20
    assert ((out[0].double() - want).abs() <= rel * want.abs()).all(), float(((out[0].double() - want) / want).abs().max())


@pytest.mark.parametrize("queries,keys,heads,kv,dim,t,ramp", [
    (3, 30000, 4, 2, 128, "f16", 0.0), (200, 17000, 2, 1, 64, "bf16", 4.0), (300, 8192 + 128, 2, 2, 128, "f16", -4.0), (70, 8193, 8, 1, 40, "f16", 8.0),
    (5, 100003, 2, 2, 64, "bf16", 0.0), (129, 16384, 1, 1, 128, "bf16", 2.0),
])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_far_errors(be, queries, keys, heads, kv, dim, t, ramp, causal):
    """Random rows whose scores rise (ramp > 0), so that the running maximum moves all the way, or fall, or neither."""
    g, dt = gen(keys), plain.TORCH[t]
    q = torch.randn(queries, heads, dim, generator=g, device="cuda")
    k, v = (torch.randn(keys, kv, dim, generator=g, device="cuda") for _ in range(2))
    q[..., 0], k[..., 0] = 1.0, torch.linspace(0, ramp * dim ** 0.5, keys, device="cuda")[:, None]
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    out, begin = torch.full_like(q, 7.0), [dev([0, queries]), dev([0, keys])]
    torch.cuda.synchronize()
    req = paged.packed_request(q, k, v, out, t, *begin, 1, heads, kv, dim, queries, keys, causal=causal)
    done(be, be.attend_packed(req))
    want, root = exact(q, k, v, dim ** -0.5, causal)
    check_rms(out, want, root, plain.HALF_STEP[t], t)
    first = out.clone()
    done(be, be.attend_packed(req))
    assert torch.equal(first, out)


@pytest.mark.parametrize("keys,dim", [(20000, 64), (8200, 128)])
def test_packed_planted_keys(be, keys, dim):
    """One key takes all of a row's weight: at both sides of every kind of border (tiles of 128, moves of 64 tiles, the ends)."""
    g = gen(keys)
    at = sorted({p for b in (0, 128, 256, 1024, 4096, 8192, 16384, keys) for p in (b - 2, b - 1, b, b + 1) if 0 <= p < keys})
    k = torch.randn(keys, 1, dim, generator=g, device="cuda").sign().bfloat16()
    v = torch.randn(keys, 1, dim, generator=g, device="cuda").bfloat16()
    q = (k[at] * 16).contiguous()                               # 2 * dim^0.5 nats between equal signs and any other sum
    out, begin = torch.zeros_like(q), [dev([0, len(at)]), dev([0, keys])]
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, "bf16", *begin, 1, 1, 1, dim, len(at), keys, causal=False)))
    assert torch.equal(out, v[at])


# ---------------------------------------------------------------- attention over the pages
def repeated(be, page_rows, page_tokens=256):
    """A cache of one page that holds these rows: tables name it as often as they like.  (cache, kept keys, kept values)"""
    k, v = page_rows
    c = Cache(1, page_tokens, k.shape[1], k.shape[2])
    slots = torch.arange(page_tokens, device="cuda")
    torch.cuda.synchronize()
    done(be, be.kv_store(paged.store_request(c.pages, k, v, "f32", slots, page_tokens)))
    return c, plain.kept(k), plain.kept(v)


@pytest.mark.parametrize("length,requests,dim,t", [(1 << 17, 1780, 32, "f32"), (1 << 20, 1780, 32, "f16"), (1 << 20, 1200, 64, "f32"), (1 << 18, 1790, 128, "bf16")])
def test_attend_equal_values_of_many_tokens(be, length, requests, dim, t):
    """So many requests that a warp walks a whole one, over tokens that are all alike: every rounding goes the same way.  The tensor
    cores cut a sum's 17 addends (16 products, the result) off at a unit of 2^-23 of the result or less, which grows over 128 such
    products; a weight has a rounding to f16 (bf16 results: two; f32: one of 22 bits), the result its own, the sums f32 ones: of 128
    weights, 8 lanes, the moves."""
    k, v = torch.zeros(256, 1, dim, device="cuda"), torch.linspace(-3, 2, dim, device="cuda").repeat(256, 1, 1)
    c, _, kept = repeated(be, (k, v))
    table, lengths = torch.zeros(requests, length // 256, dtype=torch.int32, device="cuda"), dev([length] * requests)
    q = torch.ones(requests, 8, dim, device="cuda").to(plain.TORCH[t])
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, length // 256, lengths, requests, 8, requests)))
    want = kept[0]
    rounding = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -10}[t] + plain.HALF_STEP[t]
    rel = rounding + 64 * 17 * 2.0 ** -23 + (128 + 8 + length / 2048) * 2.0 ** -24 + 2.0 ** -21
    assert ((out.double() - want).abs() <= rel * want.abs() + 1e-30).all(), float(((out.double() - want).abs() / want.abs().clamp_min(1e-9)).max())


def weight_step(t, q, k, scale):
    """What a weight is off by, roundings and (as a fraction of it) scores: a head's scores are sums over groups of 32 of products of
    (base + q) and a query value, each of four (f32 queries: eight) instructions cutting off about 2^-22 of what stands there."""
    base = 64.0 if t == "f32" else 1024.0
    score = (8 if t == "f32" else 4) * 2.0 ** -22 * base * 32 ** 0.5 * rms(q) * rms(k) / 4 * scale * (q.shape[2] / 32) ** 0.5
    return {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -10}[t], score


@pytest.mark.parametrize("lengths,rows,heads,kv,dim,t", [
    ([20001], [1], 32, 8, 128, "f16"), ([70000], [3], 8, 1, 64, "bf16"), ([30000, 3, 500, 9000], [1, 3, 2, 4], 16, 4, 128, "bf16"),
    ([12000, 12000], [3, 1], 4, 2, 96, "f16"), ([9000], [5], 8, 1, 128, "f32"), ([40000, 100], [2, 2], 16, 2, 32, "f32"), ([2500] * 40, [1] * 40, 64, 8, 128, "f16"),
    ([1000 + 37 * i for i in range(150)], [1] * 150, 8, 1, 64, "bf16"), ([5000 + i for i in range(130)], [1 + i % 3 for i in range(130)], 16, 2, 96, "f32"),
])
def test_attend_far_errors(be, lengths, rows, heads, kv, dim, t):
    rng, g = np.random.default_rng(len(lengths)), gen(len(lengths) + dim)
    c, table, k, v = filled(be, rng, g, lengths, 32, kv, dim)
    q = torch.randn(sum(rows), heads, dim, generator=g, device="cuda").to(plain.TORCH[t])
    out, begin, lens = torch.full_like(q, 7.0), dev(np.concatenate([[0], np.cumsum(rows)]).tolist()), dev(lengths)
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, table.shape[1], lens, len(lengths), heads, q.shape[0], query_begin=begin,
                                               max_queries=max(rows))))
    at, qa = 0, 0
    for length, n in zip(lengths, rows):
        kk, vv, qq = k[at:at + length], v[at:at + length], q[qa:qa + n]
        want, root = exact(qq, kk, vv, dim ** -0.5)
        check_rms(out[qa:qa + n], want, root, *weight_step(t, qq, kk, dim ** -0.5)[:1], t, weight_step(t, qq, kk, dim ** -0.5)[1])
        at, qa = at + length, qa + n


@pytest.mark.parametrize("length,rows,group,dim,page,t", [(20000, 200, 1, 64, 16, "f16"), (70001, 100, 8, 32, 256, "bf16"), (3001, 64, 2, 128, 32, "f32"), (9000, 300, 3, 96, 64, "f16")])
def test_attend_planted_keys(be, length, rows, group, dim, page, t):
    """One key takes all of a row's weight: at both sides of every kind of border (steps of 32, batches of 32 steps, moves of 64, pages,
    the ends), and anywhere, so that the borders of shares are among them."""
    rng, g = np.random.default_rng(length), gen(length)
    table, pages = tables(rng, [length], page)
    c = Cache(pages, page, 1, dim, fill=0xff)
    k = torch.randn(length, 1, dim, generator=g, device="cuda").sign()
    v = torch.randn(length, 1, dim, generator=g, device="cuda")
    slots, table = dev(slots_of(table, [0], [length], page).tolist(), torch.int64), torch.from_numpy(table).cuda()
    torch.cuda.synchronize()
    done(be, be.kv_store(paged.store_request(c.pages, k, v, "f32", slots, length)))
    seen = length - rows
    at = [p for b in (0, 16, 32, 256, 1024, 2048, 4096, seen) for p in (b - 1, b) if 0 <= p < seen]
    at = np.array((at + rng.integers(0, seen, rows * group).tolist())[:rows * group])
    q = (4 * k[at, 0]).view(rows, group, dim).to(plain.TORCH[t])     # two signs apart is 15 nats
    want = plain.kept(v)[at, 0].view(rows, group, dim).double()
    out, begin, lens = torch.zeros_like(q), dev([0, rows]), dev([length])
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, table.shape[1], lens, 1, group, rows, query_begin=begin, max_queries=rows, scale=1.0)))
    rounding = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -10}[t] + plain.HALF_STEP[t]
    assert ((out.double() - want).abs() <= rounding * want.abs() + 1e-5).all()


@pytest.mark.parametrize("requests,rows,heads,kv,length,t", [(1, 4096, 64, 1, 1 << 21, "f16"), (140, 300, 64, 1, 1 << 17, "bf16"), (100, 150, 128, 2, 150001, "f32")])
def test_attend_long_lines(be, requests, rows, heads, kv, length, t):
    """More than 2^30 steps of 32 tokens for 8 rows of a key / value head in one call, 2^31 for one request: small caches that many rows
    walk.  Tokens repeat every 256, so that weights are known by their counts; rounded alike, they are off by as much."""
    g, dim = gen(rows), 32
    c, k, v = repeated(be, [torch.randn(256, kv, dim, generator=g, device="cuda") for _ in range(2)])
    width = -(-length // 256)
    table, lens = torch.zeros(requests, width, dtype=torch.int32, device="cuda"), dev([length] * requests)
    q = torch.randn(requests * rows, heads, dim, generator=g, device="cuda").to(plain.TORCH[t])
    out, begin = torch.full_like(q, 7.0), dev([rows * b for b in range(requests + 1)])
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, width, lens, requests, heads, requests * rows, query_begin=begin, max_queries=rows)))
    seen = length - rows + 1 + torch.arange(rows, device="cuda")
    count = (seen[:, None] // 256 + (torch.arange(256, device="cuda")[None] < seen[:, None] % 256)).double()
    weight, score = weight_step(t, q, k, dim ** -0.5)
    for b in range(0, requests, max(1, requests // 7)):
        at = slice(b * rows, (b + 1) * rows)
        for h in range(heads):
            s = q[at, h].double() @ k[:, h * kv // heads].double().T * dim ** -0.5
            p = count * torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            vv = v[:, h * kv // heads].double()
            want, size = p @ vv, p @ vv.abs()
            bound = (weight + 40 * score + 64 * 17 * 2.0 ** -23 + 2.0 ** -16) * size + plain.HALF_STEP[t] * want.abs()
            err = (out[at, h].double() - want).abs()
            assert (err <= bound).all(), (b, h, float((err / bound).max()))


def test_attend_lines_beyond_count_are_reported(be):
    """More than 2^40 steps, which would take a quarter of an hour, and more tokens than a request may have: not walked, and said."""
    dim, rows, heads = 32, 4096, 64
    c, _, _ = repeated(be, [torch.zeros(256, 1, dim, device="cuda") for _ in range(2)])
    width = 1 << 23
    table, q = torch.zeros(1, width, dtype=torch.int32, device="cuda"), torch.zeros(rows, heads, dim, dtype=torch.float16, device="cuda")
    for length, n in ((0x7fffffc0, rows), (0x7fffffc1, 1), (0x7fffffff, 1)):
        out, begin, lens = torch.full_like(q, 7.0), dev([0, n]), dev([length])
        torch.cuda.synchronize()
        assert be.kv_attend(paged.attend_request(c.pages, q, out, "f16", table, width, lens, 1, heads, rows, query_begin=begin, max_queries=rows))
        assert not be.sync() and be.last_error == eb.INVALID_REQUEST
        assert be.sync() and (out == 7.0).all()
    # the longest that there may be, by one row
    v = torch.linspace(-1, 1, dim, device="cuda").repeat(256, 1, 1)
    c, _, kept = repeated(be, (torch.zeros_like(v), v))
    q1, out, lens = torch.ones(1, 8, dim, device="cuda"), torch.zeros(1, 8, dim, device="cuda"), dev([0x7fffffc0])
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q1, out, "f32", table, width, lens, 1, 8, 1)))
    assert ((out[0] - kept[0]).abs() <= 2e-4 * kept[0].abs() + 1e-30).all()


@pytest.mark.parametrize("t,q_gain,k_gain,scale", [
    ("bf16", 2.0 ** 30, 1.0, 0.125), ("f32", 2.0 ** 30, 1.0, 0.125), ("f16", 2.0 ** 12, 2.0 ** 12, 0.125), ("bf16", 2.0 ** 60, 2.0 ** 10, 8.0),
    ("f32", 2.0 ** 80, 1.0, 0.125), ("f16", 1.0, 1.0, 2.0 ** 27), ("bf16", 2.0 ** 26, 1.0, 0.125), ("bf16", 2.0 ** 20, 1.0, 0.125), ("f32", -2.0 ** 30, 1.0, 0.125),
    ("f16", 1.0, 2.0 ** 18, 1.0),
])
def test_attend_far_scores(be, t, q_gain, k_gain, scale):
    """Scores whose own rounding is far more than one: the largest takes all the weight (the next is far below it)."""
    dim, heads, lengths = 64, 16, [1500, 1, 40, 700]
    rng, g = np.random.default_rng(3), gen(3)
    c, table, k, v = filled(be, rng, g, lengths, 16, 2, dim, gain=(k_gain, 1.0))
    q = (torch.randn(8, heads, dim, generator=g, device="cuda") * q_gain).to(plain.TORCH[t])
    out, lens, begin = torch.full_like(q, 7.0), dev(lengths), dev([0, 2, 3, 5, 8])
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, table.shape[1], lens, 4, heads, 8, query_begin=begin, max_queries=3, scale=scale)))
    at = 0
    for b, (length, qa, qb) in enumerate(zip(lengths, (0, 2, 3, 5), (2, 3, 5, 8))):
        want, _ = exact(q[qa:qb], k[at:at + length], v[at:at + length], scale)
        rounding = weight_step(t, q, k, scale)[0] + 2.0 ** -16 + plain.HALF_STEP[t]
        err = (out[qa:qb].double() - want).abs()
        assert (err <= rounding * want.abs() + 1e-30).all(), (b, float(err.max()))
        at += length


@pytest.mark.parametrize("t,above", [("bf16", 2.0 ** 44), ("f32", 2.0 ** 44), ("f32", 2.0 ** 20), ("f16", 2.0 ** 12), ("bf16", 2.0 ** 100), ("f32", 2.0 ** 100)])
def test_attend_rows_keep_to_themselves(be, t, above):
    """Heads and rows of far larger and smaller values in one tile of rows: each as exact as among its like.  (Not the same bits: when
    a row's running maximum moves, the others of its tile move with it, and weights are rounded against another number.)"""
    dim, heads, length = 64, 16, 500
    rng, g = np.random.default_rng(3), gen(3)
    c, table, k, v = filled(be, rng, g, [length], 16, 2, dim)
    q = torch.randn(3, heads, dim, generator=g, device="cuda").to(plain.TORCH[t])
    lens, begin, out = dev([length]), dev([0, 3]), torch.full_like(q, 7.0)
    weight, score = weight_step(t, q, k, dim ** -0.5)
    for i, h, by in ((0, 2, above), (1, 5, above), (2, 14, 1 / above), (2, 9, above)):
        q[i, h] *= by
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, table.shape[1], lens, 1, heads, 3, query_begin=begin, max_queries=3)))
    want, _ = exact(q, k, v, dim ** -0.5)
    size, _ = exact(q, k, v.abs(), dim ** -0.5)
    bound = (weight + 40 * score + 2.0 ** -16) * size + plain.HALF_STEP[t] * want.abs()
    # Rows `above` times as large: nearly all weight to one key.  Their scores' errors are so many times larger, too: a weight among the
    # rest, p of the largest one's, is off by a factor of exp(40 * score * above) at most, and cannot pass the largest one's, so the result
    # by the rest's sum times that (or 1 a key) times the largest value.
    for i, h in ((0, 2), (1, 5), (2, 9)):
        s = q[i, h].double() @ k[:, h // 8].double().T * dim ** -0.5
        gap = (s.max() - s).sort().values[1:]
        bound[i, h] += torch.exp(torch.clamp(40 * score * above - gap, max=0)).sum() * v[:, h // 8].abs().max()
    err = (out.double() - want).abs()
    assert (err <= bound).all(), ((err / bound).amax(-1))


@pytest.mark.parametrize("t,small", [("f32", 2.0 ** -100), ("bf16", 2.0 ** -100), ("f32", 2.0 ** 100)])
def test_attend_scales_and_queries_far_apart(be, t, small):
    """Queries times a power of two and the scale times its inverse: the same scores, the same bits."""
    rng, g = np.random.default_rng(4), gen(4)
    c, table, k, v = filled(be, rng, g, [300], 16, 1, 128)
    q, lens = torch.randn(1, 8, 128, generator=g, device="cuda").to(plain.TORCH[t]), dev([300])
    outs = []
    for by in (1.0, small):
        x, out = q * by, torch.zeros_like(q)
        torch.cuda.synchronize()
        done(be, be.kv_attend(paged.attend_request(c.pages, x, out, t, table, table.shape[1], lens, 1, 8, 1, scale=128 ** -0.5 / by)))
        outs.append(out)
    assert torch.equal(*outs)


@pytest.mark.parametrize("t,dim,scales,tail", [
    ("f16", 64, (4, -10), -10), ("bf16", 64, (4, -10), -10), ("f32", 64, (4, -6), -4), ("f16", 128, (10, 0, -4, -12), -3), ("f32", 96, (0, -3, -9), -5),
    ("bf16", 128, (15, 14, 3, 0), -8), ("f16", 32, (-20,), -6), ("f32", 64, (-12, -14), -8),
])
def test_attend_values_of_groups_far_apart(be, t, dim, scales, tail):
    """Groups of 32 dims whose scales are 2^scales, one key 2^-tail above all the others: what the many small weights bring keeps its
    digits in every group."""
    g, length, page = gen(dim), 4001, 16
    rng = np.random.default_rng(dim)
    table, pages = tables(rng, [length], page)
    c = Cache(pages, page, 1, dim)
    k, v = torch.zeros(length, 1, dim, device="cuda"), torch.rand(length, 1, dim, generator=g, device="cuda") * 2 - 1
    k[700, 0, 0] = -tail
    for j, e in enumerate(scales):
        v[..., 32 * j:32 * j + 32] *= 8 * 2.0 ** e * (1 - 2.0 ** -11)
    slots, table = dev(slots_of(table, [0], [length], page).tolist(), torch.int64), torch.from_numpy(table).cuda()
    q, lens = torch.zeros(1, 4, dim, device="cuda").to(plain.TORCH[t]), dev([length])
    q[..., 0] = 1
    out, scale = torch.zeros_like(q), float(np.log(2))
    torch.cuda.synchronize()
    done(be, be.kv_store(paged.store_request(c.pages, k, v, "f32", slots, length)))
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, table.shape[1], lens, 1, 4, 1, scale=scale)))
    want, root = exact(q, plain.kept(k), plain.kept(v), scale)
    for j in range(len(scales)):
        at = slice(32 * j, 32 * j + 32)
        check_rms(out[..., at], want[..., at], root[..., at], {"f32": 2.0 ** -20, "f16": 2.0 ** -11, "bf16": 2.0 ** -10}[t], t)


@pytest.mark.parametrize("t,dim,q_gain,k_gain,scale", [
    ("f16", 64, 2.0 ** 12, 2.0 ** 12, 0.125), ("bf16", 64, 2.0 ** 30, 1.0, 0.125), ("bf16", 128, 2.0 ** 50, 2.0 ** 30, 1.0), ("f16", 128, 1.0, 1.0, 2.0 ** 26),
    ("bf16", 40, 2.0 ** 20, 1.0, 1.0), ("f16", 64, 1.0, -1.0, 2.0 ** 24), ("f16", 64, 1.0, 1.0, 2.0 ** 25),
])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_far_scores(be, t, dim, q_gain, k_gain, scale, causal):
    """Scores whose own rounding is far more than one: the largest takes all the weight (the next is far below it)."""
    queries, keys, heads, kv = [300, 1, 40, 7], [700, 1, 200, 7], 4, 2
    g, dt = gen(dim), plain.TORCH[t]
    q = (torch.randn(sum(queries), heads, dim, generator=g, device="cuda") * q_gain).to(dt)
    k = (torch.randn(sum(keys), kv, dim, generator=g, device="cuda") * k_gain).to(dt)
    v = torch.randn(sum(keys), kv, dim, generator=g, device="cuda").to(dt)
    out, qb, kb = torch.full_like(q, 7.0), np.concatenate([[0], np.cumsum(queries)]), np.concatenate([[0], np.cumsum(keys)])
    begin = [dev(qb.tolist()), dev(kb.tolist())]
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, t, *begin, 4, heads, kv, dim, sum(queries), sum(keys), causal=causal, scale=scale)))
    near = 0
    for b in range(4):
        qs, ks = slice(qb[b], qb[b + 1]), slice(kb[b], kb[b + 1])
        want, _ = exact(q[qs], k[ks], v[ks], scale, causal)
        root = exact(q[qs], k[ks], v[ks] * 0 + 1, scale, causal)[1]     # of the weights alone: 1 where one has all
        sure = (root - 1).abs() < 1e-9
        near += int((~sure[..., 0]).sum())
        err = (out[qs].double() - want).abs()
        assert torch.isfinite(out[qs]).all() and (err <= (2 * plain.HALF_STEP[t] + 2.0 ** -16) * want.abs())[sure].all(), b
    assert near <= 4                                            # a few rows' two largest scores may lie that near to one another


@pytest.mark.parametrize("keys,dim,ramp", [(20000, 64, 4.0), (20000, 128, -4.0), (17000, 40, 0.0)])
def test_packed_far_scores_of_many_keys(be, keys, dim, ramp):
    """Far scores that rise, fall or neither over moves of the result, and pairs of alike keys at both ends, which share the weight."""
    g, heads, scale = gen(keys + dim), 2, 2.0 ** 24
    k = torch.randn(keys, heads, dim, generator=g, device="cuda").sign()
    k[..., 0] = torch.linspace(0, ramp, keys, device="cuda")[:, None]
    v = torch.randn(keys, heads, dim, generator=g, device="cuda")
    pairs = [(3, keys - 2), (100, 9000), (8191, 8192), (16383, 16384), (128, 129)]
    for i, j in pairs:
        k[i] = k[j]
    q = torch.stack([k[j] for _, j in pairs])
    q[..., 0] = 0                                          # the two of a pair are the largest, whatever the ramp
    rising = torch.zeros(1, heads, dim, device="cuda")
    rising[..., 0] = 1
    q, k, v = torch.cat([q, rising]).half(), k.half(), v.half()
    out, begin = torch.full_like(q, 7.0), [dev([0, len(q)]), dev([0, keys])]
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, "f16", *begin, 1, heads, heads, dim, len(q), keys, causal=False, scale=scale)))
    want, _ = exact(q, k, v, scale, False)
    size, _ = exact(q, k, v.abs(), scale, False)
    rows = slice(0, None if ramp else len(pairs))          # without a ramp the last row's scores are all alike
    assert ((out.double() - want).abs() <= 2 * plain.HALF_STEP["f16"] * size + plain.HALF_STEP["f16"] * want.abs() + 1e-7)[rows].all()


@pytest.mark.parametrize("t,gain", [("f32", 2.0 ** 30), ("bf16", 2.0 ** 40), ("f16", 2.0 ** 13)])
def test_attend_far_scores_alike(be, t, gain):
    """The largest of far scores comes back every 256 tokens: in other steps, warps, moves and units, all of which share its weight."""
    g, dim, heads = gen(5), 64, 8
    c, k, v = repeated(be, [torch.randn(256, 1, dim, generator=g, device="cuda") for _ in range(2)])
    lengths = [1 << 20, 256, 70000, 300]
    table, lens = torch.zeros(4, 4096, dtype=torch.int32, device="cuda"), dev(lengths)
    q = (torch.randn(4, heads, dim, generator=g, device="cuda") * gain).to(plain.TORCH[t])
    out, scale = torch.full_like(q, 7.0), 2.0 ** 14
    torch.cuda.synchronize()
    done(be, be.kv_attend(paged.attend_request(c.pages, q, out, t, table, 4096, lens, 4, heads, 4, scale=scale)))
    want, _ = exact(q, k, v, scale, False)
    rounding = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -10}[t] + plain.HALF_STEP[t] + 2.0 ** -16 + 64 * 17 * 2.0 ** -23
    assert ((out.double() - want).abs() <= rounding * want.abs() + 1e-30).all()


@pytest.mark.parametrize("t,keys,lift", [("f16", 1 << 20, 22.58), ("f16", 120001, 18.6), ("bf16", 1 << 20, 22.58), ("f16", 30000, 14.3)])
def test_packed_many_small_weights(be, t, keys, lift):
    """One key 2^lift above all the others, which together still count: the first by 1, in the sum, the others by keys * 2^-lift.  A weight
    has a rounding to the type's bits, in f16 to a grid of 2^-31 of the largest at least (2^-24 over 2^7), for all of them the same."""
    dim, dt = 64, plain.TORCH[t]
    q, k = torch.zeros(2, 1, dim, device="cuda", dtype=dt), torch.zeros(keys, 1, dim, device="cuda", dtype=dt)
    q[0, 0, 0], q[1, 0, 1] = 1, 1
    k[700, 0, 0], k[keys - 3, 0, 1] = lift, lift
    v = torch.empty(keys, 1, dim, device="cuda", dtype=dt).copy_(torch.linspace(-3, 2, dim, device="cuda").to(dt))
    v[700], v[keys - 3] = -v[700], -v[keys - 3]
    out, begin, scale = torch.zeros_like(q), [dev([0, 2]), dev([0, keys])], float(np.log(2))
    torch.cuda.synchronize()
    done(be, be.attend_packed(paged.packed_request(q, k, v, out, t, *begin, 1, 1, 1, dim, 2, keys, causal=False, scale=scale)))
    want, _ = exact(q, k, v, scale, False)
    size = v[0].double().abs()
    up = float(k[700, 0, 0])
    rest = (keys - 1) * 2.0 ** -up / (1 + (keys - 1) * 2.0 ** -up)
    weight = plain.HALF_STEP[t] if t == "bf16" else max(2.0 ** -11, 2.0 ** (up - 32))
    rel = plain.HALF_STEP[t] + weight * rest + 2.0 ** -18
    assert ((out.double() - want).abs() <= rel * size + plain.HALF_STEP[t] * want.abs() + 256 * 17 * 2.0 ** -23 * rest * size).all()
