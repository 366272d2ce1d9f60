"""The paged operators' checks of their requests, and the cache's sizes.  CPU only: nothing is launched and no pointer followed."""
import ctypes as C

import pytest

import emel_cpp_b200 as eb
from emel_cpp_b200 import paged

MB = 1 << 20


def at(n):
    """An address in a region of its own."""
    return 0x7000_0000_0000 + n * 64 * MB


def cache(**kw):
    a = dict(data=at(0), count=100, page_tokens=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return paged.pages(a["data"], a["count"], a["page_tokens"], a["kv_heads"], a["head_dim"])


def test_page_bytes():
    for dim in (32, 64, 96, 128):
        for heads in (1, 3, 8):
            for page in (16, 32, 64, 128, 256):
                assert paged.page_bytes(dim, heads, page) == 2 * heads * page * dim * 18 // 32
    for dim, heads, page in ((0, 1, 16), (40, 1, 16), (160, 1, 16), (64, 0, 16), (64, 1, 8), (64, 1, 48), (64, 1, 512), (-64, 1, 16)):
        assert paged.page_bytes(dim, heads, page) == 0


def test_null_requests_and_contexts():
    lib = eb.lib()
    for name, t in paged._REQUESTS.items():
        assert getattr(lib, f"emelb_{name}_can_run")(None) == eb.INVALID_REQUEST
        assert getattr(lib, f"emelb_{name}")(None, C.byref(t())) == eb.INVALID_REQUEST
        assert paged.can_run(t()) == eb.INVALID_REQUEST


PLAN = dict(cached=at(1), fresh=at(2), table=at(3), table_width=40, free_pages=at(4), pages=500, free_count=at(5), free_left=at(6), lengths=at(7),
            query_begin=at(8), key_begin=at(9), slots=at(10), positions=at(11), shortage=at(12), requests=7, page_tokens=16, token_capacity=64)


@pytest.mark.parametrize("change,why", [
    ({}, eb.OK), (dict(lengths=at(1)), eb.OK), (dict(free_left=at(5)), eb.OK), (dict(lengths=at(1), free_left=at(5)), eb.OK),
    (dict(table_stride=50), eb.OK), (dict(requests=8192), eb.OK), (dict(page_tokens=256), eb.OK),
    (dict(requests=0), eb.INVALID_REQUEST), (dict(requests=8193), eb.UNSUPPORTED_OP), (dict(table_width=0), eb.INVALID_REQUEST),
    (dict(table_stride=39), eb.INVALID_REQUEST), (dict(pages=0), eb.INVALID_REQUEST), (dict(token_capacity=0), eb.INVALID_REQUEST),
    (dict(page_tokens=0), eb.INVALID_REQUEST), (dict(page_tokens=8), eb.UNSUPPORTED_OP), (dict(page_tokens=48), eb.UNSUPPORTED_OP),
    (dict(page_tokens=512), eb.UNSUPPORTED_OP), (dict(cached=0), eb.INVALID_REQUEST), (dict(fresh=at(2) + 2), eb.INVALID_REQUEST),
    (dict(slots=at(10) + 4), eb.INVALID_REQUEST), (dict(slots=0), eb.INVALID_REQUEST), (dict(shortage=0), eb.INVALID_REQUEST),
    (dict(lengths=at(1) + 4), eb.INVALID_REQUEST), (dict(lengths=at(2)), eb.INVALID_REQUEST), (dict(free_left=at(1)), eb.INVALID_REQUEST),
    (dict(positions=at(10) + 8), eb.INVALID_REQUEST), (dict(table=at(4) + 1996), eb.INVALID_REQUEST), (dict(key_begin=at(8) + 28), eb.INVALID_REQUEST),
    (dict(key_begin=at(8) + 32), eb.OK),
])
def test_plan_requests(change, why):
    assert paged.can_run(paged.plan_request(**{**PLAN, **change})) == why


@pytest.mark.parametrize("kw,change,why", [
    ({}, {}, eb.OK), (dict(head_dim=96, page_tokens=128), {}, eb.OK), ({}, dict(type=99), eb.UNSUPPORTED_OP), ({}, dict(type=eb.Q4_0), eb.UNSUPPORTED_OP),
    (dict(head_dim=80), {}, eb.UNSUPPORTED_OP), (dict(head_dim=0), {}, eb.INVALID_REQUEST), (dict(page_tokens=24), {}, eb.UNSUPPORTED_OP),
    (dict(kv_heads=0), {}, eb.INVALID_REQUEST), (dict(kv_heads=65536), {}, eb.UNSUPPORTED_OP), (dict(count=0), {}, eb.INVALID_REQUEST),
    (dict(data=at(0) + 8), {}, eb.INVALID_REQUEST), (dict(data=0), {}, eb.INVALID_REQUEST), ({}, dict(tokens=0), eb.INVALID_REQUEST),
    ({}, dict(tokens=-1), eb.INVALID_REQUEST), ({}, dict(k=0), eb.INVALID_REQUEST), ({}, dict(v=at(2) + 1), eb.INVALID_REQUEST),
    ({}, dict(v=at(2) + 2), eb.OK), ({}, dict(slots=at(3) + 4), eb.INVALID_REQUEST), ({}, dict(k_strides=(127, 64)), eb.OK),
    ({}, dict(k_strides=(63, 64)), eb.INVALID_REQUEST), ({}, dict(k_strides=(128, 63)), eb.INVALID_REQUEST),
    ({}, dict(v_strides=(-128, 64)), eb.INVALID_REQUEST), ({}, dict(v_strides=(64, 64 * 9)), eb.OK), ({}, dict(k=at(0) + 1024), eb.INVALID_REQUEST),
    ({}, dict(slots=at(0)), eb.INVALID_REQUEST), ({}, dict(k_strides=(1 << 41, 64)), eb.INVALID_REQUEST),
    ({}, dict(tokens=1 << 30, k_strides=(1 << 40, 64)), eb.INVALID_REQUEST), (dict(data=at(100), kv_heads=60000), dict(k=at(101), v=at(200), slots=at(300)), eb.INVALID_REQUEST),
    (dict(data=at(60000000), kv_heads=8000), dict(k=at(0), v=at(20000000), slots=at(40000000), tokens=1 << 30), eb.UNSUPPORTED_OP),
])
def test_store_requests(kw, change, why):
    a = dict(k=at(1), v=at(2), type="f16", slots=at(3), tokens=9)
    assert paged.can_run(paged.store_request(cache(**kw), **{**a, **change})) == why


@pytest.mark.parametrize("kw,change,why", [
    ({}, {}, eb.OK), ({}, dict(first=at(6)), eb.OK), ({}, dict(type="f32"), eb.OK), ({}, dict(type=7), eb.UNSUPPORTED_OP),
    (dict(head_dim=48), {}, eb.UNSUPPORTED_OP), ({}, dict(rows=0), eb.INVALID_REQUEST), ({}, dict(requests=0), eb.INVALID_REQUEST),
    ({}, dict(table_stride=3), eb.INVALID_REQUEST), ({}, dict(first=at(6) + 1), eb.INVALID_REQUEST), ({}, dict(lengths=0), eb.INVALID_REQUEST),
    ({}, dict(k_strides=(64, 64)), eb.INVALID_REQUEST),                      # a row's heads on the next row's
    ({}, dict(k_strides=(64, 640)), eb.OK), ({}, dict(v=at(1)), eb.INVALID_REQUEST), ({}, dict(v=at(1) + 64), eb.INVALID_REQUEST),
    ({}, dict(v=at(1) + 256, k_strides=(256, 64), v_strides=(256, 64)), eb.OK),   # keys and values side by side in a row
    ({}, dict(v=at(1) + 128, k_strides=(256, 128), v_strides=(256, 128)), eb.INVALID_REQUEST),
    ({}, dict(k=at(0)), eb.INVALID_REQUEST), ({}, dict(v=at(3)), eb.INVALID_REQUEST), ({}, dict(k=at(4) - 8), eb.INVALID_REQUEST),
    (dict(data=at(1000)), dict(requests=1 << 30, table_stride=1 << 30, lengths=at(5000), row_begin=at(6000)), eb.INVALID_REQUEST),
    ({}, dict(requests=300000000, table=at(100), table_width=1, lengths=at(1000), row_begin=at(2000)), eb.UNSUPPORTED_OP),
])
def test_load_requests(kw, change, why):
    a = dict(k=at(1), v=at(2), type="bf16", table=at(3), table_width=4, lengths=at(4), row_begin=at(5), requests=3, rows=10)
    assert paged.can_run(paged.load_request(cache(**kw), **{**a, **change})) == why


@pytest.mark.parametrize("kw,change,why", [
    ({}, {}, eb.OK), ({}, dict(query_begin=at(5), queries=20, max_queries=8), eb.OK), ({}, dict(type="f32"), eb.OK), ({}, dict(type=3), eb.UNSUPPORTED_OP),
    ({}, dict(heads=5), eb.INVALID_REQUEST), ({}, dict(heads=128), eb.OK), ({}, dict(heads=130), eb.UNSUPPORTED_OP), ({}, dict(heads=0), eb.INVALID_REQUEST),
    ({}, dict(scale=0.0), eb.INVALID_REQUEST), ({}, dict(scale=-1.0), eb.INVALID_REQUEST), ({}, dict(scale=float("nan")), eb.INVALID_REQUEST),
    ({}, dict(scale=float("inf")), eb.INVALID_REQUEST), ({}, dict(scale=3e38), eb.INVALID_REQUEST), ({}, dict(scale=float("nan")), eb.INVALID_REQUEST), ({}, dict(queries=2), eb.INVALID_REQUEST), ({}, dict(max_queries=0), eb.INVALID_REQUEST),
    ({}, dict(requests=8193, queries=8193), eb.UNSUPPORTED_OP), ({}, dict(out=at(1)), eb.INVALID_REQUEST), ({}, dict(out=at(0)), eb.INVALID_REQUEST),
    ({}, dict(out_strides=(64, 64)), eb.INVALID_REQUEST), ({}, dict(q_strides=(512, 64)), eb.OK), ({}, dict(table_stride=1), eb.INVALID_REQUEST),
    (dict(head_dim=160), {}, eb.UNSUPPORTED_OP), (dict(page_tokens=17), {}, eb.UNSUPPORTED_OP), ({}, dict(lengths=at(4) + 2), eb.INVALID_REQUEST),
])
def test_attend_requests(kw, change, why):
    a = dict(q=at(1), out=at(2), type="f16", table=at(3), table_width=4, lengths=at(4), requests=3, heads=4, queries=3)
    assert paged.can_run(paged.attend_request(cache(**kw), **{**a, **change})) == why


@pytest.mark.parametrize("change,why", [
    ({}, eb.OK), (dict(causal=False), eb.OK), (dict(head_dim=8), eb.OK), (dict(head_dim=72), eb.OK), (dict(keys=0), eb.OK), (dict(type="bf16"), eb.OK),
    (dict(type="f32"), eb.UNSUPPORTED_OP), (dict(head_dim=68), eb.UNSUPPORTED_OP), (dict(head_dim=136), eb.UNSUPPORTED_OP),
    (dict(head_dim=0), eb.INVALID_REQUEST), (dict(heads=3), eb.INVALID_REQUEST), (dict(heads=256), eb.OK), (dict(heads=258), eb.UNSUPPORTED_OP),
    (dict(queries=0), eb.INVALID_REQUEST), (dict(keys=-1), eb.INVALID_REQUEST), (dict(requests=0), eb.INVALID_REQUEST), (dict(scale=0.0), eb.INVALID_REQUEST),
    (dict(scale=2.0 ** 127), eb.INVALID_REQUEST), (dict(scale=2.0 ** 126), eb.OK), (dict(scale=float("nan")), eb.INVALID_REQUEST),
    (dict(q=at(0) + 2), eb.UNSUPPORTED_OP), (dict(q=at(0) + 1), eb.INVALID_REQUEST), (dict(k_strides=(132, 64)), eb.UNSUPPORTED_OP),
    (dict(k_strides=(136, 64)), eb.OK), (dict(v_strides=(64, 1280)), eb.OK), (dict(out=at(0)), eb.INVALID_REQUEST), (dict(out=at(2) + 16), eb.INVALID_REQUEST),
    (dict(out_strides=(64, 64)), eb.INVALID_REQUEST), (dict(query_begin=at(4) + 2), eb.INVALID_REQUEST), (dict(max_queries=0), eb.INVALID_REQUEST),
    (dict(keys=1 << 25, k=at(1000), v=at(2000), out=at(3000)), eb.OK), (dict(keys=(1 << 25) + 1, k=at(1000), v=at(2000), out=at(3000)), eb.UNSUPPORTED_OP),
    (dict(heads=60000, kv_heads=60000, requests=20000, q=at(10), k=at(20), v=at(30), out=at(40)), eb.UNSUPPORTED_OP),
    (dict(k=at(50), k_strides=(1 << 39, 64)), eb.UNSUPPORTED_OP), (dict(v=at(50), v_strides=(64, (1 << 39) - 8)), eb.OK),
])
def test_packed_requests(change, why):
    a = dict(q=at(0), k=at(1), v=at(2), out=at(3), type="f16", query_begin=at(4), key_begin=at(5), requests=3, heads=4, kv_heads=2, head_dim=64, queries=20,
             keys=30)
    assert paged.can_run(paged.packed_request(**{**a, **change})) == why


def test_tensors_that_do_not_fit_their_request():
    """The builders look at a tensor's type, size and innermost stride; at the same values by their address they do not."""
    import torch
    z = lambda *shape, t=torch.int32: torch.zeros(*shape, dtype=t)  # noqa: E731
    c = paged.pages(z(100 * paged.page_bytes(64, 2, 16), t=torch.uint8), 100, 16, 2, 64)
    half, wide = z(9, 2, 64, t=torch.float16), z(9, 2, 128, t=torch.float16)

    plan = dict(cached=z(7), fresh=z(7), table=z(7, 50)[:, :40], table_width=40, free_pages=z(500), pages=500, free_count=z(1), free_left=z(1), lengths=z(7),
                query_begin=z(8), key_begin=z(8), slots=z(64, t=torch.int64), positions=z(64), shortage=z(1), requests=7, page_tokens=16, token_capacity=64)
    store = dict(cache=c, k=half, v=half.clone(), type="f16", slots=z(9, t=torch.int64), tokens=9)
    load = dict(cache=c, k=half, v=half.clone(), type="f16", table=z(3, 4), table_width=4, lengths=z(3), row_begin=z(4), requests=3, rows=9)
    attend = dict(cache=c, q=z(3, 4, 64, t=torch.float16), out=z(3, 4, 64, t=torch.float16), type="f16", table=z(3, 4), table_width=4, lengths=z(3), requests=3,
                  heads=4, queries=3)
    packed = dict(q=half, k=half, v=half, out=half.clone(), type="f16", query_begin=z(4), key_begin=z(4), requests=3, heads=2, kv_heads=2, head_dim=64, queries=9,
                  keys=9)
    builders = {paged.plan_request: plan, paged.store_request: store, paged.load_request: load, paged.attend_request: attend, paged.packed_request: packed}
    for build, a in builders.items():
        assert paged.can_run(build(**a)) in (eb.OK, eb.UNSUPPORTED_OP)      # host memory may lie at any address
    for build, change in (
            (paged.plan_request, dict(cached=z(7, t=torch.int64))), (paged.plan_request, dict(fresh=z(6))), (paged.plan_request, dict(slots=z(64))),
            (paged.plan_request, dict(slots=z(63, t=torch.int64))), (paged.plan_request, dict(query_begin=z(7))), (paged.plan_request, dict(lengths=z(14)[::2])),
            (paged.plan_request, dict(table=z(7, 80)[:, ::2])), (paged.plan_request, dict(table=z(6, 40))), (paged.plan_request, dict(table=z(7, 39))),
            (paged.plan_request, dict(table=z(7, 40, t=torch.int64))), (paged.plan_request, dict(free_pages=z(499))), (paged.plan_request, dict(table=z(279))),
            (paged.store_request, dict(k=half.float())), (paged.store_request, dict(v=half.bfloat16())), (paged.store_request, dict(type="f32")),
            (paged.store_request, dict(k=wide[:, :, ::2])), (paged.store_request, dict(k=half[:8])), (paged.store_request, dict(k=half[:, :1])),
            (paged.store_request, dict(v=half[..., :32])), (paged.store_request, dict(slots=z(9))), (paged.store_request, dict(k=half.transpose(1, 2))),
            (paged.store_request, dict(k=z(9 * 2 * 64 - 1, t=torch.float16))), (paged.store_request, dict(k=wide[:, :, ::2], k_strides=(256, 128))),
            (paged.load_request, dict(lengths=z(3, t=torch.int64))), (paged.load_request, dict(row_begin=z(3))), (paged.load_request, dict(first=z(2))),
            (paged.load_request, dict(k=half[:8])), (paged.load_request, dict(table=z(2, 4))), (paged.load_request, dict(type="bf16")),
            (paged.attend_request, dict(q=z(3, 4, 64))), (paged.attend_request, dict(out=z(2, 4, 64, t=torch.float16))), (paged.attend_request, dict(lengths=z(2))),
            (paged.attend_request, dict(query_begin=z(3))), (paged.attend_request, dict(heads=6)), (paged.attend_request, dict(queries=4)),
            (paged.packed_request, dict(keys=10)), (paged.packed_request, dict(queries=10)), (paged.packed_request, dict(k=wide[:, :, 1::2])),
            (paged.packed_request, dict(type="bf16")), (paged.packed_request, dict(key_begin=z(4, t=torch.int64))), (paged.packed_request, dict(head_dim=72))):
        with pytest.raises(ValueError):
            build(**{**builders[build], **change})
    with pytest.raises(ValueError):
        paged.pages(z(100 * paged.page_bytes(64, 2, 16) - 1, t=torch.uint8), 100, 16, 2, 64)
    with pytest.raises(ValueError):
        paged.pages(z(100 * paged.page_bytes(64, 2, 16)), 100, 16, 2, 64)
    # what fits: more rows, heads and values than asked for, other layouts, addresses
    paged.store_request(c, wide[..., :64], z(12, 3, 64, t=torch.float16), "f16", z(20, t=torch.int64), 9)
    paged.store_request(c, half.transpose(0, 1).contiguous().transpose(0, 1), z(9 * 2 * 64, t=torch.float16), "f16", at(1), 9)
    paged.store_request(c, at(2), at(3), "f16", at(1), 9)


@pytest.mark.parametrize("tokens,why", [(0x7ffffff0, eb.OK), (0x7ffffff1, eb.UNSUPPORTED_OP), (0x7fffffff, eb.UNSUPPORTED_OP)])
def test_store_of_the_most_rows(tokens, why):
    """Places of a last tile of 16 rows are ints."""
    c = cache(head_dim=32, kv_heads=1, data=at(10000000))
    assert paged.can_run(paged.store_request(c, at(0), at(0), "f16", at(5000), tokens)) == why
