"""Bindings of include/emelb_paged.h: a key / value cache in 4-bit pages that many requests share, attention over it, and
attention of packed prompts.

The request builders take device memory as torch tensors or addresses.  Strides default to the tensors' own; a row's head_dim
values are contiguous.  `emel_cpp_b200.Backend` runs the requests: kv_plan, kv_store, kv_load, kv_attend, attend_packed."""
from __future__ import annotations

import ctypes as C

import emel_cpp_b200 as eb

_P = C.c_void_p
_I64 = C.c_int64
_I32 = C.c_int32

MAX_REQUESTS = 8192
TYPES = {"f32": eb.F32, "f16": eb.F16, "bf16": eb.BF16}


class Pages(C.Structure):
    _fields_ = [("data", _P), ("pages", _I32), ("page_tokens", _I32), ("kv_heads", _I32), ("head_dim", _I32)]


class PlanRequest(C.Structure):
    _fields_ = [(n, _P) for n in ("cached", "fresh", "table", "free_pages", "free_count", "free_left", "lengths", "query_begin", "key_begin", "slots",
                                  "positions", "shortage")] + [
        ("table_stride", _I64), ("requests", _I32), ("table_width", _I32), ("pages", _I32), ("page_tokens", _I32), ("token_capacity", _I32)]


class StoreRequest(C.Structure):
    _fields_ = [("cache", Pages), ("k", _P), ("v", _P), ("slots", _P), ("k_token_stride", _I64), ("k_head_stride", _I64), ("v_token_stride", _I64),
                ("v_head_stride", _I64), ("tokens", _I32), ("type", C.c_uint8)]


class LoadRequest(C.Structure):
    _fields_ = [("cache", Pages), ("k", _P), ("v", _P), ("table", _P), ("first", _P), ("lengths", _P), ("row_begin", _P), ("table_stride", _I64),
                ("k_token_stride", _I64), ("k_head_stride", _I64), ("v_token_stride", _I64), ("v_head_stride", _I64), ("requests", _I32),
                ("table_width", _I32), ("rows", _I32), ("type", C.c_uint8)]


class AttendRequest(C.Structure):
    _fields_ = [("cache", Pages), ("q", _P), ("out", _P), ("table", _P), ("lengths", _P), ("query_begin", _P), ("table_stride", _I64),
                ("q_token_stride", _I64), ("q_head_stride", _I64), ("out_token_stride", _I64), ("out_head_stride", _I64), ("requests", _I32),
                ("table_width", _I32), ("heads", _I32), ("queries", _I32), ("max_queries", _I32), ("scale", C.c_float), ("type", C.c_uint8)]


class PackedRequest(C.Structure):
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("out", _P), ("query_begin", _P), ("key_begin", _P), ("q_token_stride", _I64), ("q_head_stride", _I64),
                ("k_token_stride", _I64), ("k_head_stride", _I64), ("v_token_stride", _I64), ("v_head_stride", _I64), ("out_token_stride", _I64),
                ("out_head_stride", _I64), ("requests", _I32), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32), ("queries", _I32), ("keys", _I32),
                ("max_queries", _I32), ("causal", _I32), ("scale", C.c_float), ("type", C.c_uint8)]


_REQUESTS = {"kv_plan": PlanRequest, "kv_store": StoreRequest, "kv_load": LoadRequest, "kv_attend": AttendRequest, "attend_packed": PackedRequest}
SIGNATURES = {"emelb_kv_page_bytes": [_I32, _I32, _I32]}
for _name, _request in _REQUESTS.items():
    SIGNATURES[f"emelb_{_name}"] = [_P, C.POINTER(_request)]
    SIGNATURES[f"emelb_{_name}_can_run"] = [C.POINTER(_request)]


def register(lib):
    for name, args in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = C.c_uint32
        fn.argtypes = args
    lib.emelb_kv_page_bytes.restype = C.c_uint64


def can_run(request) -> int:
    """The error mask of a request's checks that need no GPU; 0: it may run."""
    name = next(n for n, t in _REQUESTS.items() if isinstance(request, t))
    return getattr(eb.lib(), f"emelb_{name}_can_run")(C.byref(request))


def page_bytes(head_dim: int, kv_heads: int, page_tokens: int) -> int:
    """Bytes of one page; 0 for sizes that the cache does not take."""
    return eb.lib().emelb_kv_page_bytes(head_dim, kv_heads, page_tokens)


def pages(data, count: int, page_tokens: int, kv_heads: int, head_dim: int) -> Pages:
    """A cache of `count` pages in device memory of count * page_bytes() bytes."""
    return Pages(eb.ptr(data), count, page_tokens, kv_heads, head_dim)


def _type(t) -> int:
    return TYPES[t] if isinstance(t, str) else t


def _strides(x, given, heads, dim):
    """(token, head) strides of rows: given, a 3-d tensor's own, or those of dense rows."""
    if given is not None:
        return given
    if hasattr(x, "stride") and x.dim() == 3:
        return x.stride(0), x.stride(1)
    return heads * dim, dim


def plan_request(cached, fresh, table, table_width, free_pages, pages, free_count, free_left, lengths, query_begin, key_begin, slots, positions,
                 shortage, requests, page_tokens, token_capacity, table_stride=None) -> PlanRequest:
    """lengths may be cached and free_left free_count: a step in place."""
    arrays = (cached, fresh, table, free_pages, free_count, free_left, lengths, query_begin, key_begin, slots, positions, shortage)
    stride = table_stride if table_stride is not None else table.stride(0) if hasattr(table, "stride") and table.dim() == 2 else table_width
    return PlanRequest(*(eb.ptr(a) for a in arrays), stride, requests, table_width, pages, page_tokens, token_capacity)


def store_request(cache: Pages, k, v, type, slots, tokens, k_strides=None, v_strides=None) -> StoreRequest:
    h, d = cache.kv_heads, cache.head_dim
    return StoreRequest(cache, eb.ptr(k), eb.ptr(v), eb.ptr(slots), *_strides(k, k_strides, h, d), *_strides(v, v_strides, h, d), tokens, _type(type))


def load_request(cache: Pages, k, v, type, table, table_width, lengths, row_begin, requests, rows, first=None, table_stride=None, k_strides=None,
                 v_strides=None) -> LoadRequest:
    h, d = cache.kv_heads, cache.head_dim
    stride = table_stride if table_stride is not None else table.stride(0) if hasattr(table, "stride") and table.dim() == 2 else table_width
    return LoadRequest(cache, eb.ptr(k), eb.ptr(v), eb.ptr(table), eb.ptr(first), eb.ptr(lengths), eb.ptr(row_begin), stride,
                       *_strides(k, k_strides, h, d), *_strides(v, v_strides, h, d), requests, table_width, rows, _type(type))


def attend_request(cache: Pages, q, out, type, table, table_width, lengths, requests, heads, queries, query_begin=None, max_queries=1, scale=None,
                   table_stride=None, q_strides=None, out_strides=None) -> AttendRequest:
    d = cache.head_dim
    stride = table_stride if table_stride is not None else table.stride(0) if hasattr(table, "stride") and table.dim() == 2 else table_width
    return AttendRequest(cache, eb.ptr(q), eb.ptr(out), eb.ptr(table), eb.ptr(lengths), eb.ptr(query_begin), stride, *_strides(q, q_strides, heads, d),
                         *_strides(out, out_strides, heads, d), requests, table_width, heads, queries, max_queries, max(d, 1) ** -0.5 if scale is None else scale,
                         _type(type))


def packed_request(q, k, v, out, type, query_begin, key_begin, requests, heads, kv_heads, head_dim, queries, keys, max_queries=None, causal=True,
                   scale=None, q_strides=None, k_strides=None, v_strides=None, out_strides=None) -> PackedRequest:
    return PackedRequest(eb.ptr(q), eb.ptr(k), eb.ptr(v), eb.ptr(out), eb.ptr(query_begin), eb.ptr(key_begin),
                         *_strides(q, q_strides, heads, head_dim), *_strides(k, k_strides, kv_heads, head_dim),
                         *_strides(v, v_strides, kv_heads, head_dim), *_strides(out, out_strides, heads, head_dim), requests, heads, kv_heads, head_dim,
                         queries, keys, queries if max_queries is None else max_queries, int(causal), max(head_dim, 1) ** -0.5 if scale is None else scale,
                         _type(type))
