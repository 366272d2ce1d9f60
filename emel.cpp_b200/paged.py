"""Bindings of include/emelb_paged.h: a key / value cache in 4-bit pages that many requests share, attention over it, and
attention of packed prompts.

The request builders take device memory as torch tensors or addresses.  Strides default to the tensors' own; a row's head_dim
values are contiguous.  A tensor of another type than the request's (int32 for lengths, tables and sums, int64 for slots), with too few
values or with gaps inside a row is a ValueError; an address is taken at its word.  `emel_cpp_b200.Backend` runs the requests: kv_plan, kv_store, kv_load, kv_attend, attend_packed."""
from __future__ import annotations

import ctypes as C

import emel_cpp_b200 as eb

_P = C.c_void_p
_I64 = C.c_int64
_I32 = C.c_int32

MAX_REQUESTS = 8192
TYPES = {"f32": eb.F32, "f16": eb.F16, "bf16": eb.BF16}
DTYPES = {eb.F32: "float32", eb.F16: "float16", eb.BF16: "bfloat16"}


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


def _tensor(x) -> bool:
    return hasattr(x, "data_ptr") and hasattr(x, "stride")


def _fits(name, x, dtype, enough, dense):
    if str(x.dtype) != f"torch.{dtype}":
        raise ValueError(f"{name}: {x.dtype}, not {dtype}")
    if not enough:
        raise ValueError(f"{name}: a tensor of {tuple(x.shape)} is too small for the request")
    if not dense:
        raise ValueError(f"{name}: values that have to be neighbours are {x.stride()} apart")


def _array(name, x, count, dtype="int32") -> int:
    """The address of `count` neighbouring numbers."""
    if _tensor(x):
        _fits(name, x, dtype, x.numel() >= count, x.is_contiguous())
    return eb.ptr(x)


def _rows(name, x, given, type, rows, heads, dim):
    """(token, head) strides of rows: given, a 3-d tensor's own, or those of dense rows."""
    own = _tensor(x) and x.dim() == 3
    if _tensor(x):
        dtype = DTYPES.get(type, str(x.dtype).removeprefix("torch."))     # of a type that nothing takes: refused with the request
        enough = x.shape[0] >= rows and x.shape[1] >= heads and x.shape[2] >= dim if own else x.numel() >= rows * heads * dim
        _fits(name, x, dtype, given is not None or enough, x.stride(2) == 1 or dim <= 1 if own else given is not None or x.is_contiguous())
    if given is not None:
        return given
    return (x.stride(0), x.stride(1)) if own else (heads * dim, dim)


def _table(x, stride, requests, width):
    """(address, stride) of a page table."""
    own = _tensor(x) and x.dim() == 2
    if stride is None:
        stride = x.stride(0) if own else width
    if _tensor(x):
        enough = x.shape[0] >= requests and x.shape[1] >= width if own else x.numel() >= (requests - 1) * stride + width
        _fits("table", x, "int32", enough, x.stride(1) == 1 or width <= 1 if own else x.is_contiguous())
    return eb.ptr(x), stride


def pages(data, count: int, page_tokens: int, kv_heads: int, head_dim: int) -> Pages:
    """A cache of `count` pages in device memory of count * page_bytes() bytes."""
    if _tensor(data):
        _fits("pages", data, "uint8", data.numel() >= count * page_bytes(head_dim, kv_heads, page_tokens), data.is_contiguous())
    return Pages(eb.ptr(data), count, page_tokens, kv_heads, head_dim)


def _type(t) -> int:
    return TYPES[t] if isinstance(t, str) else t


def plan_request(cached, fresh, table, table_width, free_pages, pages, free_count, free_left, lengths, query_begin, key_begin, slots, positions,
                 shortage, requests, page_tokens, token_capacity, table_stride=None) -> PlanRequest:
    """lengths may be cached and free_left free_count: a step in place."""
    at, stride = _table(table, table_stride, requests, table_width)
    return PlanRequest(_array("cached", cached, requests), _array("fresh", fresh, requests), at, _array("free_pages", free_pages, pages),
                       _array("free_count", free_count, 1), _array("free_left", free_left, 1), _array("lengths", lengths, requests),
                       _array("query_begin", query_begin, requests + 1), _array("key_begin", key_begin, requests + 1),
                       _array("slots", slots, token_capacity, "int64"), _array("positions", positions, token_capacity), _array("shortage", shortage, 1),
                       stride, requests, table_width, pages, page_tokens, token_capacity)


def store_request(cache: Pages, k, v, type, slots, tokens, k_strides=None, v_strides=None) -> StoreRequest:
    h, d, t = cache.kv_heads, cache.head_dim, _type(type)
    return StoreRequest(cache, eb.ptr(k), eb.ptr(v), _array("slots", slots, tokens, "int64"), *_rows("k", k, k_strides, t, tokens, h, d),
                        *_rows("v", v, v_strides, t, tokens, h, d), tokens, t)


def load_request(cache: Pages, k, v, type, table, table_width, lengths, row_begin, requests, rows, first=None, table_stride=None, k_strides=None,
                 v_strides=None) -> LoadRequest:
    h, d, t = cache.kv_heads, cache.head_dim, _type(type)
    at, stride = _table(table, table_stride, requests, table_width)
    return LoadRequest(cache, eb.ptr(k), eb.ptr(v), at, _array("first", first, requests), _array("lengths", lengths, requests),
                       _array("row_begin", row_begin, requests + 1), stride, *_rows("k", k, k_strides, t, rows, h, d),
                       *_rows("v", v, v_strides, t, rows, h, d), requests, table_width, rows, t)


def attend_request(cache: Pages, q, out, type, table, table_width, lengths, requests, heads, queries, query_begin=None, max_queries=1, scale=None,
                   table_stride=None, q_strides=None, out_strides=None) -> AttendRequest:
    d, t = cache.head_dim, _type(type)
    at, stride = _table(table, table_stride, requests, table_width)
    return AttendRequest(cache, eb.ptr(q), eb.ptr(out), at, _array("lengths", lengths, requests), _array("query_begin", query_begin, requests + 1), stride,
                         *_rows("q", q, q_strides, t, queries, heads, d), *_rows("out", out, out_strides, t, queries, heads, d), requests, table_width,
                         heads, queries, max_queries, max(d, 1) ** -0.5 if scale is None else scale, t)


def packed_request(q, k, v, out, type, query_begin, key_begin, requests, heads, kv_heads, head_dim, queries, keys, max_queries=None, causal=True,
                   scale=None, q_strides=None, k_strides=None, v_strides=None, out_strides=None) -> PackedRequest:
    d, t = head_dim, _type(type)
    return PackedRequest(eb.ptr(q), eb.ptr(k), eb.ptr(v), eb.ptr(out), _array("query_begin", query_begin, requests + 1),
                         _array("key_begin", key_begin, requests + 1), *_rows("q", q, q_strides, t, queries, heads, d),
                         *_rows("k", k, k_strides, t, keys, kv_heads, d), *_rows("v", v, v_strides, t, keys, kv_heads, d),
                         *_rows("out", out, out_strides, t, queries, heads, d), requests, heads, kv_heads, head_dim, queries, keys,
                         queries if max_queries is None else max_queries, int(causal), max(head_dim, 1) ** -0.5 if scale is None else scale, t)
