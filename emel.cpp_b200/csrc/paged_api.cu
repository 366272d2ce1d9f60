// C entry points of include/emelb_paged.h: what a request may be, where its memory lies, the launch.
#include "ctx.h"
#include "paged.h"

using namespace emelb;

namespace {

// what one array of a request covers, in bytes from `p`
struct Span {
  const void* p;
  uint64_t bytes;
};

bool aligned(const void* p, uint64_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
bool apart(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return x <= y ? a.bytes <= y - x : b.bytes <= x - y;
}
uint64_t elem_bytes(int type) { return type == EMELB_F32 ? 4 : type == EMELB_F16 || type == EMELB_BF16 ? 2 : 0; }

// strides between rows, or heads, that keep the address arithmetic inside 64 bits and rows apart from themselves
constexpr int64_t kMostStride = (int64_t)1 << 40;
constexpr int64_t kMostElems = (int64_t)1 << 58;
bool strides_ok(int64_t token, int64_t head, int64_t row, int tokens, int heads) {
  if (token < 0 || head < 0 || token > kMostStride || head > kMostStride) return false;
  if (tokens > 1 && token > kMostElems / (tokens - 1)) return false;   // heads, at most 2^16 of them, stay below 2^56
  return (tokens == 1 || token >= row) && (heads == 1 || head >= row);
}
// results may not fall on one another: one of the two strides steps over all of the other's
bool distinct_rows(int64_t token, int64_t head, int64_t row, int64_t tokens, int64_t heads) {
  if (tokens == 1 || heads == 1) return true;
  return token >= (heads - 1) * head + row || head >= (tokens - 1) * token + row;
}
Span rows_span(const void* p, int64_t token, int64_t head, int64_t row, int64_t tokens, int64_t heads, uint64_t size) {
  return Span{p, (uint64_t)((tokens - 1) * token + (heads - 1) * head + row) * size};
}
bool table_ok(int64_t stride, int64_t rows, int64_t width) { return stride >= width && stride <= kMostStride && stride <= kMostElems / rows; }
Span table_span(const int32_t* p, int64_t stride, int64_t rows, int64_t width) { return Span{p, (uint64_t)((rows - 1) * stride + width) * 4}; }

// a page's sizes: invalid, known but not taken, or fine
uint32_t sizes_ok(int32_t head_dim, int32_t kv_heads, int32_t page_tokens) {
  if (head_dim <= 0 || kv_heads <= 0 || page_tokens <= 0) return EMELB_INVALID_REQUEST;
  if (head_dim % 32 != 0 || head_dim > 128 || kv_heads > 65535) return EMELB_UNSUPPORTED_OP;
  if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)) != 0) return EMELB_UNSUPPORTED_OP;
  return EMELB_OK;
}
uint32_t cache_ok(const emelb_kv_pages& c) {
  if (!aligned(c.data, 16) || c.pages <= 0) return EMELB_INVALID_REQUEST;
  return sizes_ok(c.head_dim, c.kv_heads, c.page_tokens);
}
Span cache_span(const emelb_kv_pages& c) {
  return Span{c.data, (uint64_t)c.pages * emelb_kv_page_bytes(c.head_dim, c.kv_heads, c.page_tokens)};
}

// memory of the context's GPU
bool here(const emelb_ctx* c, const void* p) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  auto it = c->dev_ranges.upper_bound(a);
  if (it != c->dev_ranges.begin() && a < std::prev(it)->first + std::prev(it)->second) return true;
  cudaPointerAttributes at{};
  if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == c->device);
}

uint32_t refuse(emelb_ctx* c, uint32_t why) {
  c->diag.rejected_dispatch_calls += 1;
  return why;
}

// the call behind a guard that passed
template <class Launch>
uint32_t dispatch(emelb_ctx* c, std::initializer_list<const void*> arrays, uint64_t launches, Launch&& launch) {
  for (const void* p : arrays)
    if (p && !here(c, p)) return refuse(c, EMELB_INVALID_REQUEST);
  cudaSetDevice(c->device);
  const cudaError_t e = launch();
  if (e != cudaSuccess) {
    c->last_cuda_error = (int)e;
    cudaGetLastError();
    return EMELB_INTERNAL_ERROR;
  }
  c->diag.kernel_launches += launches;
  return EMELB_OK;
}

}  // namespace

extern "C" {

uint64_t emelb_kv_page_bytes(int32_t head_dim, int32_t kv_heads, int32_t page_tokens) {
  if (sizes_ok(head_dim, kv_heads, page_tokens) != EMELB_OK) return 0;
  return (uint64_t)kv_heads * (page_tokens / 16) * 18 * head_dim;
}

// ------------------------------------------------------------------ plan
uint32_t emelb_kv_plan_can_run(const emelb_kv_plan_request* r) {
  if (!r) return EMELB_INVALID_REQUEST;
  if (r->requests <= 0 || r->table_width <= 0 || r->pages <= 0 || r->page_tokens <= 0 || r->token_capacity <= 0) return EMELB_INVALID_REQUEST;
  if (!table_ok(r->table_stride, r->requests, r->table_width)) return EMELB_INVALID_REQUEST;
  for (const void* p : {(const void*)r->cached, (const void*)r->fresh, (const void*)r->table, (const void*)r->free_pages, (const void*)r->free_count,
                        (const void*)r->free_left, (const void*)r->lengths, (const void*)r->query_begin, (const void*)r->key_begin,
                        (const void*)r->positions, (const void*)r->shortage})
    if (!aligned(p, 4)) return EMELB_INVALID_REQUEST;
  if (!aligned(r->slots, 8)) return EMELB_INVALID_REQUEST;
  const uint64_t n = (uint64_t)r->requests, cap = (uint64_t)r->token_capacity;
  const Span out[] = {table_span(r->table, r->table_stride, r->requests, r->table_width),
                      {r->free_pages, (uint64_t)r->pages * 4},
                      {r->free_left, 4},
                      {r->lengths, n * 4},
                      {r->query_begin, n * 4 + 4},
                      {r->key_begin, n * 4 + 4},
                      {r->slots, cap * 8},
                      {r->positions, cap * 4},
                      {r->shortage, 4}};
  const Span cached{r->cached, n * 4}, fresh{r->fresh, n * 4}, count{r->free_count, 4};
  const int outs = (int)(sizeof(out) / sizeof(out[0]));
  for (int i = 0; i < outs; ++i) {
    for (int j = i + 1; j < outs; ++j)
      if (!apart(out[i], out[j])) return EMELB_INVALID_REQUEST;
    const bool same_lengths = out[i].p == r->lengths && r->lengths == r->cached;
    const bool same_count = out[i].p == r->free_left && r->free_left == r->free_count;
    if (!apart(out[i], fresh) || (!same_lengths && !apart(out[i], cached)) || (!same_count && !apart(out[i], count))) return EMELB_INVALID_REQUEST;
  }
  if (r->requests > EMELB_KV_MAX_REQUESTS) return EMELB_UNSUPPORTED_OP;
  if (r->page_tokens < 16 || r->page_tokens > 256 || (r->page_tokens & (r->page_tokens - 1)) != 0) return EMELB_UNSUPPORTED_OP;
  return EMELB_OK;
}

uint32_t emelb_kv_plan(emelb_ctx* c, const emelb_kv_plan_request* r) {
  if (!c || !r) return EMELB_INVALID_REQUEST;
  if (const uint32_t why = emelb_kv_plan_can_run(r)) return refuse(c, why);
  int launches = 0;
  const uint32_t err = dispatch(c, {r->cached, r->fresh, r->table, r->free_pages, r->free_count, r->free_left, r->lengths, r->query_begin, r->key_begin,
                                    r->slots, r->positions, r->shortage}, 0,
                                [&] { return launch_kv_plan(*r, reinterpret_cast<int*>(c->fa_part_ml), c->sm_count, &launches, c->bad_word(), c->pdl & 1, c->stream); });
  c->diag.kernel_launches += launches;
  return err;
}

// ------------------------------------------------------------------ store, load
uint32_t emelb_kv_store_can_run(const emelb_kv_store_request* r) {
  if (!r || r->tokens <= 0) return EMELB_INVALID_REQUEST;
  if (const uint32_t why = cache_ok(r->cache)) return why;
  const uint64_t size = elem_bytes(r->type);
  if (size == 0) return EMELB_UNSUPPORTED_OP;
  const int D = r->cache.head_dim, H = r->cache.kv_heads;
  if (!aligned(r->k, size) || !aligned(r->v, size) || !aligned(r->slots, 8)) return EMELB_INVALID_REQUEST;
  if (!strides_ok(r->k_token_stride, r->k_head_stride, D, r->tokens, H) || !strides_ok(r->v_token_stride, r->v_head_stride, D, r->tokens, H))
    return EMELB_INVALID_REQUEST;
  const Span cache = cache_span(r->cache);
  if (!apart(cache, rows_span(r->k, r->k_token_stride, r->k_head_stride, D, r->tokens, H, size)) ||
      !apart(cache, rows_span(r->v, r->v_token_stride, r->v_head_stride, D, r->tokens, H, size)) ||
      !apart(cache, Span{r->slots, (uint64_t)r->tokens * 8}))
    return EMELB_INVALID_REQUEST;
  if (r->tokens > 0x7ffffff0 || ((int64_t)r->tokens + 15) / 16 * H > 0x3fffffff) return EMELB_UNSUPPORTED_OP;   // places in a last tile, CTAs
  return EMELB_OK;
}

uint32_t emelb_kv_store(emelb_ctx* c, const emelb_kv_store_request* r) {
  if (!c || !r) return EMELB_INVALID_REQUEST;
  if (const uint32_t why = emelb_kv_store_can_run(r)) return refuse(c, why);
  return dispatch(c, {r->cache.data, r->k, r->v, r->slots}, 1, [&] { return launch_kv_store(*r, c->sm_count, c->bad_word(), c->pdl & 1, c->stream); });
}

uint32_t emelb_kv_load_can_run(const emelb_kv_load_request* r) {
  if (!r || r->requests <= 0 || r->table_width <= 0 || r->rows <= 0 || !table_ok(r->table_stride, r->requests, r->table_width))
    return EMELB_INVALID_REQUEST;
  if (const uint32_t why = cache_ok(r->cache)) return why;
  const uint64_t size = elem_bytes(r->type);
  if (size == 0) return EMELB_UNSUPPORTED_OP;
  const int D = r->cache.head_dim, H = r->cache.kv_heads;
  if (!aligned(r->k, size) || !aligned(r->v, size) || !aligned(r->table, 4) || !aligned(r->lengths, 4) || !aligned(r->row_begin, 4) ||
      (r->first && !aligned(r->first, 4)))
    return EMELB_INVALID_REQUEST;
  if (!strides_ok(r->k_token_stride, r->k_head_stride, D, r->rows, H) || !strides_ok(r->v_token_stride, r->v_head_stride, D, r->rows, H) ||
      !distinct_rows(r->k_token_stride, r->k_head_stride, D, r->rows, H) || !distinct_rows(r->v_token_stride, r->v_head_stride, D, r->rows, H))
    return EMELB_INVALID_REQUEST;
  const uint64_t n = (uint64_t)r->requests;
  const Span k = rows_span(r->k, r->k_token_stride, r->k_head_stride, D, r->rows, H, size);
  const Span v = rows_span(r->v, r->v_token_stride, r->v_head_stride, D, r->rows, H, size);
  const Span in[] = {cache_span(r->cache), table_span(r->table, r->table_stride, r->requests, r->table_width), {r->lengths, n * 4},
                     {r->row_begin, n * 4 + 4}, {r->first, r->first ? n * 4 : 0}};
  for (const Span& s : in)
    if (s.bytes && (!apart(s, k) || !apart(s, v))) return EMELB_INVALID_REQUEST;
  // keys and values may share the rows of one buffer, each in columns of its own
  if (!apart(k, v)) {
    const int64_t off = (static_cast<const char*>(r->v) - static_cast<const char*>(r->k)) / (int64_t)size;
    const int64_t step = r->k_token_stride, row = (H - 1) * r->k_head_stride + D, from = off < 0 ? off + step : off;
    if (r->rows == 1 || r->v_token_stride != step || r->v_head_stride != r->k_head_stride || from < row || from > step - row) return EMELB_INVALID_REQUEST;
  }
  if (((int64_t)r->rows / 16 + (int64_t)r->requests * 2) * H > 0x3fffffff) return EMELB_UNSUPPORTED_OP;   // CTAs
  return EMELB_OK;
}

uint32_t emelb_kv_load(emelb_ctx* c, const emelb_kv_load_request* r) {
  if (!c || !r) return EMELB_INVALID_REQUEST;
  if (const uint32_t why = emelb_kv_load_can_run(r)) return refuse(c, why);
  return dispatch(c, {r->cache.data, r->k, r->v, r->table, r->first, r->lengths, r->row_begin}, 1,
                  [&] { return launch_kv_load(*r, c->sm_count, c->bad_word(), c->pdl & 1, c->stream); });
}

// ------------------------------------------------------------------ attend
uint32_t emelb_kv_attend_can_run(const emelb_kv_attend_request* r) {
  if (!r || r->requests <= 0 || r->table_width <= 0 || r->heads <= 0 || r->queries <= 0 || r->max_queries <= 0 ||
      !table_ok(r->table_stride, r->requests, r->table_width))
    return EMELB_INVALID_REQUEST;
  if (const uint32_t why = cache_ok(r->cache)) return why;
  const uint64_t size = elem_bytes(r->type);
  if (size == 0) return EMELB_UNSUPPORTED_OP;
  const int D = r->cache.head_dim;
  if (r->heads % r->cache.kv_heads != 0 || !(r->scale > 0.0f && r->scale < 0x1p127f)) return EMELB_INVALID_REQUEST;
  if (!r->query_begin && r->queries < r->requests) return EMELB_INVALID_REQUEST;
  if (!aligned(r->q, size) || !aligned(r->out, size) || !aligned(r->table, 4) || !aligned(r->lengths, 4) || (r->query_begin && !aligned(r->query_begin, 4)))
    return EMELB_INVALID_REQUEST;
  if (!strides_ok(r->q_token_stride, r->q_head_stride, D, r->queries, r->heads) || !strides_ok(r->out_token_stride, r->out_head_stride, D, r->queries, r->heads) ||
      !distinct_rows(r->out_token_stride, r->out_head_stride, D, r->queries, r->heads))
    return EMELB_INVALID_REQUEST;
  const uint64_t n = (uint64_t)r->requests;
  const Span out = rows_span(r->out, r->out_token_stride, r->out_head_stride, D, r->queries, r->heads, size);
  const Span in[] = {cache_span(r->cache), rows_span(r->q, r->q_token_stride, r->q_head_stride, D, r->queries, r->heads, size),
                     table_span(r->table, r->table_stride, r->requests, r->table_width), {r->lengths, n * 4},
                     {r->query_begin, r->query_begin ? n * 4 + 4 : 0}};
  for (const Span& s : in)
    if (s.bytes && !apart(s, out)) return EMELB_INVALID_REQUEST;
  if (r->requests > EMELB_KV_MAX_REQUESTS || r->heads / r->cache.kv_heads > 64 || (int64_t)r->heads * r->max_queries > 0x3fffffff)
    return EMELB_UNSUPPORTED_OP;
  return EMELB_OK;
}

uint32_t emelb_kv_attend(emelb_ctx* c, const emelb_kv_attend_request* r) {
  if (!c || !r) return EMELB_INVALID_REQUEST;
  if (const uint32_t why = emelb_kv_attend_can_run(r)) return refuse(c, why);
  const KvAttendScratch s{c->fa_part_acc, kFlashPartFloats, c->fa_part_ml, kFlashPartFloats / 32, c->grp_cnt, c->grp_cnt_ints};
  return dispatch(c, {r->cache.data, r->q, r->out, r->table, r->lengths, r->query_begin}, 1,
                  [&] { return launch_kv_attend(*r, s, c->sm_count, c->bad_word(), c->pdl & 1, c->stream); });
}

// ------------------------------------------------------------------ packed prompts
uint32_t emelb_attend_packed_can_run(const emelb_attend_packed_request* r) {
  if (!r || r->requests <= 0 || r->heads <= 0 || r->kv_heads <= 0 || r->head_dim <= 0 || r->queries <= 0 || r->keys < 0 || r->max_queries <= 0)
    return EMELB_INVALID_REQUEST;
  if (r->heads % r->kv_heads != 0 || !(r->scale > 0.0f && r->scale < 0x1p127f)) return EMELB_INVALID_REQUEST;
  const uint64_t size = elem_bytes(r->type);
  if (size != 2) return EMELB_UNSUPPORTED_OP;
  const int D = r->head_dim, keys = r->keys > 0 ? r->keys : 1;
  if (!aligned(r->q, size) || !aligned(r->k, size) || !aligned(r->v, size) || !aligned(r->out, size) || !aligned(r->query_begin, 4) ||
      !aligned(r->key_begin, 4))
    return EMELB_INVALID_REQUEST;
  if (!strides_ok(r->q_token_stride, r->q_head_stride, D, r->queries, r->heads) || !strides_ok(r->k_token_stride, r->k_head_stride, D, keys, r->kv_heads) ||
      !strides_ok(r->v_token_stride, r->v_head_stride, D, keys, r->kv_heads) ||
      !strides_ok(r->out_token_stride, r->out_head_stride, D, r->queries, r->heads) ||
      !distinct_rows(r->out_token_stride, r->out_head_stride, D, r->queries, r->heads))
    return EMELB_INVALID_REQUEST;
  const uint64_t n = (uint64_t)r->requests;
  const Span out = rows_span(r->out, r->out_token_stride, r->out_head_stride, D, r->queries, r->heads, size);
  const Span in[] = {rows_span(r->q, r->q_token_stride, r->q_head_stride, D, r->queries, r->heads, size),
                     rows_span(r->k, r->k_token_stride, r->k_head_stride, D, keys, r->kv_heads, size),
                     rows_span(r->v, r->v_token_stride, r->v_head_stride, D, keys, r->kv_heads, size), {r->query_begin, n * 4 + 4}, {r->key_begin, n * 4 + 4}};
  for (const Span& s : in)
    if (!apart(s, out)) return EMELB_INVALID_REQUEST;
  const int group = r->heads / r->kv_heads;
  if (D % 8 != 0 || D > 128 || group > 128 || r->kv_heads > 65535) return EMELB_UNSUPPORTED_OP;
  // a walk that its waits would take for one that hangs, pairs of row tiles that the CTAs count, and strides that a tensor map holds
  if (r->keys > 1 << 25) return EMELB_UNSUPPORTED_OP;
  if (((int64_t)r->queries / (256 / group) + r->requests) * r->kv_heads > 0x3fffffff) return EMELB_UNSUPPORTED_OP;
  for (int64_t s : {r->q_token_stride, r->q_head_stride, r->k_token_stride, r->k_head_stride, r->v_token_stride, r->v_head_stride})
    if (s >= (int64_t)1 << 39) return EMELB_UNSUPPORTED_OP;
  for (const void* p : {r->q, r->k, r->v, (const void*)r->out})
    if (!aligned(p, 16)) return EMELB_UNSUPPORTED_OP;
  for (int64_t s : {r->q_token_stride, r->q_head_stride, r->k_token_stride, r->k_head_stride, r->v_token_stride, r->v_head_stride, r->out_token_stride,
                    r->out_head_stride})
    if (s % 8 != 0) return EMELB_UNSUPPORTED_OP;
  return EMELB_OK;
}

uint32_t emelb_attend_packed(emelb_ctx* c, const emelb_attend_packed_request* r) {
  if (!c || !r) return EMELB_INVALID_REQUEST;
  if (const uint32_t why = emelb_attend_packed_can_run(r)) return refuse(c, why);
  return dispatch(c, {r->q, r->k, r->v, r->out, r->query_begin, r->key_begin}, 1,
                  [&] { return launch_attend_packed(*r, c->next_sched(), c->fa_part_acc, c->sm_count, c->bad_word(), c->status_word(), c->pdl & 1, c->stream); });
}

}  // extern "C"
