// Attention over a paged cache (pg_attention, pg_attention_ex in include/ptxgen_b200.h): the checks of
// arguments, and which kernel takes a batch.
#include "attention_any.cuh"

namespace {

int check(const char *what, const pg_attention_args *p, int size) {
  if (p->batch < 0 || p->queries < 0 || p->heads < 1 || p->group < 1 || p->dim < 1 ||
      p->page_size < 1 || p->pages < 1 || p->width < 1 || p->slot_rows < (p->batch > 0))
    return pg::argument_fail("%s: batch %d, queries %d, heads %d, group %d, dim %d, page_size %d, "
                             "pages %d, width %d, slot_rows %d: out of range", what, p->batch,
                             p->queries, p->heads, p->group, p->dim, p->page_size, p->pages,
                             p->width, p->slot_rows);
  if (p->dim > PG_ATTENTION_DIM || p->dim * size % 16)
    return pg::argument_fail("%s: head size %d of %d-byte elements: want a multiple of 16 bytes "
                             "and at most %d", what, p->dim, size, PG_ATTENTION_DIM);
  if (static_cast<int64_t>(p->page_size) * p->width > INT32_MAX / 2 || p->heads > 65535 ||
      static_cast<int64_t>(p->queries) * p->group > INT32_MAX / 2)
    return pg::argument_fail("%s: %d pages of %d keys, %d kv heads or %d queries of %d heads: too "
                             "many", what, p->width, p->page_size, p->heads, p->queries, p->group);
  if (p->window < 0 || p->sinks < 0 || p->max_len < 0 || !(p->scale == p->scale))
    return pg::argument_fail("%s: window %d, sinks %d, max_len %d, scale %g", what, p->window,
                             p->sinks, p->max_len, p->scale);
  if (!p->starts && p->queries != p->batch)
    return pg::argument_fail("%s: %d queries for %d sequences and no starts", what, p->queries,
                             p->batch);
  if (!p->batch || !p->queries) return PG_OK;
  if (!p->q || !p->k || !p->v || !p->out || !p->table || !p->lens || !p->workspace)
    return pg::argument_fail("%s: null pointer", what);
  if ((p->q | p->k | p->v |
       static_cast<uint64_t>(p->q_token | p->q_head | p->k_page | p->k_head | p->v_page |
                             p->v_head)) & 15)
    return pg::argument_fail("%s: q, k, v and their strides must be multiples of 16 bytes", what);
  if ((p->out | static_cast<uint64_t>(p->out_token | p->out_head)) & 15)
    return pg::argument_fail("%s: out and its strides must be multiples of 16 bytes", what);
  if ((p->starts | p->slots | p->table | p->lens) & 3 || p->workspace & 255)
    return pg::argument_fail("%s: starts, slots, table and lens must be 4-byte aligned and the "
                             "workspace 256-byte aligned", what);
  if (p->workspace_bytes < PG_ATTENTION_WORKSPACE)
    return pg::argument_fail("%s: a workspace of %lld bytes, want %d", what,
                             static_cast<long long>(p->workspace_bytes), PG_ATTENTION_WORKSPACE);
  return PG_OK;
}

int check_more(const char *what, const pg_attention_args *p, const pg_attention_more *m) {
  if (!m->k_scale != !m->v_scale)
    return pg::argument_fail("%s: the keys have scales and the values have none, or the reverse", what);
  if (m->k_scale && p->dim % 16)
    return pg::argument_fail("%s: head size %d of a cache in 8 bits: want a multiple of 16", what,
                             p->dim);
  if ((m->k_scale | m->v_scale |
       static_cast<uint64_t>(m->k_scale_page | m->k_scale_head | m->v_scale_page |
                             m->v_scale_head)) & 3)
    return pg::argument_fail("%s: scales and their strides must be multiples of 4 bytes", what);
  if (m->mask & 7) return pg::argument_fail("%s: mask must be 8-byte aligned", what);
  if (m->mask && !p->starts)
    return pg::argument_fail("%s: a tree of tokens has no starts", what);
  return PG_OK;
}

int attend(const char *what, const pg_attention_args *p, const pg_attention_more *m,
           uint64_t stream) {
  if (!p) return pg::argument_fail("%s: null arguments", what);
  const int dtype = p->dtype;
  if (dtype != PG_DT_F32 && dtype != PG_DT_BF16 && dtype != PG_DT_F16)
    return pg::argument_fail("%s: dtype %d, want f32, bf16 or f16", what, dtype);
  int rc = check(what, p, dtype == PG_DT_F32 ? 4 : 2);
  if (!rc && m) rc = check_more(what, p, m);
  if (rc || !p->batch || !p->queries) return rc;
  int sms;
  if ((rc = pg::sm_count(&sms))) return rc;
  const auto ptr = [](uint64_t x) { return reinterpret_cast<char *>(static_cast<uintptr_t>(x)); };
  Attention a = {};
  a.q = ptr(p->q), a.k = ptr(p->k), a.v = ptr(p->v), a.out = ptr(p->out);
  a.starts = reinterpret_cast<int *>(ptr(p->starts));
  a.slots = reinterpret_cast<int *>(ptr(p->slots));
  a.table = reinterpret_cast<int *>(ptr(p->table));
  a.lens = reinterpret_cast<int *>(ptr(p->lens));
  a.status = reinterpret_cast<unsigned *>(ptr(p->workspace));
  a.arrived = a.status + 64;
  a.partial = reinterpret_cast<float *>(a.arrived + pg::kCounters);
  a.q_token = p->q_token, a.q_head = p->q_head;
  a.out_token = p->out_token, a.out_head = p->out_head;
  a.k_page = p->k_page, a.k_head = p->k_head, a.v_page = p->v_page, a.v_head = p->v_head;
  a.table_row = p->table_stride;
  a.batch = p->batch, a.queries = p->queries, a.heads = p->heads, a.group = p->group;
  a.dim = p->dim, a.page_size = p->page_size, a.pages = p->pages, a.width = p->width;
  a.slot_rows = p->slot_rows, a.sinks = p->sinks;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  // 2^32 (2^l / d - 1) rounded up, with the smallest l that makes 2^l d or more: exact below 2^31
  while (1ll << a.page_shift < a.page_size) ++a.page_shift;
  a.page_mul = static_cast<uint32_t>(
      ((1ull << 32) * ((1ull << a.page_shift) - a.page_size)) / a.page_size + 1);
  if (m) {
    a.k_scale = ptr(m->k_scale), a.v_scale = ptr(m->v_scale);
    a.ks_page = m->k_scale_page, a.ks_head = m->k_scale_head;
    a.vs_page = m->v_scale_page, a.vs_head = m->v_scale_head;
    a.mask = reinterpret_cast<const uint64_t *>(ptr(m->mask));
  }
  const int64_t most = static_cast<int64_t>(p->width) * p->page_size;
  // A window that the longest sequence fits in hides nothing. Positions less a smaller one stay in 32
  // bits, those of queries before a sequence's start too.
  a.window = p->window >= most ? 0 : p->window;
  const int max_len = static_cast<int>(p->max_len && p->max_len < most ? p->max_len : most);
  const int64_t partial_bytes = p->workspace_bytes - 256 - pg::kCounters * 4ll;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(stream));
  const bool f32 = dtype == PG_DT_F32, bf16 = dtype == PG_DT_BF16;
  const bool counts = a.dim <= 128 && pg::decode_counts(a, static_cast<int>(most));
  // as in decode_takes: rows that tiles of 128 are worth while for
  const bool tiles = a.starts && a.dim <= 128 && !f32 && a.scale_log2 != 0.0f &&
                     static_cast<int64_t>(a.queries) * a.group > 48ll * a.batch;
  if (a.k_scale && tiles) return pg::prompt_8bit(a, bf16, max_len, partial_bytes, sms, s);
  if (a.mask) {
    if (tiles) return pg::prompt_tree(a, bf16, max_len, partial_bytes, sms, s);
    return counts ? pg::decode_tree(a, dtype, sms, s)
                  : pg::any_rows_tree(a, dtype, max_len, partial_bytes, sms, s);
  }
  if (a.k_scale)
    return counts ? pg::decode_8bit(a, dtype, sms, s)
                  : pg::any_rows_8bit(a, dtype, max_len, partial_bytes, sms, s);
  if (a.dim <= 128) {
    if (pg::decode_takes(a, f32, static_cast<int>(most), max_len))
      return pg::decode(a, dtype, sms, s);
    // which masks a score before it is scaled, and 0 times a masked one's -inf is NaN
    if (a.starts && !f32 && a.scale_log2 != 0.0f)
      return pg::prompt_16bit(a, bf16, max_len, partial_bytes, sms, s);
  }
  if (f32) return run<float, float, 64, false>(a, max_len, partial_bytes, sms, s);
  if (bf16)
    return run<__nv_bfloat16, __nv_bfloat16, 64, false>(a, max_len, partial_bytes, sms, s);
  return run<__half, __half, 64, false>(a, max_len, partial_bytes, sms, s);
}

}  // namespace

extern "C" int pg_attention(const pg_attention_args *p, uint64_t stream) {
  return attend("pg_attention", p, nullptr, stream);
}

extern "C" int pg_attention_ex(const pg_attention_args *p, const pg_attention_more *more,
                               uint64_t stream) {
  return attend("pg_attention_ex", p, more, stream);
}
