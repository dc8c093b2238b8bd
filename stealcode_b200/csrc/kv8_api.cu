// kv8_api.cu -- the C entry points of the paged 8-bit key/value cache
// (sc_kv8_* in include/stealcode_b200.h): argument checks, then the launchers
// of kv8_append.cu, kv8_attend.cu and kv8_pages.cu.
#include "kv8.cuh"
#include "sc_kernels.cuh"

using namespace sc;

namespace {

int bad(const char *what) {
  set_error("%s", what);
  return kErrInvalid;
}

bool misaligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; }

int check_cache(const sc_kv8_cache *c) {
  if (!c) return bad("kv8: null cache");
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->table || !c->length || !c->refs || !c->status)
    return bad("kv8: null pointer in the cache");
  if (c->head_dim != 64 && c->head_dim != 128) {
    set_error("kv8: head_dim %d (64 and 128 are supported)", c->head_dim);
    return kErrUnsupported;
  }
  if (c->block != 16 && c->block != 32 && c->block != 64) {
    set_error("kv8: block %d (16, 32 and 64 tokens are supported)", c->block);
    return kErrUnsupported;
  }
  if (c->page < c->block || c->page > 1024 || c->page % c->block) {
    set_error("kv8: page %d has to be a multiple of block %d, at most 1024", c->page, c->block);
    return kErrUnsupported;
  }
  if (c->n_kv_heads < 1 || c->n_kv_heads > 1024) return bad("kv8: n_kv_heads outside 1..1024");
  if (c->n_layers < 1 || c->n_pages < 1 || c->n_seqs < 1 || c->max_pages < 1)
    return bad("kv8: empty cache dimension");
  if (c->n_pages > INT32_MAX / 2 || c->n_seqs > (1 << 20) || c->max_pages * (int64_t)c->page > INT32_MAX / 2 ||
      c->n_seqs > INT32_MAX / c->max_pages || c->max_pages > INT32_MAX / 2)
    return bad("kv8: cache dimension too large (2^30 pages, tokens a sequence; 2^20 sequences; 2^31 table entries)");
  if (c->max_pages * (int64_t)c->page / 16 * c->n_kv_heads > INT32_MAX)  // work units of one sequence
    return bad("kv8: more than 2^35 tokens x kv heads in one sequence");
  if (misaligned(c->k, 16) || misaligned(c->v, 16) || misaligned(c->refs, 16))
    return bad("kv8: k, v and refs have to be 16-byte aligned");
  if (misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4) || misaligned(c->table, 4) || misaligned(c->length, 4) ||
      misaligned(c->status, 4))
    return bad("kv8: misaligned pointer in the cache");
  return kOk;
}

int check_batch(const sc_kv8_cache *c, const sc_kv8_batch *b) {
  if (!b) return bad("kv8: null batch");
  if (b->m < 0 || b->n < 0 || b->total < 0) return bad("kv8: negative batch size");
  if (!b->seqs && b->m > c->n_seqs) return bad("kv8: more sequences than the cache has");
  if (b->m > (1 << 20) || b->n > (1 << 24)) return bad("kv8: batch of more than 2^20 sequences or 2^24 rows each");
  if (b->m * b->n > INT32_MAX) return bad("kv8: m * n above 2^31");
  if (!b->cu && b->total != b->m * b->n) return bad("kv8: total has to be m * n without cu");
  if (misaligned(b->seqs, 4) || misaligned(b->cu, 4)) return bad("kv8: misaligned pointer in the batch");
  return kOk;
}

int check_layer(const sc_kv8_cache *c, int64_t layer) {
  if (layer < 0 || layer >= c->n_layers) return bad("kv8: layer outside the cache");
  return kOk;
}

int dtype_size(int32_t dtype) {
  return dtype == SC_DTYPE_F32 ? 4 : dtype == SC_DTYPE_F16 || dtype == SC_DTYPE_BF16 ? 2 : 0;
}

kv8::Layer layer_of(const sc_kv8_cache *c, int64_t layer) {
  kv8::Layer l;
  const int64_t codes = layer * c->n_pages * c->n_kv_heads * c->page * (int64_t)c->head_dim;
  const int64_t scales = layer * c->n_pages * c->n_kv_heads * (int64_t)(c->page / c->block);
  l.k = c->k + codes;
  l.v = c->v + codes;
  l.ks = c->k_scale + scales;
  l.vs = c->v_scale + scales;
  l.table = c->table;
  l.length = c->length;
  l.status = c->status;
  l.n_pages = (int)c->n_pages;
  l.n_seqs = (int)c->n_seqs;
  l.max_pages = (int)c->max_pages;
  l.kv = c->n_kv_heads;
  l.page = c->page;
  l.block = c->block;
  l.block_shift = c->block == 16 ? 4 : c->block == 32 ? 5 : 6;
  const uint32_t d = (uint32_t)c->page / 16;
  l.page_magic = d == 1 ? 0 : (uint32_t)(((1ull << 32) + d - 1) / d);
  return l;
}

kv8::Batch batch_of(const sc_kv8_batch *b) {
  return kv8::Batch{b->seqs, b->cu, (int)b->m, (int)b->n, b->total};
}

kv8::PageArgs pages_of(const sc_kv8_cache *c, void *ws) {
  return kv8::PageArgs{c->k, c->v, c->k_scale, c->v_scale, c->table, c->length, c->refs, c->status, c->n_layers,
                       (int)c->n_pages, (int)c->n_seqs, (int)c->max_pages, c->n_kv_heads, c->head_dim, c->page,
                       c->block, ws};
}

int check_ws(const void *ws, int64_t bytes, size_t need) {
  if (!ws) return bad("kv8: null workspace");
  if (misaligned(ws, 256) || bytes < 0 || (size_t)bytes < need) {
    set_error("kv8: workspace needs %zu bytes at 256-byte alignment", need);
    return kErrInvalid;
  }
  return kOk;
}

int check_seqs(const sc_kv8_cache *c, const int32_t *seqs, int64_t m) {
  if (m < 0) return bad("kv8: negative number of sequences");
  if (m > c->n_seqs) return bad("kv8: more sequences than the cache has");
  if (misaligned(seqs, 4)) return bad("kv8: misaligned sequence ids");
  return kOk;
}

}  // namespace

extern "C" {

int sc_kv8_append(const sc_kv8_cache *c, int64_t layer, const sc_kv8_batch *b, const void *k, int64_t k_row,
                  int64_t k_head, const void *v, int64_t v_row, int64_t v_head, int32_t dtype, void *stream) {
  int rc = check_cache(c);
  if (!rc) rc = check_batch(c, b);
  if (!rc) rc = check_layer(c, layer);
  if (rc) return rc;
  const int size = dtype_size(dtype);
  if (!size) return bad("kv8_append: unknown dtype");
  if (b->m == 0 || b->n == 0 || b->total == 0) return kOk;
  if (!k || !v) return bad("kv8_append: null pointer");
  if (misaligned(k, size) || misaligned(v, size)) return bad("kv8_append: misaligned rows");
  kv8::AppendArgs a{layer_of(c, layer), batch_of(b), k, v, k_row, k_head, v_row, v_head, dtype, c->head_dim};
  return kv8::append(a, (cudaStream_t)stream);
}

int sc_kv8_rows(const sc_kv8_cache *c, int64_t layer, const sc_kv8_batch *b, void *k, void *v, int32_t dtype,
                void *stream) {
  int rc = check_cache(c);
  if (!rc) rc = check_batch(c, b);
  if (!rc) rc = check_layer(c, layer);
  if (rc) return rc;
  const int size = dtype_size(dtype);
  if (!size) return bad("kv8_rows: unknown dtype");
  if (b->m == 0 || b->n == 0 || b->total == 0 || (!k && !v)) return kOk;
  if (misaligned(k, 16) || misaligned(v, 16)) return bad("kv8_rows: outputs have to be 16-byte aligned");
  kv8::RowsArgs a{layer_of(c, layer), batch_of(b), k, v, dtype, c->head_dim};
  return kv8::read_rows(a, (cudaStream_t)stream);
}

int64_t sc_kv8_attend_workspace_bytes(void) {
  int dev, sms;
  const int rc = current_device(&dev, &sms);
  if (rc) return rc;
  return (int64_t)kv8::attend_ws_bytes(sms);
}

int sc_kv8_attend(const sc_kv8_cache *c, int64_t layer, const sc_kv8_batch *b, const void *q, int64_t q_row,
                  int64_t q_head, int32_t n_heads, float scale, int64_t window, int64_t sinks, int64_t max_len,
                  void *out, int64_t out_row, int64_t out_head, float *lse, int32_t dtype, void *workspace,
                  int64_t workspace_bytes, void *stream) {
  int rc = check_cache(c);
  if (!rc) rc = check_batch(c, b);
  if (!rc) rc = check_layer(c, layer);
  if (rc) return rc;
  const int size = dtype_size(dtype);
  if (!size) return bad("kv8_attend: unknown dtype");
  if (n_heads < 1 || n_heads % c->n_kv_heads) return bad("kv8_attend: n_heads has to be a multiple of n_kv_heads");
  if (n_heads / c->n_kv_heads > 1024) return bad("kv8_attend: more than 1024 query heads to a kv head");
  if (window < 0 || sinks < 0) return bad("kv8_attend: negative window or sinks");
  if (b->m == 0 || b->n == 0 || b->total == 0) return kOk;
  if (!q || !out) return bad("kv8_attend: null pointer");
  if (misaligned(q, size) || misaligned(out, size) || misaligned(lse, 4)) return bad("kv8_attend: misaligned tensor");
  int dev, sms;
  rc = current_device(&dev, &sms);
  if (!rc) rc = check_ws(workspace, workspace_bytes, kv8::attend_ws_bytes(sms));
  if (rc) return rc;
  const int64_t most = c->max_pages * (int64_t)c->page;  // tokens a sequence can hold
  if (max_len <= 0 || max_len > most) max_len = most;
  kv8::AttendArgs a{layer_of(c, layer), batch_of(b), q, out, lse, q_row, q_head, out_row, out_head, dtype,
                    c->head_dim, n_heads, scale, 0, 0, max_len, workspace};
  // a window that no sequence can outgrow hides nothing
  if (window > 0 && window < most) {
    a.window = (int)window;
    a.sinks = (int)(sinks < most ? sinks : most);
  }
  const int64_t group = n_heads / c->n_kv_heads;
  if (b->n * group > INT32_MAX / 2 || b->m * (b->n * group / 8 + 1) > INT32_MAX / 2)
    return bad("kv8_attend: too many query rows");
  return kv8::attend(a, sms, (cudaStream_t)stream);
}

int64_t sc_kv8_page_workspace_bytes(const sc_kv8_cache *c) {
  const int rc = check_cache(c);
  if (rc) return rc;
  return (int64_t)kv8::page_ws_bytes(c->n_pages, c->n_seqs, c->max_pages);
}

static int page_call(const sc_kv8_cache *c, void *ws, int64_t ws_bytes) {
  int rc = check_cache(c);
  if (!rc) rc = check_ws(ws, ws_bytes, kv8::page_ws_bytes(c->n_pages, c->n_seqs, c->max_pages));
  return rc;
}

int sc_kv8_reserve(const sc_kv8_cache *c, const int32_t *seqs, const int32_t *counts, int64_t m, void *workspace,
                   int64_t workspace_bytes, void *stream) {
  int rc = page_call(c, workspace, workspace_bytes);
  if (!rc) rc = check_seqs(c, seqs, m);
  if (rc) return rc;
  if (m == 0) return kOk;
  if (!counts || misaligned(counts, 4)) return bad("kv8_reserve: counts null or misaligned");
  return kv8::reserve(pages_of(c, workspace), seqs, counts, (int)m, (cudaStream_t)stream);
}

int sc_kv8_fork(const sc_kv8_cache *c, const int32_t *parents, const int32_t *children, int64_t m, void *workspace,
                int64_t workspace_bytes, void *stream) {
  int rc = page_call(c, workspace, workspace_bytes);
  if (!rc) rc = check_seqs(c, children, m);
  if (rc) return rc;
  if (m == 0) return kOk;
  if (!parents || !children || misaligned(parents, 4)) return bad("kv8_fork: null or misaligned ids");
  int dev, sms;
  rc = current_device(&dev, &sms);
  if (rc) return rc;
  return kv8::fork(pages_of(c, workspace), parents, children, (int)m, sms, (cudaStream_t)stream);
}

int sc_kv8_release(const sc_kv8_cache *c, const int32_t *seqs, int64_t m, void *stream) {
  int rc = check_cache(c);
  if (!rc) rc = check_seqs(c, seqs, m);
  if (rc || m == 0) return rc;
  return kv8::release(pages_of(c, nullptr), seqs, (int)m, (cudaStream_t)stream);
}

int sc_kv8_slide(const sc_kv8_cache *c, const int32_t *seqs, int64_t m, int64_t window, int64_t sinks, void *stream) {
  int rc = check_cache(c);
  if (!rc) rc = check_seqs(c, seqs, m);
  if (rc) return rc;
  if (window < 1 || sinks < 0) return bad("kv8_slide: window has to be positive, sinks not negative");
  const int64_t most = c->max_pages * (int64_t)c->page;
  if (m == 0 || window >= most) return kOk;  // nothing can lie before the window
  return kv8::slide(pages_of(c, nullptr), seqs, (int)m, (int)window, (int)(sinks < most ? sinks : most),
                    (cudaStream_t)stream);
}

int sc_kv8_compact(const sc_kv8_cache *c, void *workspace, int64_t workspace_bytes, void *stream) {
  int rc = page_call(c, workspace, workspace_bytes);
  if (rc) return rc;
  int dev, sms;
  rc = current_device(&dev, &sms);
  if (rc) return rc;
  return kv8::compact(pages_of(c, workspace), sms, (cudaStream_t)stream);
}

}  // extern "C"
