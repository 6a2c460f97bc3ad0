// The paged key/value cache of sc_kv_pages on the device: where a slot's keys and values are, a sequence's length as
// the kernels take it, and the host's checks shared by the entry points that read the cache.
#pragma once

#include "common.cuh"

namespace sc {

struct Pages {
  const char *k, *v;  // byte strides below
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lengths;
  int pool_pages, max_pages, shift;  // page = 1 << shift
};

inline Pages pages_of(const sc_kv_pages& c) {
  Pages p{};
  p.k = static_cast<const char*>(c.k);
  p.v = static_cast<const char*>(c.v);
  p.k_page = 2 * c.k_page, p.k_token = 2 * c.k_token, p.k_head = 2 * c.k_head;
  p.v_page = 2 * c.v_page, p.v_token = 2 * c.v_token, p.v_head = 2 * c.v_head;
  p.table = c.table, p.table_row = c.table_row, p.lengths = c.lengths;
  p.pool_pages = c.pool_pages, p.max_pages = c.max_pages;
  while ((1 << p.shift) < c.page) ++p.shift;
  return p;
}

// the sequence's length, held to what its row of the table can name
__device__ __forceinline__ int length_of(const Pages& p, int b, int* err) {
  const int n = p.lengths[b], most = p.max_pages << p.shift;
  if (n >= 0 && n <= most) return n;
  record_error(err, SC_ERR_PAGE);
  return n < 0 ? 0 : most;
}

// the page of slot s of sequence b, -1 (recorded) when the table names one outside the pool
__device__ __forceinline__ int page_of(const Pages& p, int b, int s, int* err) {
  const int id = p.table[b * p.table_row + (s >> p.shift)];
  if (unsigned(id) < unsigned(p.pool_pages)) return id;
  record_error(err, SC_ERR_PAGE);
  return -1;
}

inline int check_pages(const sc_kv_pages* c) {
  if (!c || !c->k || !c->v || c->batch < 0 || (c->batch && (!c->table || !c->lengths))) return SC_ERR_ARG;
  if (c->dtype != SC_F16 && c->dtype != SC_BF16) return SC_ERR_DTYPE;
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8 || c->kv_heads < 1 || c->pool_pages < 1 ||
      c->max_pages < 1 || c->page < 1 || c->page > 4096 || (c->page & (c->page - 1)) ||
      int64_t(c->max_pages) * c->page > (int64_t(1) << 30) || c->batch > 65535)
    return SC_ERR_SHAPE;
  const int64_t strides = used(c->pool_pages, c->k_page | c->v_page) | used(c->page, c->k_token | c->v_token) |
                          used(c->kv_heads, c->k_head | c->v_head);
  if ((strides & 7) || ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15))
    return SC_ERR_ALIGN;
  return SC_OK;
}

}  // namespace sc
