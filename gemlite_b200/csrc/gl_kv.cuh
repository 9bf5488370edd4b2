// Shared pieces of the quantised key/value cache: argument checks and the mapping of token rows to sequences and slots.
#pragma once
#include "gl_common.cuh"

// what a kernel needs of gl_kv_args to find a token's slot
struct KvBatch {
  const int32_t* page_table;
  const int32_t* lens;
  const int32_t* q_offsets;
  int64_t pt_stride;
  int32_t batch, max_pages, num_pages, page_size, hkv, n_tokens;
};

static inline KvBatch gl_kv_batch(const gl_kv_args* a) {
  return KvBatch{a->page_table, a->lens, a->q_offsets, a->page_table_stride, a->batch, a->max_pages, a->num_pages, a->page_size, a->n_kv_heads, a->n_tokens};
}
static inline int gl_kv_row_bytes(const gl_kv_args* a) { return a->format == GL_KV_INT4 ? a->head_dim / 2 : a->head_dim; }

// checks that all three entry points share (gl_kv.cu)
int gl_kv_check(const char* fn, const gl_kv_args* a);

#ifdef __CUDACC__
// [first, end) rows of sequence b's new tokens; malformed offsets are cut to the operands' rows
__device__ __forceinline__ void kv_new_rows(const KvBatch& kb, int b, int& first, int& end) {
  if (kb.q_offsets != nullptr) {
    first = min(max(kb.q_offsets[b], 0), kb.n_tokens);
    end = min(max(kb.q_offsets[b + 1], first), kb.n_tokens);
  } else {
    const int t = kb.n_tokens / kb.batch;
    first = b * t;
    end = first + t;
  }
}
// tokens that the cache holds of sequence b before its new ones, and the most that its table has room for
__device__ __forceinline__ int64_t kv_capacity(const KvBatch& kb) { return (int64_t)kb.max_pages * kb.page_size; }
__device__ __forceinline__ int kv_len(const KvBatch& kb, int b) {
  return (int)min((int64_t)max(kb.lens[b], 0), min(kv_capacity(kb), (int64_t)0x7fffff00));
}
// row of (page, head, place) in the scales; times the row bytes in the codes.  -1: no such slot.
__device__ __forceinline__ int64_t kv_slot(const KvBatch& kb, int b, int head, int64_t pos) {
  const int64_t pi = pos / kb.page_size;
  if (pos < 0 || pi >= kb.max_pages) return -1;
  const int page = kb.page_table[b * kb.pt_stride + pi];
  if ((unsigned)page >= (unsigned)kb.num_pages) return -1;
  return ((int64_t)page * kb.hkv + head) * kb.page_size + (pos - pi * kb.page_size);
}
#endif
