// What the kernels of the paged cache share: the new tokens' sequences, their positions and pages, the status words.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace paged {

// Status words, a cache's own or the device's (see mca_paged_status): {kind and two details of what was refused first, how many were} and
// the four words of a bounded wait (tc_common.cuh).
enum Refusal : int { REFUSED_LENGTHS = 1, REFUSED_PAGE = 2, REFUSED_POSITION = 3, REFUSED_WAIT = 4 };
constexpr int BEING_WRITTEN = -1;      // kind, while the details are
constexpr int WAIT_WORDS = 4;          // where a wait's words begin
static __device__ int* g_fail_words;   // this device's failure words (McaFailWord), or null

// Counted before the first one's place is tried for, and the place is given up before the count is taken (paged_attn.cu): what another
// stream refuses while the words are read is found by this reading or the next.
static __device__ __noinline__ void refuse(int* status, int kind, int a, int b) {
  atomicAdd(status + 3, 1);
  __threadfence();
  if (atomicCAS(status, 0, BEING_WRITTEN) == 0) {
    status[1] = a;
    status[2] = b;
    __threadfence();
    atomicExch(status, kind);
  }
  __threadfence();
  mca_raise_fail_word(g_fail_words, MCA_FAIL_PAGED);
}

struct Batch {
  const int* starts;
  const int* lengths;
  const int* table;
  int* status;
  int table_stride, n_seqs, n_tokens, max_new, max_len, n_pages, page_shift;
};

struct Sequence {
  int start, count, length;
  bool good;
};
__device__ __forceinline__ Sequence sequence(const Batch& t, int b) {
  Sequence s;
  s.start = t.starts[b];
  s.count = t.starts[b + 1] - s.start;
  s.length = t.lengths[b];
  // a sequence without new tokens may have any length: nothing of it is read
  s.good = s.start >= 0 && s.count >= 0 && s.count <= t.max_new && s.start <= t.n_tokens - s.count &&
           (s.count == 0 || (s.length >= s.count && s.length <= t.max_len));
  return s;
}
// The sequence a token row belongs to: the last one that starts at or before it; -1: none (a row behind the last sequence).
__device__ __forceinline__ int sequence_of(const Batch& t, int row) {
  if (row >= t.starts[t.n_seqs]) return -1;
  int lo = 0, hi = t.n_seqs;   // starts[lo] <= row < starts[hi], once row >= starts[0]
  if (row < t.starts[0]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Host: the checks of the descriptors that all calls make; fills the kernels' view.
static inline int check(const McaPagedCache* c, const McaPagedBatch* b, Batch* out) {
  if (!c || !b || !c->k_pages || !c->v_pages || !b->starts || !b->lengths || !b->page_table) return ERROR_PARAM_NULL;
  if (c->dtype != MCA_DTYPE_F32 && c->dtype != MCA_DTYPE_BF16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  if (!mca_decode_head_size_supported(c->head_size)) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  if (c->n_pages <= 0 || c->n_heads <= 0 || c->n_kv_heads <= 0 || c->n_heads % c->n_kv_heads != 0 || c->n_heads > 65535) return ERROR_PARAM_OUT_OF_RANGE;
  if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)) != 0) return ERROR_PARAM_OUT_OF_RANGE;
  const int vec = c->dtype == MCA_DTYPE_BF16 ? 8 : 4;
  if (c->page_stride % vec != 0 || c->page_stride < (int64_t)c->page_size * c->n_kv_heads * c->head_size) return ERROR_PARAM_OUT_OF_RANGE;
  if ((((uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 15) != 0) return ERROR_PARAM_OUT_OF_RANGE;
  if (((uintptr_t)c->status & 15) != 0) return ERROR_PARAM_OUT_OF_RANGE;
  if ((((uintptr_t)b->starts | (uintptr_t)b->lengths | (uintptr_t)b->page_table) & 3) != 0) return ERROR_PARAM_OUT_OF_RANGE;
  if (b->n_seqs <= 0 || b->n_seqs > 65535 || b->n_tokens < 0 || b->max_new <= 0 || b->max_len <= 0 || b->table_stride <= 0) return ERROR_PARAM_OUT_OF_RANGE;
  if (b->max_len > (int64_t)b->table_stride * c->page_size || b->max_len > (1 << 30) || b->n_tokens > (1 << 30)) return ERROR_PARAM_OUT_OF_RANGE;
  out->starts = b->starts; out->lengths = b->lengths; out->table = b->page_table; out->status = c->status;
  out->table_stride = b->table_stride; out->n_seqs = b->n_seqs; out->n_tokens = b->n_tokens;
  out->max_new = b->max_new; out->max_len = b->max_len; out->n_pages = c->n_pages;
  out->page_shift = 0;
  while ((1 << out->page_shift) < c->page_size) ++out->page_shift;
  return 0;
}
// Host: the words that a call records in: those of its cache, or the current device's.
static inline int find_status(int** status) { return *status != nullptr ? 0 : mca_paged_device_status(status); }
// Host: a view whose rows are read and written as 16-byte vectors.
static inline int check_heads(const McaHeads* h, int dtype, bool batched) {
  if (!h || !h->data) return ERROR_PARAM_NULL;
  const int vec = dtype == MCA_DTYPE_BF16 ? 8 : 4;
  if (((uintptr_t)h->data & 15) != 0 || h->stride_t % vec != 0 || h->stride_h % vec != 0 || (batched && h->stride_b % vec != 0)) return ERROR_PARAM_OUT_OF_RANGE;
  return 0;
}

}  // namespace paged
