// What the operators on paged K/V caches share: the pages as the kernels take them, the lookup of a
// slot, and the checks of a cortex_kv_pages.
#pragma once

#include "common.h"
#include "cortex_hip.h"

namespace cortex {

constexpr int KV_ERR = 4;  // bit of *err: a malformed page id, length or slot

// The pools of a cortex_kv_pages with the block table of a call.
struct KvPages {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  float* weight;
  int32_t* position;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int32_t* table;
  int64_t ld_table;
  int32_t num_pages, kv_heads, head_dim;
  int32_t shift;      // log2(page_size)
  int64_t max_slots;  // max_pages * page_size

  // page of slot j of sequence b, or -1
  __device__ __forceinline__ int page_of(int64_t b, int64_t j) const {
    if (j < 0 || j >= max_slots) return -1;
    const int p = table[b * ld_table + (j >> shift)];
    return (uint32_t)p < (uint32_t)num_pages ? p : -1;
  }
  __device__ __forceinline__ int row_of(int64_t j) const { return (int)(j & ((1ll << shift) - 1)); }
  // index of a row in the per-row arrays
  __device__ __forceinline__ int64_t scalar_at(int page, int head, int row) const {
    return ((((int64_t)page * kv_heads + head) << shift)) + row;
  }
  // lengths[b] cut to [0, most]; *ok cleared where it had to be
  __device__ __forceinline__ int64_t length_of(const int64_t* lengths, int64_t b, int64_t most, bool* ok) const {
    const int64_t n = lengths[b];
    if (n < 0 || n > most) *ok = false;
    return n < 0 ? 0 : (n > most ? most : n);
  }
};

__device__ __forceinline__ void kv_flag(int32_t* err) {
  if (err) atomicOr(err, KV_ERR);
}

// Checks `pages` and the block table and fills *out; 0 or a negative status.
int kv_check(const char* who, const cortex_kv_pages* pages, int64_t B, const int32_t* table, int64_t ld_table,
             int64_t max_pages, KvPages* out);

// Whether rows of k and v that an operator writes share memory, among themselves or with each other (an expanded pool, the
// same one for both).  Views of whole pools never do: ordered by stride, every dimension steps over all of those before.
// Pools of other strides than each other's are only looked at for themselves.
bool kv_rows_meet(const cortex_kv_pages* pages);

}  // namespace cortex
