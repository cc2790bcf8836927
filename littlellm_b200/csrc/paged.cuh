// paged.cuh — the paged KV cache as the kernels see it, and its checks.
#pragma once

#include "ops.cuh"

namespace kb {

// Addressing of a paged cache in a kernel's parameters. Row indexes
// (page * kv_heads + head) * page_size + offset are 64-bit: a cache passes
// 2^32 elements at 256 K rows of 128 values.
struct PagedView {
  const int32_t* table;  // [n_seqs, max_pages]
  int64_t max_pages;
  int64_t n_seqs;
  int n_pages;
  int n_kv_heads;
  int page_shift;
  int capacity;  // max_pages * page_size, <= 2^30
};

// What a token's (position, sequence) pair amounts to.
enum TokenState { kTokenOk = 0, kTokenPadding = 1, kTokenBad = 2 };

// Position and sequence of one token checked against the view; `flag` gets
// the KLLM_B200_FLAG_* bits of a bad one.
__device__ __forceinline__ TokenState token_state(const PagedView& v, int pos, int seq, int& flag) {
  flag = 0;
  if (pos == -1) return kTokenPadding;
  if (pos < 0 || pos >= v.capacity) flag |= KLLM_B200_FLAG_BAD_POSITION;
  if (seq < 0 || seq >= v.n_seqs) flag |= KLLM_B200_FLAG_BAD_SEQ;
  return flag == 0 ? kTokenOk : kTokenBad;
}

__device__ __forceinline__ bool page_ok(const PagedView& v, int page) {
  return static_cast<unsigned>(page) < static_cast<unsigned>(v.n_pages);
}

// Launchers behind the C ABI. Hidden: the descriptor's name in their mangled
// names would pass for entry points of the library.
#pragma GCC visibility push(hidden)

// Checks a cache descriptor (host) and fills the kernel's view.
int paged_view(const kllm_b200_paged_cache* c, const char* what, PagedView* v);

int qkv_norm_rope_kv_append_paged(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                  int64_t v_stride, const void* bq, const void* bk, const void* bv, int bias_dtype,
                                  const void* q_norm, const void* k_norm, int norm_dtype, float eps, float theta,
                                  const int32_t* positions, const int32_t* seqs, int64_t n_tokens, int64_t n_heads,
                                  const kllm_b200_paged_cache* cache, void* q_out, int64_t q_out_stride,
                                  int32_t* err_flags, const LaunchOpts& o);

int kv_read_paged(const kllm_b200_paged_cache* cache, const int32_t* positions, const int32_t* seqs, int64_t n_tokens,
                  const int32_t* out_slots, int64_t n_out_slots, int64_t out_max_seq, void* k_out, void* v_out,
                  int32_t* err_flags, const LaunchOpts& o);

int attention_paged_workspace_bytes(int64_t n_tokens, int64_t n_heads, const kllm_b200_paged_cache* cache,
                                    int64_t* bytes);

int attention_paged(const void* q, int64_t q_stride, const kllm_b200_paged_cache* cache, const int32_t* positions,
                    const int32_t* seqs, int64_t n_tokens, int64_t n_heads, void* out, int64_t out_stride,
                    void* workspace, int64_t workspace_bytes, int32_t* err_flags, const LaunchOpts& o);

#pragma GCC visibility pop

}  // namespace kb
