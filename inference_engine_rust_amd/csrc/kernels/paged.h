// The paged KV cache (iek_paged_kv): arguments of its launchers (kernels/paged.hip, kernels/paged_attention.hip).
#pragma once
#include "../iek_internal.h"

namespace iek {

// k, v: [n_pages][n_kv][page][hd] of f32 or fp16; entry j of sequence b is slot j % page of page
// table[b * max_pages + j / page]. page = 1 << shift, at least 16.
struct Paged {
  void *k, *v;
  const int* table;
  int n_pages, n_kv, shift, hd, batch, max_pages;
  bool f16;
  int cap() const { return max_pages << shift; }
};

struct PagedAppend {
  const float *q, *k, *v;  // rows [batch][n], `stride` floats apart; q may be null
  int n_heads, n;          // n_heads 0 without q
  size_t stride;
  const float* rope;       // [position][pairs] (cos, sin), or null
  int pairs;
  const int *start, *count;  // [batch] or null: 0, n
  int* len_out;              // [batch] or null
  float* q_out;
  size_t q_out_stride;
};
void launch_paged_append(const Paged& c, const PagedAppend& a, hipStream_t st);

struct PagedAttn {
  const float* q;  // rows of q_stride floats, [batch][n_q]
  size_t q_stride;
  int n_heads, n_q;
  const int* len;  // [batch]
  int max_len;
  const int* shared_pages;  // of the first *shared entries of every sequence (max_shared 0: null)
  const int* shared;
  int max_shared, window;  // window 0: none
  float scale;
  float* out;  // [batch][n_q][n_heads][hd]
};
size_t paged_attention_workspace(const Paged& c, int n_heads, int n_q, int max_len, int max_shared);
void launch_paged_attention(const Paged& c, const PagedAttn& a, void* ws, hipStream_t st);

}  // namespace iek
