// The 8-bit KV cache (iek_kv8): arguments of its launchers (kernels/kv8.hip, kernels/kv8_attention.hip).
#pragma once
#include "../iek_internal.h"

namespace iek {

constexpr int KV8_BLOCK = 32;         // cache slots that share a scale
constexpr int DT_I8 = 5, DT_E4M3 = 6;  // iek_dtype's IEK_I8 and IEK_E4M3

// k, v: [batch][n_kv][cap][hd] codes; ks, vs: [batch][n_kv][nblk] power-of-two scales.
struct Kv8 {
  uint8_t *k, *v;
  float *ks, *vs;
  int batch, n_kv, cap, hd, nblk;
  bool e4m3;
};

// Rows start[b] + i, i < min(n, count[b]) (count may be null: n). start null: 0.
void launch_kv8_append(const Kv8& c, const float* k, const float* v, int n, size_t stride, const int* start,
                       const int* count, int* len_out, float* weights, hipStream_t st);
void launch_kv8_load(const Kv8& c, int n, size_t stride, const int* start, const int* count, float* k, float* v,
                     hipStream_t st);

struct Kv8Attn {
  const float* q;       // rows of q_stride floats, [batch][n_q]
  size_t q_stride;
  int n_heads, n_q;
  const int* len;       // [batch]
  int max_len, window;  // window 0: none
  float scale;
  float* out;           // [batch][n_q][n_heads][hd]
  const float* w_in;    // [batch][n_kv][cap] or null
  float* w_out;         // the same, or null: no weights
};
size_t kv8_attention_workspace(const Kv8& c, int n_heads, int n_q, int max_len, bool weights);
void launch_kv8_attention(const Kv8& c, const Kv8Attn& a, void* ws, hipStream_t st);

struct Kv8Evict {
  const float* w;  // [batch][n_kv][src cap]
  float* w_out;    // [batch][n_kv][dst cap]
  const int* len;
  int* len_out;
  int max_len, keep, first, last;
  int* index_out;  // [batch][n_kv][keep] or null
};
size_t kv8_evict_workspace(const Kv8& src, int max_len, int keep);
// src and dst may be the same buffers.
void launch_kv8_evict(const Kv8& src, const Kv8& dst, const Kv8Evict& a, void* ws, hipStream_t st);

}  // namespace iek
