// Attention of one or several new tokens per sequence over the 8-bit KV cache (kv8.h).
//
// Column c = t * G + g of a KV head is query token t, query head g of its group of G. It sees the
// entries [lo, hi): hi = len - (n_q - 1 - t), lo = hi - window with a window, else 0. A chunk's
// partial of a column is (m, l, o): m the largest score in base 2, l = sum 2^(s - m),
// o = sum 2^(s - m) v; the second launch joins the chunks and, with weights, adds each entry's
// share 2^(s - m) / l, summed over the KV head's columns, from the stored scores.
#include "common.cuh"
#include "kv8.h"
#include "kv8_codes.cuh"

namespace iek {

namespace {

struct Plan {
  int cols, chunk, nsplit, spad;  // columns of a KV head, slots a chunk, chunks, stored scores a column
  float* ml;                      // [batch * n_kv][cols][nsplit][2]
  float* o;                       // [batch * n_kv][cols][nsplit][hd]
  float* s;                       // [batch * n_kv][cols][spad] or null
};

IEK_DEV void col_range(const Kv8Attn& a, int n, int t, int& lo, int& hi) {
  hi = n - (a.n_q - 1 - t);
  lo = a.window > 0 ? max(0, hi - a.window) : 0;
}

// One wave per (column, chunk).
template <int HD, bool E4M3>
__global__ __launch_bounds__(64) void part_kernel(Kv8 c, Kv8Attn a, Plan p) {
  constexpr int DPL = HD / 64;
  const int lane = threadIdx.x;
  int id = blockIdx.x;
  const int cp = id % p.nsplit;
  id /= p.nsplit;
  const int col = id % p.cols, bh = id / p.cols;
  const int b = bh / c.n_kv, h = bh % c.n_kv, G = a.n_heads / c.n_kv, t = col / G;
  const int n = max(0, min(a.len[b], a.max_len));
  int lo, hi;
  col_range(a, n, t, lo, hi);
  const int c0 = cp * p.chunk, c1 = min(n, c0 + p.chunk);
  const size_t pi = ((size_t)bh * p.cols + col) * p.nsplit + cp;
  __shared__ __align__(16) float q[HD];
  __shared__ float ps[64];
  const float* qr = a.q + ((size_t)b * a.n_q + t) * a.q_stride + (size_t)(h * G + col % G) * HD;
  for (int d = lane; d < HD; d += 64) q[d] = qr[d];
  __syncthreads();
  const uint8_t* K = c.k + (size_t)bh * c.cap * HD;
  const uint8_t* V = c.v + (size_t)bh * c.cap * HD;
  float m = -INFINITY, l = 0.f, o[DPL] = {};
  for (int j0 = c0; j0 < c1; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < c1 && j >= lo && j < hi) {
      float dot = 0.f;
      for (int d = 0; d < HD; d += 4) {
        const float4 k4 = kv8_unpack<E4M3>(*reinterpret_cast<const uint32_t*>(K + (size_t)j * HD + d));
        dot += q[d] * k4.x + q[d + 1] * k4.y + q[d + 2] * k4.z + q[d + 3] * k4.w;
      }
      s = dot * (c.ks[(size_t)bh * c.nblk + j / KV8_BLOCK] * (a.scale * 1.44269504088896340736f));
    }
    if (p.s && j < c1) p.s[((size_t)bh * p.cols + col) * p.spad + j] = s;
    const bool in = j < c1 && j >= lo && j < hi;
    const float mn = fmaxf(m, wave_max(s));
    const float corr = m == -INFINITY ? 1.f : exp2f(m - mn);
    const float e = in ? exp2f(s - mn) : 0.f;
    l = l * corr + wave_sum(e);
    m = mn;
    ps[lane] = e;
    __syncthreads();
    for (int i = 0; i < DPL; ++i) o[i] *= corr;
    for (int i = 0; i < 64 && j0 + i < c1; ++i) {
      if (j0 + i < lo || j0 + i >= hi) continue;
      const float w = ps[i] * c.vs[(size_t)bh * c.nblk + (j0 + i) / KV8_BLOCK];
      for (int d = 0; d < DPL; ++d) {
        const uint32_t by = V[(size_t)(j0 + i) * HD + lane + 64 * d];
        o[d] += w * kv8_unpack<E4M3>(by).x;
      }
    }
    __syncthreads();
  }
  if (lane == 0) {
    p.ml[2 * pi] = isnan(l) ? l : m;  // (a NaN reaches the output: the maximum passes it over)
    p.ml[2 * pi + 1] = l;
  }
  for (int d = 0; d < DPL; ++d) p.o[pi * HD + lane + 64 * d] = o[d];
}

// Workgroups [0, batch * n_kv * cols): the output of a column; those behind them: weights of 256 entries.
template <int HD>
__global__ __launch_bounds__(256) void join_kernel(Kv8 c, Kv8Attn a, Plan p, int wblocks) {
  const int t = threadIdx.x, ncol = c.batch * c.n_kv * p.cols, G = a.n_heads / c.n_kv;
  if ((int)blockIdx.x < ncol) {
    const int bh = blockIdx.x / p.cols, col = blockIdx.x % p.cols, b = bh / c.n_kv, h = bh % c.n_kv;
    const float* ml = p.ml + (size_t)blockIdx.x * p.nsplit * 2;
    const float* o = p.o + (size_t)blockIdx.x * p.nsplit * HD;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < p.nsplit; ++i) m = fmaxf(m, ml[2 * i]);
    for (int i = 0; i < p.nsplit; ++i) l += ml[2 * i] == -INFINITY ? 0.f : ml[2 * i + 1] * exp2f(ml[2 * i] - m);
    for (int d = t; d < HD; d += 256) {
      float x = 0.f;
      for (int i = 0; i < p.nsplit; ++i)
        if (ml[2 * i] != -INFINITY) x += o[(size_t)i * HD + d] * exp2f(ml[2 * i] - m);
      a.out[(((size_t)b * a.n_q + col / G) * a.n_heads + h * G + col % G) * HD + d] = m == -INFINITY && l == 0.f ? 0.f : x / l;
    }
    return;
  }
  const int id = blockIdx.x - ncol, bh = id / wblocks, j = (id % wblocks) * 256 + t, b = bh / c.n_kv;
  const int n = max(0, min(a.len[b], a.max_len));
  if (j >= n) return;
  float w = 0.f;
  for (int col = 0; col < p.cols; ++col) {
    int lo, hi;
    col_range(a, n, col / G, lo, hi);
    const float* ml = p.ml + ((size_t)bh * p.cols + col) * p.nsplit * 2;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < p.nsplit; ++i) m = fmaxf(m, ml[2 * i]);
    for (int i = 0; i < p.nsplit; ++i) l += ml[2 * i] == -INFINITY ? 0.f : ml[2 * i + 1] * exp2f(ml[2 * i] - m);
    if (j >= lo && j < hi) w += exp2f(p.s[((size_t)bh * p.cols + col) * p.spad + j] - m) / l;
  }
  const size_t at = (size_t)bh * c.cap + j;
  a.w_out[at] = (a.w_in ? a.w_in[at] : 0.f) + w;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

Plan make_plan(const Kv8& c, int n_heads, int n_q, int max_len, bool weights, void* ws, size_t* bytes) {
  Plan p{};
  p.cols = n_heads / c.n_kv * n_q;
  p.chunk = std::max(256, (max_len + 63) / 64);
  p.nsplit = std::max(1, (max_len + p.chunk - 1) / p.chunk);
  p.spad = (max_len + 31) / 32 * 32;
  const size_t rows = (size_t)c.batch * c.n_kv * p.cols;
  const size_t ml = up256(rows * p.nsplit * 8), o = up256(rows * p.nsplit * c.hd * 4);
  char* base = static_cast<char*>(ws);
  p.ml = reinterpret_cast<float*>(base);
  p.o = reinterpret_cast<float*>(base + ml);
  p.s = weights ? reinterpret_cast<float*>(base + ml + o) : nullptr;
  if (bytes) *bytes = ml + o + (weights ? up256(rows * p.spad * 4) : 0);
  return p;
}

template <int HD>
void launch_hd(const Kv8& c, const Kv8Attn& a, const Plan& p, hipStream_t st) {
  const int rows = c.batch * c.n_kv * p.cols, wblocks = a.w_out ? (a.max_len + 255) / 256 : 0;
  auto fn = c.e4m3 ? part_kernel<HD, true> : part_kernel<HD, false>;
  hipLaunchKernelGGL(fn, dim3((unsigned)rows * p.nsplit), dim3(64), 0, st, c, a, p);
  hipLaunchKernelGGL(join_kernel<HD>, dim3((unsigned)rows + c.batch * c.n_kv * wblocks), dim3(256), 0, st, c, a, p,
                     wblocks);
}

}  // namespace

size_t kv8_attention_workspace(const Kv8& c, int n_heads, int n_q, int max_len, bool weights) {
  size_t bytes = 0;
  make_plan(c, n_heads, n_q, max_len, weights, nullptr, &bytes);
  return bytes;
}

void launch_kv8_attention(const Kv8& c, const Kv8Attn& a, void* ws, hipStream_t st) {
  const Plan p = make_plan(c, a.n_heads, a.n_q, a.max_len, a.w_out != nullptr, ws, nullptr);
  switch (c.hd) {
    case 64: launch_hd<64>(c, a, p, st); break;
    case 128: launch_hd<128>(c, a, p, st); break;
    case 256: launch_hd<256>(c, a, p, st); break;
    default: launch_hd<512>(c, a, p, st); break;
  }
}

}  // namespace iek
