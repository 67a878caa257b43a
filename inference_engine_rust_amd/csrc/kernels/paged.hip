// Append to the paged KV cache, with the rotation of the position on the way (the attention over it:
// paged_attention.hip).
//
// A row's position p is its entry's number. Adjacent pairs of the first 2 * pairs dims of every query and key
// head are turned, (x0, x1) -> (x0 c - x1 s, x0 s + x1 c) with (c, s) = rope[p][pair], each product and sum
// rounded by itself as in the op-level RoPE, so both give the same bits; keys and values then go to their slot.
// A row is read once and written once: bandwidth is the bound of prompts, the two dependent loads (start, then
// the page's number and (c, s)) that of single tokens: 369 MB of prompts (8 sequences of up to 2045 rows, 32 and 8 heads
// of 128, fp16) 75 us, 4.9 TB/s as a large copy; one row 3.4 us, 64 4.7.
#include "common.cuh"
#include "paged.h"

namespace iek {

namespace {

constexpr int AT = 256;

typedef float pf4_t __attribute__((ext_vector_type(4)));
typedef _Float16 ph4_t __attribute__((ext_vector_type(4)));

// Two pairs.
IEK_DEV pf4_t turn(pf4_t x, pf4_t cs) {
#pragma clang fp contract(off)
  return pf4_t{x[0] * cs[0] - x[1] * cs[1], x[0] * cs[1] + x[1] * cs[0], x[2] * cs[2] - x[3] * cs[3],
               x[2] * cs[3] + x[3] * cs[2]};
}

// Four dims a thread and turn; AT is a multiple of a head's quads, so that a thread has the same dims in every
// head it comes to, and loads their (c, s) once. A workgroup has a whole row: all of a sequence's work at n = 1,
// so that the length can be written over `start` (by then every wave has read it).
template <int HD, bool F16>
__global__ __launch_bounds__(AT) void append_kernel(Paged c, PagedAppend a) {
  constexpr int QUADS = HD / 4, U = 4;
  static_assert(AT % QUADS == 0, "dims of a thread");
  const int i = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
  const int start = a.start ? a.start[b] : 0;
  const int want = a.count ? max(0, min(a.count[b], a.n)) : a.n;
  const int cap = c.max_pages << c.shift;
  const int live = start < 0 || start > cap ? 0 : min(want, cap - start);
  if (a.n == 1) __syncthreads();
  if (i == 0 && t == 0 && a.len_out) a.len_out[b] = max(0, min(start, cap)) + live;
  if (i >= live) return;
  const int pos = start + i, page = c.table[(size_t)b * c.max_pages + (pos >> c.shift)];
  const bool there = (unsigned)page < (unsigned)c.n_pages;  // (rows without a page are dropped)
  const int d = 4 * (t % QUADS);
  const bool turned = d < 2 * a.pairs, both = d + 2 < 2 * a.pairs;  // (of an odd number of pairs the last one is alone)
  pf4_t cs = {1.f, 0.f, 1.f, 0.f};
  if (turned) {
    const float* e = a.rope + ((size_t)pos * a.pairs + d / 2) * 2;
    // (rows may be 8-byte aligned)
    cs[0] = e[0];
    cs[1] = e[1];
    if (both) {
      cs[2] = e[2];
      cs[3] = e[3];
    }
  }
  const int nq = a.n_heads, heads = nq + 2 * c.n_kv;
  const size_t row = ((size_t)b * a.n + i);
  const float *q = a.q + row * a.stride, *k = a.k + row * a.stride, *v = a.v + row * a.stride;
  float* qo = a.q_out + row * a.q_out_stride;
  const size_t slot = ((size_t)page * c.n_kv << c.shift) + (pos & ((1 << c.shift) - 1));
  for (int h0 = t / QUADS; h0 < heads; h0 += U * (AT / QUADS)) {
    pf4_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * (AT / QUADS);
      const float* from = h < nq ? q + (size_t)h * HD : h < nq + c.n_kv ? k + (size_t)(h - nq) * HD : v + (size_t)(h - nq - c.n_kv) * HD;
      if (h < heads) x[u] = *reinterpret_cast<const pf4_t*>(from + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * (AT / QUADS);
      if (h >= heads) break;
      const bool value = h >= nq + c.n_kv;
      pf4_t y = x[u];
      if (turned && !value) {
        y = turn(x[u], cs);
        if (!both) y = pf4_t{y[0], y[1], x[u][2], x[u][3]};
      }
      if (h < nq) {
        *reinterpret_cast<pf4_t*>(qo + (size_t)h * HD + d) = y;
      } else if (there) {
        const size_t at = (slot + ((size_t)(h - nq - (value ? c.n_kv : 0)) << c.shift)) * HD + d;
        void* pool = value ? c.v : c.k;
        if (F16) {
          // rounded to nearest even; beyond fp16's range it is an infinity
          *reinterpret_cast<ph4_t*>(static_cast<_Float16*>(pool) + at) =
              ph4_t{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
        } else {
          *reinterpret_cast<pf4_t*>(static_cast<float*>(pool) + at) = y;
        }
      }
    }
  }
}

// len_out given over start itself: every workgroup of the append has read it by now
__global__ void paged_advance_kernel(int batch, int cap, const int* count, int n, int* len) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= batch) return;
  const int start = len[b], want = count ? max(0, min(count[b], n)) : n;
  len[b] = max(0, min(start, cap)) + (start < 0 || start > cap ? 0 : min(want, cap - start));
}

}  // namespace

void launch_paged_append(const Paged& c, const PagedAppend& a, hipStream_t st) {
  const bool later = a.n > 1 && a.len_out && a.len_out == a.start;
  PagedAppend x = a;
  if (later) x.len_out = nullptr;
  const dim3 grid((unsigned)a.n, (unsigned)c.batch);
  auto go = [&](auto fn) { hipLaunchKernelGGL(fn, grid, dim3(AT), 0, st, c, x); };
  switch (c.hd) {
    case 64: c.f16 ? go(append_kernel<64, true>) : go(append_kernel<64, false>); break;
    case 128: c.f16 ? go(append_kernel<128, true>) : go(append_kernel<128, false>); break;
    case 256: c.f16 ? go(append_kernel<256, true>) : go(append_kernel<256, false>); break;
    default: c.f16 ? go(append_kernel<512, true>) : go(append_kernel<512, false>); break;
  }
  if (later)
    hipLaunchKernelGGL(paged_advance_kernel, dim3((unsigned)((c.batch + 63) / 64)), dim3(64), 0, st, c.batch, c.cap(), a.count,
                       a.n, a.len_out);
}

}  // namespace iek
