// The 8-bit KV cache: append, load and eviction (the attention over it: kv8_attention.hip).
//
// A head's rows are 8-bit codes (int8, or e4m3) with one scale s per block of 32 slots; a row's values
// are code * s. Scales are powers of two, s(a) = the smallest 2^e >= 2^-100 with a <= M 2^e for the
// block's largest |value| a (M: the codes' largest value, 127 or 448), so that x / s is exact, a
// value is rounded once, to its code, and moving a row to a larger scale rounds its code once more:
// with the scales doubling at each move the roundings add up to less than one step of the last
// scale. A scale of amax / M would be up to 2x finer, and inexact in every one of these steps.
// A non-finite value makes the block's scale NaN, so that whatever attends to it is NaN.
#include "common.cuh"
#include "kv8.h"
#include "kv8_codes.cuh"

namespace iek {

namespace {

// ---- append --------------------------------------------------------------------------------------
// One workgroup per (sequence, KV head, touched block, K or V): it holds the block's new rows in
// registers, takes their largest |value| (as integer bits: a NaN is larger than anything finite) and
// writes the codes and the scale. Rows of the block before `start` keep their values: when the scale
// grows, their codes are rounded again. Rows behind the new ones are dead and not looked at.
constexpr int AT = 256;

template <int HD, bool E4M3>
__global__ __launch_bounds__(AT) void append_kernel(Kv8 c, const float* __restrict__ kin, const float* __restrict__ vin,
                                                    int n, size_t stride, const int* __restrict__ start_p,
                                                    const int* __restrict__ count_p, int* __restrict__ len_out,
                                                    float* __restrict__ weights, int nspan) {
  constexpr int TPR = HD / 4;          // threads per row (four values each)
  constexpr int RPP = AT / TPR;        // rows per pass
  constexpr int NP = (KV8_BLOCK + RPP - 1) / RPP;
  const int t = threadIdx.x;
  int id = blockIdx.x;
  const int which = id & 1;
  id >>= 1;
  const int h = id % c.n_kv;
  id /= c.n_kv;
  const int span = id % nspan, b = id / nspan;
  const int start = start_p ? start_p[b] : 0;
  int count = count_p ? min(count_p[b], n) : n;
  if (start < 0 || start > c.cap) count = 0;  // (nothing is written)
  count = max(0, min(count, c.cap - start));
  if (span == 0 && h == 0 && which == 0 && t == 0 && len_out) len_out[b] = max(0, min(start, c.cap)) + count;
  const int blk = start / KV8_BLOCK + span, lo = blk * KV8_BLOCK;
  const int r0 = max(start - lo, 0), r1 = min(start + count - lo, KV8_BLOCK);  // the new rows of this block
  if (count == 0 || r1 <= r0) return;  // uniform
  const size_t head = (size_t)b * c.n_kv + h;
  const float* in = (which ? vin : kin) + (size_t)b * n * stride + (size_t)h * HD;
  uint8_t* codes = (which ? c.v : c.k) + (head * c.cap + lo) * HD;
  float* sp = (which ? c.vs : c.ks) + head * c.nblk + blk;
  const int tr = t / TPR, td = 4 * (t % TPR);
  float4 x[NP];
  uint32_t top = 0;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int r = p * RPP + tr;
    x[p] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r >= r0 && r < r1) x[p] = *reinterpret_cast<const float4*>(in + (size_t)(lo + r - start) * stride + td);
  }
#pragma unroll
  for (int p = 0; p < NP; ++p)
    top = max(max(max(top, abs_bits(x[p].x)), max(abs_bits(x[p].y), abs_bits(x[p].z))), abs_bits(x[p].w));
  __shared__ uint32_t red[AT / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if ((t & 63) == 0) red[t >> 6] = top;
  const float old = r0 > 0 ? *sp : 0.f;
  __syncthreads();  // (every thread has read the old scale: it is loaded before it is used below)
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  float s = kv8_scale<E4M3>(top);
  if (r0 > 0 && !(old <= s)) s = isnan(s) ? s : old;  // the earlier rows' scale is larger, or NaN
  const float inv = 1.f / s;                          // exact
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int r = p * RPP + tr;
    if (r >= r0 && r < r1) *reinterpret_cast<uint32_t*>(codes + (size_t)r * HD + td) = kv8_pack<E4M3>(x[p], inv);
  }
  if (r0 > 0 && s > old) {  // (not with a NaN: the codes stay)
    const float f = old * inv;
    for (int r = tr; r < r0; r += RPP) {
      uint32_t* w = reinterpret_cast<uint32_t*>(codes + (size_t)r * HD + td);
      *w = kv8_pack<E4M3>(kv8_unpack<E4M3>(*w), f);
    }
  }
  if (weights && which == 0 && t >= r0 && t < r1) weights[head * c.cap + lo + t] = 0.f;
  __syncthreads();
  if (t == 0) *sp = s;
}

// len_out given over start itself: every workgroup of the append has read it by now
__global__ void advance_kernel(int batch, int cap, const int* count, int n, int* len) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= batch) return;
  const int s = len[b];
  const int cnt = s < 0 || s > cap ? 0 : max(0, min(count ? min(count[b], n) : n, cap - s));
  len[b] = max(0, min(s, cap)) + cnt;
}

// ---- load ----------------------------------------------------------------------------------------
template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void load_kernel(Kv8 c, int n, size_t stride, const int* __restrict__ start_p,
                                                   const int* __restrict__ count_p, float* __restrict__ k,
                                                   float* __restrict__ v, size_t total) {
  constexpr int TPR = HD / 4;
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int d = 4 * (int)(i % TPR);
    size_t row = i / TPR;
    const int h = (int)(row % c.n_kv);
    row /= c.n_kv;
    const int j = (int)(row % n), b = (int)(row / n);
    const int start = start_p ? start_p[b] : 0, count = count_p ? min(count_p[b], n) : n;
    const long long slot = (long long)start + j;
    if (j >= count || slot < 0 || slot >= c.cap) continue;
    const size_t head = (size_t)b * c.n_kv + h;
    const size_t src = (head * c.cap + slot) * HD + d, dst = ((size_t)b * n + j) * stride + (size_t)h * HD + d;
    const size_t sc = head * c.nblk + slot / KV8_BLOCK;
    const float4 a = kv8_unpack<E4M3>(*reinterpret_cast<const uint32_t*>(c.k + src));
    const float4 z = kv8_unpack<E4M3>(*reinterpret_cast<const uint32_t*>(c.v + src));
    const float sk = c.ks[sc], sv = c.vs[sc];
    *reinterpret_cast<float4*>(k + dst) = make_float4(a.x * sk, a.y * sk, a.z * sk, a.w * sk);
    *reinterpret_cast<float4*>(v + dst) = make_float4(z.x * sv, z.y * sv, z.z * sv, z.w * sv);
  }
}

// ---- eviction ------------------------------------------------------------------------------------
// Order of the weights: NaN above everything, -0 as +0.
IEK_DEV uint32_t weight_key(float w) {
  if (isnan(w)) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int ST = 1024;

// One workgroup per (sequence, KV head). The keep - first - last largest weights of the entries
// [first, len - last): the bits of the smallest key among them, eight at a time from the top by
// histograms, then one pass in order that writes the kept entries' slots (of the entries with that
// very key the first ones). It also puts the old scales by (an eviction in place overwrites them)
// and gives each block of the result its scale, the largest of its rows' old ones.
__global__ __launch_bounds__(ST) void select_kernel(Kv8 src, Kv8 dst, Kv8Evict a, int* __restrict__ index,
                                                    float* __restrict__ old_scales) {
  const int head = blockIdx.x, b = head / src.n_kv, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int n = max(0, min(a.len[b], a.max_len));
  const int kept = min(n, a.keep);
  int* idx = index + (size_t)head * a.keep;
  float* olds = old_scales + (size_t)head * 2 * src.nblk;
  const float* w = a.w + (size_t)head * src.cap;
  __shared__ int hist[256];
  __shared__ int wsum[2][ST / 64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int nb_old = (n + KV8_BLOCK - 1) / KV8_BLOCK;
  for (int i = t; i < nb_old; i += ST) {
    olds[i] = src.ks[(size_t)head * src.nblk + i];
    olds[src.nblk + i] = src.vs[(size_t)head * src.nblk + i];
  }
  if (n <= a.keep) {
    for (int i = t; i < n; i += ST) idx[i] = i;
  } else {
    const int lo = a.first, hi = n - a.last;
    int need = a.keep - a.first - a.last;
    uint32_t prefix = 0xFFFFFFFFu;
    if (need > 0) {
      prefix = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int j = lo + t; j < hi; j += ST) {
          const uint32_t key = weight_key(w[j]);
          if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (wave == 0) {  // lane l: bins 255 - 4 l downwards
          int c[4], sum = 0;
          for (int i = 0; i < 4; ++i) sum += c[i] = hist[255 - 4 * lane - i];
          int incl = sum;
          for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(incl, o);
            if (lane >= o) incl += up;
          }
          int before = incl - sum;
          if (before < need && need <= incl) {
            for (int i = 0; i < 4; ++i) {
              if (before + c[i] >= need) {
                s_prefix = prefix | (uint32_t)(255 - 4 * lane - i) << shift;
                s_need = need - before;
                break;
              }
              before += c[i];
            }
          }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
      }
    }
    // `need` entries with the key `prefix` itself are kept. Wave w takes the w-th run of entries.
    const int run = ((n + ST - 1) / ST) * 64, j0 = wave * run, j1 = min(n, j0 + run);
    const int ties = need;
    int more = 0, same = 0;
    for (int j = j0 + lane; j - lane < j1; j += 64) {
      const bool in = j < j1, free_ = in && j >= lo && j < hi;
      const uint32_t key = free_ ? weight_key(w[j]) : 0;
      more += __popcll(__ballot(in && (!free_ || key > prefix)));
      same += __popcll(__ballot(free_ && key == prefix));
    }
    if (lane == 0) {
      wsum[0][wave] = more;
      wsum[1][wave] = same;
    }
    __syncthreads();
    int before = 0, eq = 0;
    for (int i = 0; i < wave; ++i) {
      before += wsum[0][i];
      eq += wsum[1][i];
    }
    for (int j = j0 + lane; j - lane < j1; j += 64) {
      const bool in = j < j1, free_ = in && j >= lo && j < hi;
      const uint32_t key = free_ ? weight_key(w[j]) : 0;
      const bool big = in && (!free_ || key > prefix), tie = free_ && key == prefix;
      const unsigned long long mb = __ballot(big), mt = __ballot(tie), below = (1ull << lane) - 1;
      const int tb = eq + __popcll(mt & below);
      if (big || (tie && tb < ties)) idx[before + __popcll(mb & below) + min(tb, ties)] = j;
      before += __popcll(mb);
      eq += __popcll(mt);
    }
  }
  __syncthreads();  // idx and olds are this workgroup's own writes
  const int nb = (kept + KV8_BLOCK - 1) / KV8_BLOCK;
  for (int i = t; i < 2 * nb; i += ST) {
    const int which = i >= nb, blk = which ? i - nb : i;
    float s = 0.f;
    const int e = min(kept, (blk + 1) * KV8_BLOCK);
    for (int r = blk * KV8_BLOCK; r < e; ++r) {
      const float o = olds[which * src.nblk + idx[r] / KV8_BLOCK];
      s = isnan(o) || isnan(s) ? NAN : fmaxf(s, o);
    }
    (which ? dst.vs : dst.ks)[(size_t)head * dst.nblk + blk] = s;
  }
  if (t == 0 && head % src.n_kv == 0 && a.len_out != a.len) a.len_out[b] = kept;
}

// Row r of the result is row idx[r] >= r of the source, its codes rounded to the block's new scale.
// A workgroup takes 64 bytes of K's or V's rows (or the weights) over a run of blocks. In place
// (one run) it goes through the blocks in order: a block's sources lie at or behind it, so reading
// all of them before the first write is all that is needed.
constexpr int MT = 256;

template <bool E4M3>
__global__ __launch_bounds__(MT) void move_kernel(Kv8 src, Kv8 dst, Kv8Evict a, const int* __restrict__ index,
                                                  const float* __restrict__ old_scales, int parts, bool in_place) {
  const int slices = src.hd / 64, t = threadIdx.x;
  int id = blockIdx.x;
  const int slice = id % (2 * slices + 1);
  id /= 2 * slices + 1;
  const int part = id % parts, head = id / parts, b = head / src.n_kv;
  const int n = max(0, min(a.len[b], a.max_len)), kept = min(n, a.keep);
  if (in_place && n <= a.keep) return;
  const int* idx = index + (size_t)head * a.keep;
  const int nb = (kept + KV8_BLOCK - 1) / KV8_BLOCK;
  const int b0 = (int)((long long)nb * part / parts), b1 = (int)((long long)nb * (part + 1) / parts);
  if (slice == 2 * slices) {
    const float* w = a.w + (size_t)head * src.cap;
    float* wo = a.w_out + (size_t)head * dst.cap;
    const int e = min(kept, b1 * KV8_BLOCK);
    for (int r0 = b0 * KV8_BLOCK; r0 < e; r0 += MT) {
      const int r = r0 + t;
      float x = 0.f;
      if (r < e) x = w[idx[r]];
      if (in_place) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
      }
      if (r < e) wo[r] = x;
    }
    return;
  }
  const int which = slice >= slices, d = (slice % slices) * 64 + 8 * (t & 7);
  const uint8_t* from = (which ? src.v : src.k) + (size_t)head * src.cap * src.hd + d;
  uint8_t* to = (which ? dst.v : dst.k) + (size_t)head * dst.cap * dst.hd + d;
  const float* olds = old_scales + ((size_t)head * 2 + which) * src.nblk;
  const float* news = (which ? dst.vs : dst.ks) + (size_t)head * dst.nblk;
  for (int blk = b0; blk < b1; ++blk) {
    const int last = min(kept, (blk + 1) * KV8_BLOCK) - 1;
    if (in_place && idx[last] == last) continue;  // (uniform) nothing before it is gone either
    const int r = blk * KV8_BLOCK + (t >> 3);
    uint2 x;
    if (r < kept) {
      const int s = idx[r];
      x = *reinterpret_cast<const uint2*>(from + (size_t)s * src.hd);
      const float f = olds[s / KV8_BLOCK] / news[blk];
      if (f < 1.f) {
        x.x = kv8_pack<E4M3>(kv8_unpack<E4M3>(x.x), f);
        x.y = kv8_pack<E4M3>(kv8_unpack<E4M3>(x.y), f);
      }
    }
    if (in_place) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
    if (r < kept) *reinterpret_cast<uint2*>(to + (size_t)r * dst.hd) = x;
  }
}

// len_out given over len itself: the kernels before have read it
__global__ void clip_kernel(int batch, int max_len, int keep, int* len) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < batch) len[b] = min(max(0, min(len[b], max_len)), keep);
}

}  // namespace

#define KV8_HD(HD_, ...)                                             \
  switch (HD_) {                                                     \
    case 64: { constexpr int HD = 64; __VA_ARGS__; } break;          \
    case 128: { constexpr int HD = 128; __VA_ARGS__; } break;        \
    case 256: { constexpr int HD = 256; __VA_ARGS__; } break;        \
    default: { constexpr int HD = 512; __VA_ARGS__; } break;         \
  }

void launch_kv8_append(const Kv8& c, const float* k, const float* v, int n, size_t stride, const int* start,
                       const int* count, int* len_out, float* weights, hipStream_t st) {
  const int nspan = (n + 2 * KV8_BLOCK - 2) / KV8_BLOCK;  // blocks that n rows can touch
  const size_t grid = (size_t)2 * c.n_kv * nspan * c.batch;
  if (grid > INT32_MAX) fail(ST_OP, "kv8 append: too many rows");
  const bool over = len_out && len_out == start;
  KV8_HD(c.hd, {
    auto fn = c.e4m3 ? append_kernel<HD, true> : append_kernel<HD, false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(AT), 0, st, c, k, v, n, stride, start, count,
                       over ? nullptr : len_out, weights, nspan);
  })
  if (over)
    hipLaunchKernelGGL(advance_kernel, dim3((c.batch + 63) / 64), dim3(64), 0, st, c.batch, c.cap, count, n, len_out);
}

void launch_kv8_load(const Kv8& c, int n, size_t stride, const int* start, const int* count, float* k, float* v,
                     hipStream_t st) {
  const size_t total = (size_t)c.batch * n * c.n_kv * (c.hd / 4);
  const unsigned grid = (unsigned)std::min<size_t>((total + 255) / 256, 256 * 32);
  KV8_HD(c.hd, {
    auto fn = c.e4m3 ? load_kernel<HD, true> : load_kernel<HD, false>;
    hipLaunchKernelGGL(fn, dim3(grid), dim3(256), 0, st, c, n, stride, start, count, k, v, total);
  })
}

// [old scales: batch * n_kv * 2 * nblk floats][kept slots: batch * n_kv * keep ints]
static size_t evict_scales_bytes(const Kv8& src) {
  return ((size_t)src.batch * src.n_kv * 2 * src.nblk * 4 + 255) / 256 * 256;
}
size_t kv8_evict_workspace(const Kv8& src, int, int keep) {
  return evict_scales_bytes(src) + (size_t)src.batch * src.n_kv * keep * 4;
}

void launch_kv8_evict(const Kv8& src, const Kv8& dst, const Kv8Evict& a, void* ws, hipStream_t st) {
  const int heads = src.batch * src.n_kv;
  const bool in_place = src.k == dst.k;
  float* olds = static_cast<float*>(ws);
  int* index = a.index_out ? a.index_out : reinterpret_cast<int*>(static_cast<char*>(ws) + evict_scales_bytes(src));
  hipLaunchKernelGGL(select_kernel, dim3(heads), dim3(ST), 0, st, src, dst, a, index, olds);
  const int slices = 2 * (src.hd / 64) + 1;
  const int nb = (std::min(a.keep, a.max_len) + KV8_BLOCK - 1) / KV8_BLOCK;
  const int parts = in_place ? 1 : std::max(1, std::min(nb, 2048 / (heads * slices)));
  if (nb > 0) {
    auto fn = src.e4m3 ? move_kernel<true> : move_kernel<false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)heads * slices * parts), dim3(MT), 0, st, src, dst, a, index, olds, parts,
                       in_place);
  }
  if (a.len_out == a.len)
    hipLaunchKernelGGL(clip_kernel, dim3((src.batch + 63) / 64), dim3(64), 0, st, src.batch, a.max_len, a.keep,
                       a.len_out);
}

}  // namespace iek
