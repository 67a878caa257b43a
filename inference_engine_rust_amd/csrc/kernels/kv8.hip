// The 8-bit KV cache: append, load and eviction (the attention over it: kv8_attention.hip).
//
// A head's rows are 8-bit codes (int8, or e4m3) with one scale s per block of 32 slots; a row's values
// are code * s. Scales are powers of two, s(a) = the smallest 2^e >= 2^-100 with a <= M 2^e for the
// block's largest |value| a (M: the codes' largest value, 127 or 448), so that x / s is exact, a
// value is rounded once, to its code, and moving a row to a larger scale rounds its code once more:
// with the scales doubling at each move the roundings add up to less than one step of the last
// scale. A scale of amax / M would be up to 2x finer, and inexact in every one of these steps.
// A non-finite value makes the block's scale NaN, so that whatever attends to it is NaN.
#include <type_traits>

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
                                                    float* __restrict__ weights) {
  constexpr int TPR = HD / 4;          // threads per row (four values each)
  constexpr int RPP = AT / TPR;        // rows per pass
  constexpr int NP = (KV8_BLOCK + RPP - 1) / RPP;
  const int t = threadIdx.x;
  const int which = blockIdx.x & 1, span = blockIdx.x >> 1, h = blockIdx.y, b = blockIdx.z;
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
// One workgroup per (32 rows, KV head, sequence): 4 codes of K and of V to 16 bytes of f32 a lane. Bound by HBM
// (24576 rows of 8 heads of 128, 252 MB: 47 us). Nontemporal stores, so that the rows leave the caches to what comes next:
// this kernel takes as long without, but the move of the eviction that follows 33 us instead of 21.5.
typedef float kf4_t __attribute__((ext_vector_type(4)));
template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void load_kernel(Kv8 c, int n, size_t stride, const int* __restrict__ start_p,
                                                   const int* __restrict__ count_p, float* __restrict__ k,
                                                   float* __restrict__ v) {
  constexpr int TPR = HD / 4, RPP = 256 / TPR, NP = 32 / RPP;
  const int h = blockIdx.y, b = blockIdx.z, d = 4 * (threadIdx.x % TPR);
  const int start = start_p ? start_p[b] : 0, count = count_p ? min(count_p[b], n) : n;
  const size_t head = (size_t)b * c.n_kv + h;
  const int j0 = 32 * blockIdx.x + threadIdx.x / TPR;
  if (32 * (int)blockIdx.x >= count) return;
#pragma unroll 4
  for (int p = 0; p < NP; ++p) {
    const int j = j0 + RPP * p;
    const long long slot = (long long)start + j;
    if (j >= count || slot < 0 || slot >= c.cap) continue;
    const size_t src = (head * c.cap + slot) * HD + d, dst = ((size_t)b * n + j) * stride + (size_t)h * HD + d;
    const size_t sc = head * c.nblk + slot / KV8_BLOCK;
    const float4 a = kv8_unpack<E4M3>(*reinterpret_cast<const uint32_t*>(c.k + src));
    const float4 z = kv8_unpack<E4M3>(*reinterpret_cast<const uint32_t*>(c.v + src));
    const float sk = c.ks[sc], sv = c.vs[sc];
    __builtin_nontemporal_store(kf4_t{a.x * sk, a.y * sk, a.z * sk, a.w * sk}, reinterpret_cast<kf4_t*>(k + dst));
    __builtin_nontemporal_store(kf4_t{z.x * sv, z.y * sv, z.z * sv, z.w * sv}, reinterpret_cast<kf4_t*>(v + dst));
  }
}

// ---- eviction ------------------------------------------------------------------------------------
// Order of the weights: NaN above everything, -0 as +0.
IEK_DEV uint32_t weight_key(float w) {
  if (isnan(w)) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The bin in which the running sum from the top of `hist` passes `need` (> 0, at most the sum); need
// becomes what is left of it in that bin. Wave w sums the w-th part of the bins, then every wave looks
// through the part that holds it (sums: NW ints).
template <int NW, int BINS>
IEK_DEV int pick_bin(const int* hist, int* sums, int& need) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int PER = BINS / NW, NK = (PER + 255) / 256;  // bins of a part, as pieces of four a lane
  static_assert(PER % 256 == 0 || PER < 256, "pieces");
  // descending: part, piece, lane, then w, z, y, x
  auto four = [&](int part, int k) {
    const int at = 256 * k + 4 * lane;
    return at < PER ? *reinterpret_cast<const int4*>(&hist[BINS - 4 - part * PER - at]) : make_int4(0, 0, 0, 0);
  };
  int mine = 0;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int4 c = four(wave, k);
    mine += c.x + c.y + c.z + c.w;
  }
  mine = wave_scan(mine);
  if (lane == 63) sums[wave] = mine;
  __syncthreads();
  const int each = lane < NW ? sums[lane] : 0, upto = wave_scan(each);
  const int part = __ffsll(__ballot(lane < NW && need <= upto)) - 1;
  need -= __builtin_amdgcn_readlane(upto - each, part);
  int bin = 0;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int4 c = four(part, k);
    const int sum = c.x + c.y + c.z + c.w, incl = wave_scan(sum), all = __builtin_amdgcn_readlane(incl, 63);
    if (need > all) {  // uniform
      need -= all;
      continue;
    }
    const int winner = __ffsll(__ballot(need <= incl)) - 1;
    int left = need - (incl - sum);
    bin = BINS - 1 - part * PER - 256 * k - 4 * lane;
    if (left > c.w) {
      left -= c.w, --bin;
      if (left > c.z) {
        left -= c.z, --bin;
        if (left > c.y) left -= c.y, --bin;
      }
    }
    need = __builtin_amdgcn_readlane(left, winner);
    bin = __builtin_amdgcn_readlane(bin, winner);
    break;
  }
  return bin;
}

// Adds the wave's lanes with `in` to their bins, those that share the first one's bin at once if there are many.
IEK_DEV void add_bins(int* hist, int bin, bool in) {
  const unsigned long long all = __ballot(in);
  if (all == 0) return;
  const int bin0 = __builtin_amdgcn_readlane(bin, __ffsll(all) - 1);
  const int same = __popcll(__ballot(bin == bin0) & all);
  if (same >= 8) {
    if (in && bin != bin0) atomicAdd(&hist[bin], 1);
    if ((threadIdx.x & 63) == 0) atomicAdd(&hist[bin0], same);
  } else if (in) {
    atomicAdd(&hist[bin], 1);
  }
}

// One workgroup per (sequence, KV head): the slots of the entries that stay, in order. The smallest
// key that stays is found by histograms of its bits from the top, 12, 10 and 10 at a time (12 at first,
// sign, exponent and three bits more, spread weights over many bins and so the LDS atomics; entries that
// share the bin of their wave's first are added at once if there are many); then an entry's place is the number of
// larger ones before it plus those of that very key, of which the first ones stay. A wave has a run of
// entries to itself, their keys in LDS. Bound by one workgroup's latency and instructions, so few of both:
// two barriers per digit, four rows of 64 entries at a time, the ends of [first, n - last) apart.
// counts[head] = the entries that the sequence has. In place (olds given) the scales, which the move
// overwrites, are put by.
template <int ST, int CAP>
__global__ __launch_bounds__(ST) void select_kernel(Kv8 src, Kv8Evict a, int* __restrict__ index,
                                                    int* __restrict__ counts, float* __restrict__ olds) {
  constexpr int NW = ST / 64, RU = 4;
  const int head = blockIdx.x, b = head / src.n_kv, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = max(0, min(a.len[b], a.max_len));
  int* idx = index + (size_t)head * a.keep;
  const float* w = a.w + (size_t)head * src.cap;
  if (t == 0) counts[head] = n;
  if (n <= a.keep) {
    for (int i = t; i < n; i += ST) idx[i] = i;
    return;
  }
  __shared__ uint32_t keys[CAP];  // (max_len <= CAP)
  __shared__ __align__(16) int hist[4096 + 1024 + 1024];
  __shared__ int wsum[NW][2], sums[3][NW];
  const int lo = a.first, hi = n - a.last;
  const int rows = (n + ST * RU - 1) / (ST * RU) * RU;  // of 64 entries, a wave
  const int j0 = wave * rows * 64;                      // the wave's first entry
  // sixteen rows in flight, those that do not exist as the last entry (keys are read again by the
  // lane that wrote them)
  constexpr int LU = 16;
  for (int i = 0; i < rows; i += LU) {
    float x[LU];
#pragma unroll
    for (int r = 0; r < LU; ++r) x[r] = w[min(j0 + 64 * (i + r) + lane, n - 1)];
#pragma unroll
    for (int r = 0; r < LU; ++r)
      if (i + r < rows) keys[j0 + 64 * (i + r) + lane] = weight_key(x[r]);
  }
  for (int i = t; i < 6144 / 4; i += ST) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
  if (olds) {
    const int nb = (n + KV8_BLOCK - 1) / KV8_BLOCK;
    for (int i = t; i < nb; i += ST) {
      olds[(size_t)head * 2 * src.nblk + i] = src.ks[(size_t)head * src.nblk + i];
      olds[((size_t)head * 2 + 1) * src.nblk + i] = src.vs[(size_t)head * src.nblk + i];
    }
  }
  // f(first entry of a row, keys of the row, every entry in [lo, hi)?)
  auto each_row = [&](auto f) {
    for (int i = 0; i < rows; i += RU) {
      const int jb = j0 + 64 * i;
      if (jb >= n) break;
      uint32_t k[RU];
#pragma unroll
      for (int r = 0; r < RU; ++r) k[r] = keys[jb + 64 * r + lane];
      if (jb >= lo && jb + 64 * RU <= hi) {
#pragma unroll
        for (int r = 0; r < RU; ++r) f(jb + 64 * r, k[r], std::true_type{});
      } else {
#pragma unroll
        for (int r = 0; r < RU; ++r) f(jb + 64 * r, k[r], std::false_type{});
      }
    }
  };
  auto open = [&](int j, auto inner) { return inner.value || (j + lane >= lo && j + lane < hi); };
  uint32_t prefix = 0xFFFFFFFFu;
  int need = a.keep - a.first - a.last;
  int larger = 0, equal = 0;       // of the wave's entries: surely larger, and equal
  uint32_t unsure = 0xFFFFFFFFu;   // rows that hold entries which share its upper 22 bits
  __syncthreads();
  if (need > 0) {
    prefix = 0;
    // one digit: BITS bits from SHIFT on, among the entries that share all above
    auto digit = [&](auto shift_, auto bits_, int* h, int* part_sums) {
      constexpr int SHIFT = decltype(shift_)::value, BITS = decltype(bits_)::value;
      constexpr bool TOP = SHIFT + BITS == 32, LAST = SHIFT == 0;
      if (LAST) unsure = 0;
      each_row([&](int j, uint32_t key, auto inner) {
        bool in = open(j, inner);
        const bool o = in;
        if constexpr (!TOP) in = in && (key ^ prefix) >> (SHIFT + BITS) == 0;
        const unsigned long long all = __ballot(in);
        if (LAST) {
          if (all != 0) unsure |= 1u << ((j - j0) >> 6);
          else larger += __popcll(__ballot(o ? key > prefix : j + lane < n));
        }
        if (all == 0) return;
        const int bin = key >> SHIFT & ((1 << BITS) - 1);
        if (__popcll(all) >= 8) {
          const int bin0 = __builtin_amdgcn_readlane(bin, __ffsll(all) - 1);
          const int same = __popcll(__ballot(bin == bin0) & all);
          if (same >= 8) {
            if (in && bin != bin0) atomicAdd(&h[bin], 1);
            if (lane == 0) atomicAdd(&h[bin0], same);
            return;
          }
        }
        if (in) atomicAdd(&h[bin], 1);
      });
      __syncthreads();
      prefix |= (uint32_t)pick_bin<NW, 1 << BITS>(h, part_sums, need) << SHIFT;
    };
    using std::integral_constant;
    digit(integral_constant<int, 20>{}, integral_constant<int, 12>{}, hist, sums[0]);
    digit(integral_constant<int, 10>{}, integral_constant<int, 10>{}, hist + 4096, sums[1]);
    digit(integral_constant<int, 0>{}, integral_constant<int, 10>{}, hist + 5120, sums[2]);
  }
  // `need` of the entries with the key `prefix` stay
  auto count = [&](int j, uint32_t key, auto inner) {
    const bool o = open(j, inner);
    larger += __popcll(__ballot(o ? key > prefix : j + lane < n));
    equal += __popcll(__ballot(o && key == prefix));
  };
  for (; unsure != 0; unsure &= unsure - 1) {
    const int i = __ffs(unsure) - 1, j = j0 + 64 * i;
    if (i >= rows || j >= n) break;
    count(j, keys[j + lane], std::false_type{});
  }
  if (lane == 0) {
    wsum[wave][0] = larger;
    wsum[wave][1] = equal;
  }
  __syncthreads();
  larger = equal = 0;
  for (int i = 0; i < wave; ++i) {
    larger += wsum[i][0];
    equal += wsum[i][1];
  }
  each_row([&](int j, uint32_t key, auto inner) {
    const bool o = open(j, inner), g = o ? key > prefix : j + lane < n, e = o && key == prefix;
    const unsigned long long mg = __ballot(g), me = __ballot(e), below = (1ull << lane) - 1;
    const int gb = larger + __popcll(mg & below) + min(equal, need);
    if (me == 0) {
      if (g) idx[gb] = j + lane;
    } else {
      const int eb = equal + __popcll(me & below);
      if (g || (e && eb < need)) idx[gb - min(equal, need) + min(eb, need)] = j + lane;
      equal += __popcll(me);
    }
    larger += __popcll(mg);
  });
}

// The same selection of long sequences by several workgroups a head, one per segment of its entries: the
// histogram of the upper twelve bits (survey), the keys that share those of the smallest key that stays, a histogram of
// their next ten, and how many are surely larger (gather), then that key from the gathered ones and the segment's places
// (place). There every workgroup goes through all gathered keys, which are most of the entries where most weights are equal
// (those of fresh entries are zeros): once only, and those of a common value are counted in registers. Each launch
// waits for the one before it, so this pays where one workgroup's time over the entries is more than theirs.
constexpr int MAX_SEGS = 32, SEG_CHUNK = 4096, SEG_ROWS = SEG_CHUNK / 256;

struct Segs {
  int n, size;     // segments a head, entries a segment (whole chunks)
  int* hist;       // [heads][n][4096]
  int* next;       // [heads][n][1024], of the gathered keys
  uint32_t* keys;  // [heads][n][size]
  int* found;      // [heads][n] gathered keys, then [heads][n] surely larger ones
  int* state;      // [heads] prefix, then [heads] need
};

// The wave's sixteen rows of 64 entries of a chunk, the ones past the last as the last.
IEK_DEV void segment_keys(const float* w, int j0, int n, uint32_t (&key)[SEG_ROWS]) {
  float x[SEG_ROWS];
#pragma unroll
  for (int r = 0; r < SEG_ROWS; ++r) x[r] = w[min(j0 + 64 * r + (int)(threadIdx.x & 63), n - 1)];
#pragma unroll
  for (int r = 0; r < SEG_ROWS; ++r) key[r] = weight_key(x[r]);
}

__global__ __launch_bounds__(256) void survey_kernel(Kv8 src, Kv8Evict a, Segs g, int* __restrict__ counts,
                                                     float* __restrict__ olds) {
  const int head = blockIdx.y, s = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = max(0, min(a.len[head / src.n_kv], a.max_len));
  const int e0 = s * g.size, e1 = min(n, e0 + g.size), lo = a.first, hi = n - a.last;
  if (s == 0 && t == 0) counts[head] = n;
  if (n <= a.keep || e0 >= n) return;
  if (olds) {
    const int b0 = e0 / KV8_BLOCK, b1 = (e1 + KV8_BLOCK - 1) / KV8_BLOCK;
    for (int i = b0 + t; i < b1; i += 256) {
      olds[(size_t)head * 2 * src.nblk + i] = src.ks[(size_t)head * src.nblk + i];
      olds[((size_t)head * 2 + 1) * src.nblk + i] = src.vs[(size_t)head * src.nblk + i];
    }
  }
  if (a.keep - a.first - a.last == 0) return;
  __shared__ __align__(16) int h[4096];
  const float* w = a.w + (size_t)head * src.cap;
  for (int i = t; i < 1024; i += 256) reinterpret_cast<int4*>(h)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  for (int c0 = e0; c0 < e1; c0 += SEG_CHUNK) {
    const int j0 = c0 + wave * 64 * SEG_ROWS;
    uint32_t key[SEG_ROWS];
    segment_keys(w, j0, n, key);
#pragma unroll
    for (int r = 0; r < SEG_ROWS; ++r) {
      const int j = j0 + 64 * r + lane;
      add_bins(h, key[r] >> 20, j >= lo && j < hi);
    }
  }
  __syncthreads();
  int4* out = reinterpret_cast<int4*>(g.hist + ((size_t)head * g.n + s) * 4096);
  for (int i = t; i < 1024; i += 256) out[i] = reinterpret_cast<const int4*>(h)[i];
}

__global__ __launch_bounds__(256) void gather_kernel(Kv8 src, Kv8Evict a, Segs g) {
  const int head = blockIdx.y, s = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = max(0, min(a.len[head / src.n_kv], a.max_len));
  const int e0 = s * g.size, e1 = min(n, e0 + g.size), lo = a.first, hi = n - a.last;
  if (n <= a.keep || e0 >= n) return;
  __shared__ __align__(16) int h[4096];
  __shared__ __align__(16) int h2[1024];
  __shared__ int sums[4], wsum[2][4], gsum[4];
  const float* w = a.w + (size_t)head * src.cap;
  int need = a.keep - a.first - a.last;
  uint32_t prefix = 0xFFFFFFFFu;
  const bool any = need > 0;  // (else only the protected ones stay)
  if (any) {
    const int live = (n + g.size - 1) / g.size;
    const int4* in = reinterpret_cast<const int4*>(g.hist + (size_t)head * g.n * 4096) + t;
    int4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_int4(0, 0, 0, 0);
#pragma unroll 4
    for (int k = 0; k < live; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int4 y = in[k * 1024 + 256 * i];
        x[i].x += y.x, x[i].y += y.y, x[i].z += y.z, x[i].w += y.w;
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(h)[t + 256 * i] = x[i];
    reinterpret_cast<int4*>(h2)[t] = make_int4(0, 0, 0, 0);
    __syncthreads();
    prefix = (uint32_t)pick_bin<4, 4096>(h, sums, need) << 20;
  }
  if (s == 0 && t == 0) {
    g.state[head] = (int)prefix;
    g.state[gridDim.y + head] = need;
  }
  int run = 0, larger = 0, turn = 0;
  uint32_t* out = g.keys + ((size_t)head * g.n + s) * g.size;
  for (int c0 = e0; c0 < e1; c0 += SEG_CHUNK, turn ^= 1) {
    const int j0 = c0 + wave * 64 * SEG_ROWS;
    uint32_t key[SEG_ROWS];
    segment_keys(w, j0, n, key);
    int mine = 0;
#pragma unroll
    for (int r = 0; r < SEG_ROWS; ++r) {
      const int j = j0 + 64 * r + lane;
      const bool o = j >= lo && j < hi;
      mine += __popcll(__ballot(any && o && (key[r] ^ prefix) >> 20 == 0));
      larger += __popcll(__ballot(o ? any && key[r] >> 20 > prefix >> 20 : j < n));
    }
    if (lane == 0) wsum[turn][wave] = mine;
    __syncthreads();
    int at = run;
    for (int i = 0; i < wave; ++i) at += wsum[turn][i];
    run += wsum[turn][0] + wsum[turn][1] + wsum[turn][2] + wsum[turn][3];
    const bool few = mine <= 64;  // (of the wave's 1024)
#pragma unroll
    for (int r = 0; r < SEG_ROWS; ++r) {
      const int j = j0 + 64 * r + lane;
      const bool in = any && j >= lo && j < hi && (key[r] ^ prefix) >> 20 == 0;
      const unsigned long long m = __ballot(in);
      if (in) out[at + __popcll(m & ((1ull << lane) - 1))] = key[r];
      at += __popcll(m);
      const int bin = key[r] >> 10 & 1023;
      if (!few) add_bins(h2, bin, in);
      else if (in) atomicAdd(&h2[bin], 1);
    }
  }
  if (lane == 0) gsum[wave] = larger;
  __syncthreads();
  if (any) reinterpret_cast<int4*>(g.next + ((size_t)head * g.n + s) * 1024)[t] = reinterpret_cast<const int4*>(h2)[t];
  if (t == 0) {
    const size_t at = (size_t)head * g.n + s;
    g.found[at] = run;
    g.found[(size_t)gridDim.y * g.n + at] = gsum[0] + gsum[1] + gsum[2] + gsum[3];
  }
}

__global__ __launch_bounds__(256) void place_kernel(Kv8 src, Kv8Evict a, Segs g, int* __restrict__ index) {
  const int head = blockIdx.y, s = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = max(0, min(a.len[head / src.n_kv], a.max_len));
  const int e0 = s * g.size, e1 = min(n, e0 + g.size), lo = a.first, hi = n - a.last;
  int* idx = index + (size_t)head * a.keep;
  if (n <= a.keep) {
    for (int i = e0 + t; i < e1; i += 256) idx[i] = i;
    return;
  }
  if (e0 >= n) return;
  constexpr int BATCH = 4096;  // keys at a time
  __shared__ __align__(16) int h[2][2][1024];
  __shared__ int first[MAX_SEGS + 1], sums[2][4], wsum[2][4][2], before[4];
  const float* w = a.w + (size_t)head * src.cap;
  const int live = (n + g.size - 1) / g.size;
  // the segments' gathered keys as one list, and what lies before this segment
  const int mine = lane < live ? g.found[(size_t)head * g.n + lane] : 0, upto = wave_scan(mine);
  const int sure = lane < s ? g.found[(size_t)gridDim.y * g.n + (size_t)head * g.n + lane] : 0;
  const int listed = __builtin_amdgcn_readlane(upto, 63);
  int larger = __builtin_amdgcn_readlane(wave_scan(sure), 63), equal = 0;
  uint32_t prefix = (uint32_t)g.state[head];
  int need = g.state[gridDim.y + head];
  for (int i = t; i < 1024; i += 256) reinterpret_cast<int4*>(h[0][0])[i] = make_int4(0, 0, 0, 0);
  if (t <= MAX_SEGS) first[t] = upto - mine;  // (segments behind the last one: the list's end)
  __syncthreads();
  if (need > 0) {
    // Sixteen keys a lane, of which those that share the digits above are added to the bins of the digit at `shift`, of
    // all and of those before this segment. A value that many have is counted in registers.
    auto place = [&](int i0, int q) { return i0 + 1024 * (q >> 2) + 4 * t + (q & 3); };
    auto add = [&](const uint32_t(&key)[16], int i0, int end, int prior_end, int shift, int(&bins)[2][1024]) {
      auto in = [&](int q) { return place(i0, q) < end && (key[q] ^ prefix) >> shift >> 10 == 0; };
      int some = -1;
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        if (i0 + 1024 * (q >> 2) >= end) break;  // uniform
        if (in(q)) some = key[q] >> shift & 1023;
      }
      const unsigned long long any = __ballot(some >= 0);
      if (any == 0) return;
      const int common = __builtin_amdgcn_readlane(some, __ffsll(any) - 1);
      int many = 0;  // and those before this segment, from bit 16 on
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        if (i0 + 1024 * (q >> 2) >= end) break;
        if (!in(q)) continue;
        const int bin = key[q] >> shift & 1023;
        const bool prior = place(i0, q) < prior_end;
        if (bin == common) {
          many += prior ? 0x10001 : 1;
        } else {
          atomicAdd(&bins[0][bin], 1);
          if (prior) atomicAdd(&bins[1][bin], 1);
        }
      }
      many = wave_scan(many);
      if (lane == 63) {
        atomicAdd(&bins[0][common], many & 0xFFFF);
        atomicAdd(&bins[1][common], many >> 16);
      }
    };
    uint32_t key[16];
    const bool held = listed <= BATCH;
    if (held) {  // the second digit of a short list, whose keys stay in registers for the third
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        if (1024 * (q >> 2) >= listed) break;
        const int i = min(place(0, q), listed - 1);  // the i-th: in the last segment that begins at or before it
        int k = 0;
#pragma unroll
        for (int step = MAX_SEGS / 2; step; step >>= 1)
          if (first[k + step] <= i) k += step;
        key[q] = g.keys[((size_t)head * g.n + k) * g.size + i - first[k]];
      }
      add(key, 0, listed, first[s], 10, h[0]);
    } else {  // and of a long one
      const int4* in = reinterpret_cast<const int4*>(g.next + (size_t)head * g.n * 1024) + t;
      int4 x = make_int4(0, 0, 0, 0), y = x;
#pragma unroll 8
      for (int k = 0; k < live; ++k) {
        const int4 z = in[k * 256];
        x.x += z.x, x.y += z.y, x.z += z.z, x.w += z.w;
        if (k < s) y = x;
      }
      reinterpret_cast<int4*>(h[0][0])[t] = x;
      reinterpret_cast<int4*>(h[0][1])[t] = y;
    }
    __syncthreads();
    const int second = pick_bin<4, 1024>(h[0][0], sums[0], need);
    prefix |= (uint32_t)second << 10;
    if (held) {
      add(key, 0, listed, first[s], 0, h[1]);
    } else {
      for (int k = 0; k < live; ++k) {
        const uint32_t* from = g.keys + ((size_t)head * g.n + k) * g.size;
        const int here = first[k + 1] - first[k];
        for (int i0 = 0; i0 < here; i0 += BATCH) {
#pragma unroll
          for (int q = 0; q < 16; q += 4) {  // (a segment has room for whole fours)
            const int i = place(i0, q);
            const uint4 x = i < here ? *reinterpret_cast<const uint4*>(from + i) : make_uint4(0, 0, 0, 0);
            key[q] = x.x, key[q + 1] = x.y, key[q + 2] = x.z, key[q + 3] = x.w;
          }
          add(key, i0, here, k < s ? here : 0, 0, h[1]);
        }
      }
    }
    __syncthreads();
    const int third = pick_bin<4, 1024>(h[1][0], sums[1], need);
    prefix |= (uint32_t)third;
    int gb = 0;
    for (int i = t; i < 1024; i += 256) gb += (i > second ? h[0][1][i] : 0) + (i > third ? h[1][1][i] : 0);
    gb = wave_scan(gb);
    if (lane == 63) before[wave] = gb;
    __syncthreads();
    larger += before[0] + before[1] + before[2] + before[3];
    equal = h[1][1][third];
  }
  // `need` of the entries with the key `prefix` stay
  int turn = 0;
  for (int c0 = e0; c0 < e1; c0 += SEG_CHUNK, turn ^= 1) {
    const int j0 = c0 + wave * 64 * SEG_ROWS;
    uint32_t key[SEG_ROWS];
    segment_keys(w, j0, n, key);
    int gr = 0, er = 0;
#pragma unroll
    for (int r = 0; r < SEG_ROWS; ++r) {
      const int j = j0 + 64 * r + lane;
      const bool o = j >= lo && j < hi;
      gr += __popcll(__ballot(o ? key[r] > prefix : j < n));
      er += __popcll(__ballot(o && key[r] == prefix));
    }
    if (lane == 0) {
      wsum[turn][wave][0] = gr;
      wsum[turn][wave][1] = er;
    }
    __syncthreads();
    int gl = larger, eq = equal;
    for (int i = 0; i < 4; ++i) {
      if (i < wave) {
        gl += wsum[turn][i][0];
        eq += wsum[turn][i][1];
      }
      larger += wsum[turn][i][0];
      equal += wsum[turn][i][1];
    }
#pragma unroll
    for (int r = 0; r < SEG_ROWS; ++r) {
      const int j = j0 + 64 * r + lane;
      const bool o = j >= lo && j < hi, gt = o ? key[r] > prefix : j < n, e = o && key[r] == prefix;
      const unsigned long long mg = __ballot(gt), me = __ballot(e), below = (1ull << lane) - 1;
      const int eb = eq + __popcll(me & below);
      if (gt || (e && eb < need)) idx[gl + __popcll(mg & below) + min(eb, need)] = j;
      gl += __popcll(mg);
      eq += __popcll(me);
    }
  }
}

// Row r of the result is row idx[r] >= r of the source, its codes rounded to the block's new scale, the
// largest of its rows' old ones. A wave takes MB blocks of 32 rows at a time, SW bytes of each row of K or V,
// 16 bytes a lane; lanes 0 .. 31 look up the rows' slots and scales. Bound by HBM. In place one
// workgroup goes through all of a head's blocks in order, 64 bytes of the rows: the sources of
// what it takes at a time lie at or behind it, so reading all of them before the first write is all the
// order needed; a stretch that stays where it is is skipped.
template <bool E4M3, int SW, bool IN_PLACE, int MB>
__global__ __launch_bounds__(IN_PLACE ? 1024 : 256) void move_kernel(Kv8 src, Kv8 dst, Kv8Evict a,
                                                                     const int* __restrict__ index,
                                                                     const int* __restrict__ counts,
                                                                     const float* __restrict__ put_by, int parts) {
  constexpr int LPR = SW / 16, RPI = 64 / LPR, NI = KV8_BLOCK / RPI;  // lanes a row, rows a load, loads a block
  constexpr int NW = IN_PLACE ? 16 : 4;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), slices = src.hd / SW;
  int id = blockIdx.x;
  const int part = id % parts;
  id /= parts;
  const int slice = id % (2 * slices), head = id / (2 * slices);
  const int n = counts[head], kept = min(n, a.keep);
  if (slice == 0 && part == 0 && head % src.n_kv == 0 && t == 0) a.len_out[head / src.n_kv] = kept;
  if (IN_PLACE && n <= a.keep) return;
  const int* idx = index + (size_t)head * a.keep;
  const int nb = (kept + KV8_BLOCK - 1) / KV8_BLOCK;
  const int which = slice >= slices, d = (which ? slice - slices : slice) * SW + 16 * (lane % LPR);
  const uint8_t* from = (which ? src.v : src.k) + (size_t)head * src.cap * src.hd + d;
  uint8_t* to = (which ? dst.v : dst.k) + (size_t)head * dst.cap * dst.hd + d;
  const float* olds = IN_PLACE ? put_by + ((size_t)head * 2 + which) * src.nblk
                               : (which ? src.vs : src.ks) + (size_t)head * src.nblk;
  float* news = (which ? dst.vs : dst.ks) + (size_t)head * dst.nblk;
  const bool first = d < SW, weights = which == 0 && first;  // (first: the slice that writes the scales)
  const float* w = a.w + (size_t)head * src.cap;
  float* w_out = a.w_out + (size_t)head * dst.cap;
  for (int b0 = part * NW * MB; b0 < nb; b0 += parts * NW * MB) {
    if (IN_PLACE) {
      const int last = min(kept, (b0 + NW * MB) * KV8_BLOCK) - 1;
      if (idx[last] == last) continue;  // uniform: nothing up to there is gone
    }
    uint4 x[MB][NI];
    float f[MB][NI], s_new[MB], wv[MB];
#pragma unroll
    for (int k = 0; k < MB; ++k) {
      const int r0 = (b0 + wave * MB + k) * KV8_BLOCK, r = r0 + (lane & 31);
      // (the slot without waiting for `kept`: the list has `keep` places)
      const int listed = idx[min(r, a.keep - 1)], slot = r < kept ? listed : 0;
      const float s = r < kept ? olds[slot / KV8_BLOCK] : 0.f;
      wv[k] = weights && r < kept ? w[slot] : 0.f;
      s_new[k] = __any(isnan(s)) ? NAN : wave_max(s);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + lane / LPR;
        const int from_slot = __shfl(slot, row);
        f[k][i] = __shfl(s, row) / s_new[k];
        x[k][i] = make_uint4(0, 0, 0, 0);
        if (r0 + row < kept) x[k][i] = *reinterpret_cast<const uint4*>(from + (size_t)from_slot * src.hd);
      }
    }
    if (IN_PLACE) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < MB; ++k) {
      const int r0 = (b0 + wave * MB + k) * KV8_BLOCK;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int row = i * RPI + lane / LPR;
        if (f[k][i] < 1.f) {
          x[k][i].x = kv8_pack<E4M3>(kv8_unpack<E4M3>(x[k][i].x), f[k][i]);
          x[k][i].y = kv8_pack<E4M3>(kv8_unpack<E4M3>(x[k][i].y), f[k][i]);
          x[k][i].z = kv8_pack<E4M3>(kv8_unpack<E4M3>(x[k][i].z), f[k][i]);
          x[k][i].w = kv8_pack<E4M3>(kv8_unpack<E4M3>(x[k][i].w), f[k][i]);
        }
        if (r0 + row < kept) *reinterpret_cast<uint4*>(to + (size_t)(r0 + row) * dst.hd) = x[k][i];
      }
      if (weights && lane < KV8_BLOCK && r0 + lane < kept) w_out[r0 + lane] = wv[k];
      if (first && lane == 0 && r0 < kept) news[r0 / KV8_BLOCK] = s_new[k];
    }
  }
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
  const unsigned nspan = (unsigned)((n + 2 * KV8_BLOCK - 2) / KV8_BLOCK);  // blocks that n rows can touch
  const dim3 grid(2 * nspan, (unsigned)c.n_kv, (unsigned)c.batch);
  const bool over = len_out && len_out == start;
  KV8_HD(c.hd, {
    auto fn = c.e4m3 ? append_kernel<HD, true> : append_kernel<HD, false>;
    hipLaunchKernelGGL(fn, grid, dim3(AT), 0, st, c, k, v, n, stride, start, count, over ? nullptr : len_out, weights);
  })
  if (over)
    hipLaunchKernelGGL(advance_kernel, dim3((c.batch + 63) / 64), dim3(64), 0, st, c.batch, c.cap, count, n, len_out);
}

void launch_kv8_load(const Kv8& c, int n, size_t stride, const int* start, const int* count, float* k, float* v,
                     hipStream_t st) {
  const dim3 grid((unsigned)(n + 31) / 32, (unsigned)c.n_kv, (unsigned)c.batch);
  KV8_HD(c.hd, {
    auto fn = c.e4m3 ? load_kernel<HD, true> : load_kernel<HD, false>;
    hipLaunchKernelGGL(fn, grid, dim3(256), 0, st, c, n, stride, start, count, k, v);
  })
}

// One workgroup a head selects from up to SELECT_MOST entries, several from more: an eviction of 8 heads of 128 takes
// 33 us either way at 32768 (of 128 heads 76 against 102), 37 against 63 at 65536, 42 against 111 at 131072; with all
// weights equal 56 either way at 40000, 67 against 82 at 65536, 103 against 151 at 131072.
constexpr int SELECT_MOST = 32768;

static size_t up256(size_t x) { return (x + 255) / 256 * 256; }
namespace {
// [entries of each head][scales put by: 2 * nblk floats a head][kept slots: keep ints a head][segments]
struct EvictWs {
  int *counts, *index;
  float* olds;
  bool spread;
  Segs g;
  size_t bytes;
};
EvictWs evict_ws(const Kv8& c, int max_len, int keep, void* ws) {
  const size_t heads = (size_t)c.batch * c.n_kv;
  char* const base = static_cast<char*>(ws);
  EvictWs o{};
  size_t at = 0;
  auto part = [&](auto*& p, size_t n) {
    p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
    at += up256(n * 4);
  };
  part(o.counts, heads);
  part(o.olds, heads * 2 * c.nblk);
  part(o.index, heads * keep);
  o.spread = max_len > SELECT_MOST;
  if (o.spread) {
    const int chunks = (max_len + SEG_CHUNK - 1) / SEG_CHUNK;
    o.g.size = (chunks + MAX_SEGS - 1) / MAX_SEGS * SEG_CHUNK;
    o.g.n = (max_len + o.g.size - 1) / o.g.size;
    part(o.g.hist, heads * o.g.n * 4096);
    part(o.g.next, heads * o.g.n * 1024);
    part(o.g.keys, heads * o.g.n * o.g.size);
    part(o.g.found, heads * o.g.n * 2);
    part(o.g.state, heads * 2);
  }
  o.bytes = at;
  return o;
}
}  // namespace
size_t kv8_evict_workspace(const Kv8& src, int max_len, int keep) { return evict_ws(src, max_len, keep, nullptr).bytes; }

void launch_kv8_evict(const Kv8& src, const Kv8& dst, const Kv8Evict& a, void* ws, hipStream_t st) {
  const int heads = src.batch * src.n_kv;
  const bool in_place = src.k == dst.k;
  const EvictWs o = evict_ws(src, a.max_len, a.keep, ws);
  int* const index = a.index_out ? a.index_out : o.index;
  float* const put_by = in_place ? o.olds : nullptr;
  // Four waves up to 1024 entries, whose barriers are cheaper, sixteen above: an eviction from 8 heads of 128 takes with
  // four, eight and sixteen 16.9, 17.3 and 17.6 us at 1000 entries, 21.8, 20.7 and 21.1 at 2000, 27.8, 25.0 and 24.3 at 4000
  // (eight would gain 2 % around 2000 alone).
  auto select = a.max_len <= 1024 ? select_kernel<256, 1024> : select_kernel<1024, SELECT_MOST>;
  if (o.spread) {
    const dim3 grid((unsigned)o.g.n, (unsigned)heads);
    hipLaunchKernelGGL(survey_kernel, grid, dim3(256), 0, st, src, a, o.g, o.counts, put_by);
    hipLaunchKernelGGL(gather_kernel, grid, dim3(256), 0, st, src, a, o.g);
    hipLaunchKernelGGL(place_kernel, grid, dim3(256), 0, st, src, a, o.g, index);
  } else {
    hipLaunchKernelGGL(select, dim3(heads), dim3(a.max_len <= 1024 ? 256 : 1024), 0, st, src, a, index, o.counts, put_by);
  }
  // Not in place a wave takes 128 bytes a row (the lines of L2), one block where all waves fit the chip at once
  // (1024 entries of 8 heads of 128: 18.9 us against 20.0 for the eviction), else two (8192 of 24 heads: 102 against 104).
  const int sw = in_place || src.hd == 64 ? 64 : 128, slices = 2 * src.hd / sw;
  const int nb = (std::min(a.keep, a.max_len) + KV8_BLOCK - 1) / KV8_BLOCK;
  const int mb = in_place || (long long)heads * slices * nb > 8192 ? 2 : 1;
  const int parts = in_place ? 1 : std::max(1, std::min((nb + 4 * mb - 1) / (4 * mb), ((1 << 24) - 1) / (heads * slices)));
  void (*fn)(Kv8, Kv8, Kv8Evict, const int*, const int*, const float*, int);
  if (in_place) fn = src.e4m3 ? move_kernel<true, 64, true, 2> : move_kernel<false, 64, true, 2>;
  else if (sw == 64 && mb == 1) fn = src.e4m3 ? move_kernel<true, 64, false, 1> : move_kernel<false, 64, false, 1>;
  else if (sw == 64) fn = src.e4m3 ? move_kernel<true, 64, false, 2> : move_kernel<false, 64, false, 2>;
  else if (mb == 1) fn = src.e4m3 ? move_kernel<true, 128, false, 1> : move_kernel<false, 128, false, 1>;
  else fn = src.e4m3 ? move_kernel<true, 128, false, 2> : move_kernel<false, 128, false, 2>;
  hipLaunchKernelGGL(fn, dim3((unsigned)heads * slices * parts), dim3(in_place ? 1024 : 256), 0, st, src, dst,
                     a, index, o.counts, o.olds, parts);
}

}  // namespace iek
