// Sampling with temperature, top-k, top-p and min-p, a row of logits per sequence (iek_dev_sample).
//
// Of a row with maximum M, token i has the weight w_i = exp((l_i - M) / T). The filters keep a prefix of the tokens
// in descending order (equal ones: the lower index first):
//   top-k: the first k;  top-p: of those the ones before which the sum of weights is below p times their total;
//   min-p: the ones with w_i >= min_p (M's token has 1).
// The pick is the first token in index order up to which the kept weights sum to more than r times their total.
//
// Weights are summed as integers, w 2^S rounded, with S as large as n of them allow in 64 bits and at most 50: sums do
// not depend on their order, so atomics on histograms and any split give the same token every time. A weight is off by
// 2^-(S + 1) of the largest (2^-50 at 32000 tokens) and 2^-48.4 of itself at most, where f32 sums would move the borders of
// tokens by 1e-7 of the total.
//
// A row of up to 32768 logits stays in the LDS of one workgroup. A border (top-k, top-p) is found by one histogram over
// the distance to the maximum, of counts or of weights, in 2048 bins; the few tokens of the bin that the border is in
// are ranked against each other. For a top-k of up to 1024 the threads' own maxima come first: the k-th largest of them
// is no larger than the k-th logit, so what lies below it (all but about k tokens) is out, and the rest goes on as a
// list; so do the tokens that top-p or min-p leave. A list of up to 512 is ranked as a whole.
// Larger rows are cut into slices over several workgroups, in four launches: the maxima; the row's histogram; the slices'
// candidates and sums; the border and the slice that has the token.
// Rows that the bins do not suit take any_row: a radix selection on the logits' bits as ordered integers, 11, 11 and 10 bits
// at a time, from memory, by one workgroup. These are
//   rows with more than NEAR tokens in the bin that a border is in: thousands of equal logits; top-k where masks of f32's lowest value
//     stretch the bins; and of large rows ordinary ones, since top-p's bins are 1/64 of an octave of weight (8 rows of 262144
//     normal logits: at a temperature of 1 and a p of 0.9 36 us, of 0.98 545; at 1.3 and 0.9 557);
//   rows of several slices with a top-k above 1024 (8 rows of 262144: 1000 27 us, 5000 403), or with more than SEGMENT of its
//     candidates in one slice (256 rows of 40000, whose slices are 32768 long: 100 51 us, 500 124);
//   draws of exactly 0.
// Bound by the latency of one workgroup's phases, and by the exponentials where every token needs one. 32000 logits, one
// row: 4.8 us greedy, 10.4 with top-k 50, 19 with top-p, 24 with a top-k of 5000; 256 rows of mixed filters 32 (their bytes
// take 5). 8 rows of 262144 with top-p of 0.9 at a temperature of 1: 4 + 10 + 10 + 15 us.
#include "common.cuh"
#include "sampling.h"

namespace iek {

namespace {

constexpr int ST = 1024, NW = ST / 64, BINS = 2048;

typedef unsigned long long u64;

// Order of the logits as unsigned integers (-0 is 0; no NaN comes here).
IEK_DEV uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
IEK_DEV float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// Weights of a row: w 2^S as an integer. 2^(y / 64), y = i + f, is a table's entry of 64 (in LDS) times a polynomial in
// f of degree 4: the exponential's first terms, and in place of z^5 / 120 (z = f L, L = ln 2 / 64, |z| <= L / 2) the cubic nearest to
// it, (L / 2)^2 z^3 / 96 - (L / 2)^4 z / 384 (Chebyshev: 16 x^5 = 20 x^3 - 5 x + T_5(x)), which leaves out (L / 2)^5 / 1920 <
// 2^-48.5; without the cubic it were 2^-44.5. The additions of 1.5 2^52 round to integers.
struct Weigh {
  double top, rate;  // 64 log2 e / T
  double one;        // 2^S
  const double* table;
  IEK_DEV double real(float x) const {  // (2^-64 stands for everything below it)
    const double y = fmax(((double)x - top) * rate, -4096.0), n = y + 0x1.8p52, f = y - (n - 0x1.8p52);
    constexpr double L = 0.693147180559945309417232 / 64;
    double e = L * L * L * L / 24;
    e = fma(e, f, L * L * L / 6 * (1 + L * L / 64));
    e = fma(e, f, L * L / 2);
    e = fma(e, f, L * (1 - L * L * L * L / 6144));
    e = fma(e, f, 1.0);
    const int i = (int)__double_as_longlong(n);
    e *= table[i & 63];
    return __longlong_as_double(__double_as_longlong(e) + ((long long)(i >> 6) << 52));
  }
  IEK_DEV u64 whole(double w) const {  // w 2^S <= 2^50, to nearest
    return (u64)__double_as_longlong(fma(w, one, 0x1p52)) & 0xFFFFFFFFFFFFFull;
  }
  IEK_DEV u64 operator()(float x) const { return whole(real(x)); }
};
IEK_DEV int scale_bits(int n) { return min(50, 32 + __clz(n)); }

template <int CTRL, int ROWS = 0xF>
IEK_DEV u64 dpp64(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
  return (u64)hi << 32 | lo;
}
// Inclusive prefix sums over a row of 16 lanes, and over the wave.
IEK_DEV u64 row_scan64(u64 v) {
  v += dpp64<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp64<0x112>(v);
  v += dpp64<0x114>(v);
  return v + dpp64<0x118>(v);
}
IEK_DEV u64 wave_scan64(u64 v) {
  v = row_scan64(v);
  v += dpp64<DPP_BCAST15, 0xA>(v);
  return v + dpp64<DPP_BCAST31, 0xC>(v);
}
IEK_DEV u64 lane64(u64 v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return (u64)hi << 32 | lo;
}

constexpr int SLICE = 32768, LIST = 2048, NEAR = 512;  // tokens of a workgroup, of a list, and of a bin that are ranked

// What the phases share beside the tokens.
struct Smem {
  double table[64];
  u64 part[2][NW];
  u64 word;
  int word2, count, ties;
  float border;
};
// Room for a histogram and for the tokens of its border: their keys << 32 | ~index (larger ones come first in
// descending order) and weights.
struct Bins {
  u64 hist[BINS];
  u64 near[NEAR], near_w[NEAR];
};

// What a row keeps: the keys above `key` and the first `ties` of those that are it.
struct Kept {
  uint32_t key;
  int ties;
};

// A row's parameters, its maximum, and whether there is a token to choose.
struct Head {
  float t, p, m, r;
  int k;
  float top;
  bool good;
};
// (all loads at once, of an array that is there in place of those that are not)
IEK_DEV SampleParams params_of(const SampleArgs& a, int b) {
  if (!a.temperature) return a.one;
  const float *p = a.top_p ? a.top_p : a.r, *m = a.min_p ? a.min_p : a.r;
  const int* k = a.top_k ? a.top_k : reinterpret_cast<const int*>(a.r);
  SampleParams o{a.temperature[b], p[b], m[b], a.r[b], k[b]};
  if (!a.top_p) o.top_p = 1.f;
  if (!a.min_p) o.min_p = 0.f;
  if (!a.top_k) o.top_k = 0;
  return o;
}
IEK_DEV Head head_of(const SampleParams& o, int n, float top) {  // (top: +inf if there is a NaN)
  Head h{o.temperature, o.top_p, o.min_p, o.r, o.top_k >= n ? 0 : o.top_k, top, false};
  // (a NaN parameter fails its comparison)
  h.good = fabsf(h.top) < INFINITY && h.t >= 0.f && h.t < INFINITY && h.r >= 0.f && h.r < 1.f && h.p == h.p && h.m == h.m;
  return h;
}
IEK_DEV void store(const SampleArgs& a, int b, uint32_t index, float prob) {
  a.index[b] = index;
  if (a.prob) a.prob[b] = prob;
}
IEK_DEV Weigh weigh_of(const Head& h, int n, const double* table) {
  return Weigh{(double)h.top, 64 * 1.44269504088896340735992 / (double)h.t, (double)(1ull << scale_bits(n)), table};
}
// (the table is there after the next barrier)
IEK_DEV void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x / 64);
}
// The probability of a token that was chosen.
IEK_DEV float share(const Head& h, const Weigh& w, float x, u64 total) {
  return (float)(exp(((double)x - w.top) / (double)h.t) / ((double)total / w.one));
}

// Sums over the workgroup, one barrier each: two of them in a row use different parts of m.part.
struct Group {
  Smem& m;
  int turn;
  IEK_DEV explicit Group(Smem& s) : m(s), turn(0) {}
  // The sum of v over the threads before this one; total: over all.
  IEK_DEV u64 before(u64 v, u64& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u64 incl = wave_scan64(v);
    if (lane == 63) m.part[turn][wave] = incl;
    __syncthreads();
    const u64 each = m.part[turn][lane & (NW - 1)], upto = row_scan64(each);
    turn ^= 1;
    total = lane64(upto, NW - 1);
    return lane64(upto - each, wave) + incl - v;
  }
  IEK_DEV u64 sum(u64 v) {
    u64 total;
    before(v, total);
    return total;
  }
  // The largest v, in every thread.
  IEK_DEV float most(float v) {
    v = wave_max(v);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* part = reinterpret_cast<float*>(m.part[turn]);
    if (lane == 0) part[wave] = v;
    __syncthreads();
    v = row16_max(part[lane & (NW - 1)]);
    turn ^= 1;
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
  }
};
static_assert(NW == 16, "a row of lanes has the waves' parts");

// ---- any row, from memory ---------------------------------------------------------------------------

// The bin, from the top, in which the running sum of the histogram passes, and the sum above it. (Some bin does.)
template <class Passes>
IEK_DEV int pick_bin(Group& q, const u64* hist, Passes passes, u64& above) {
  Smem& m = q.m;
  const int t = threadIdx.x;
  // thread t: bins BINS - 1 - 2 t and the next below
  const u64 a = hist[BINS - 1 - 2 * t], b = hist[BINS - 2 - 2 * t];
  u64 total;
  const u64 before = q.before(a + b, total);
  // (sums only grow: the one thread where it first passes)
  if (!passes(before) && passes(before + a + b)) {
    const bool first = passes(before + a);
    m.word = first ? before : before + a;
    m.word2 = BINS - 1 - 2 * t - (first ? 0 : 1);
  }
  __syncthreads();
  above = m.word;
  const int bin = m.word2;
  __syncthreads();
  return bin;
}

// A wave's run of the row: groups of 256 logits, four a lane.
struct Row {
  const float* x;
  int n, groups, first;  // of a wave: groups of 256, from index `first`
  template <class F>
  IEK_DEV void each(F f) const {  // f(value, index) in the lane's order
    const int lane = threadIdx.x & 63;
    for (int g = 0; g < groups; ++g) {
      const int i0 = first + 256 * g + 4 * lane;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (i0 + c < n) f(x[i0 + c], i0 + c);
    }
  }
};

template <bool WEIGHTS, class Passes>
IEK_DEV Kept select(const Row& row, Group& q, u64* hist, const Kept& now, const Weigh& weigh, Passes passes, u64& above) {
  uint32_t prefix = 0;
  u64 sum = 0;
  const uint32_t shifts[3] = {21, 10, 0};
  for (int d = 0; d < 3; ++d) {
    const uint32_t shift = shifts[d], bits = d == 2 ? 10 : 11;
    for (int i = threadIdx.x; i < BINS; i += ST) hist[i] = 0;
    __syncthreads();
    row.each([&](float x, int) {
      const uint32_t k = key_of(x);
      if (k <= now.key || (d > 0 && (k >> (shift + bits)) != prefix)) return;
      atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], WEIGHTS ? weigh(x) : 1ull);
    });
    // of the last key kept so far only its first ones
    if (threadIdx.x == 0 && (d == 0 || (now.key >> (shift + bits)) == prefix) && now.ties > 0)
      atomicAdd(&hist[(now.key >> shift) & ((1u << bits) - 1)], (u64)now.ties * (WEIGHTS ? weigh(value_of(now.key)) : 1ull));
    __syncthreads();
    u64 up;
    const int bin = pick_bin(q, hist, [&](u64 s) { return passes(sum + s); }, up);
    sum += up;
    prefix = prefix << bits | (uint32_t)bin;
  }
  above = sum;
  return Kept{prefix, 0};
}

// How many tokens of one weight the sum `above` them leaves room for below the limit of top-p (the first always).
IEK_DEV int ties_below(double limit, u64 above, u64 weight) {
  const double fit = ceil((limit - (double)above) / (double)weight);
  return fit < 1 ? 1 : fit > 1e9 ? 1000000000 : (int)fit;
}

// A draw of 0 takes the first token of any weight, however small: `any` counts them.
IEK_DEV void any_row(const SampleArgs& a, int b, const Head& h, Smem& m, u64* hist) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  Group q(m);
  __syncthreads();
  Row row{a.logits + (size_t)b * a.stride, a.n, 0, 0};
  row.groups = ((a.n + 255) / 256 + NW - 1) / NW;
  row.first = wave * row.groups * 256;
  const Weigh weigh = weigh_of(h, a.n, m.table);
  Kept kept{0, 0};
  u64 unused;
  if (h.k > 0) {
    u64 above;
    kept = select<false>(row, q, hist, kept, weigh, [&](u64 s) { return s >= (u64)h.k; }, above);
    kept.ties = h.k - (int)above;
  }
  if (h.p < 1.f) {
    u64 total = 0;
    row.each([&](float x, int) {
      if (key_of(x) > kept.key) total += weigh(x);
    });
    total = q.sum(total);
    total += (u64)kept.ties * weigh(value_of(kept.key));
    const double limit = (double)h.p * (double)total;
    u64 above;
    // (of p <= 0 the first token stays)
    const Kept next = select<true>(row, q, hist, kept, weigh, [&](u64 s) { return s > 0 && !((double)s < limit); }, above);
    const int ties = ties_below(limit, above, weigh(value_of(next.key)));
    kept.ties = next.key == kept.key ? min(kept.ties, ties) : ties;
    kept.key = next.key;
  }
  // in index order: each wave's ties, then its sum of kept weights
  int equal = 0;
  row.each([&](float x, int) { equal += kept.ties > 0 && key_of(x) == kept.key; });
  const int seen = __shfl((int)q.before(equal, unused), 0);  // ties before the wave's run
  const double least = fminf(h.m, 1.f);
  auto weight = [&](float x, bool tie_kept, bool any) -> u64 {
    const uint32_t key = key_of(x);
    if (!(key > kept.key || (tie_kept && key == kept.key))) return 0;
    double w = weigh.real(x);
    if (!any) return w >= least ? weigh.whole(w) : 0;
    if (w < 0x1p-60) w = exp(((double)x - weigh.top) / (double)h.t);  // (min_p may be below all that is told apart above)
    return w > 0 && w >= least;
  };
  // one pass over the run, group by group: f(weights of the lane's four, their index)
  auto walk = [&](bool any, auto f) {
    int before = seen;
    for (int g = 0; g < row.groups; ++g) {
      const int i0 = row.first + 256 * g + 4 * lane;
      float x[4];
      int mine = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = i0 + c < row.n ? row.x[i0 + c] : -INFINITY;
        mine += i0 + c < row.n && key_of(x[c]) == kept.key;
      }
      const u64 upto = wave_scan64(mine);
      int rank = before + (int)upto - mine;
      before += (int)__shfl(upto, 63);
      u64 w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool tie = i0 + c < row.n && key_of(x[c]) == kept.key;
        w[c] = i0 + c < row.n ? weight(x[c], tie && rank < kept.ties, any) : 0;
        rank += tie;
      }
      if (f(w, i0)) break;
    }
  };
  auto sums = [&](bool any, u64& mine, u64& base, u64& total) {
    u64 s = 0;
    walk(any, [&](const u64(&w)[4], int) {
      s += w[0] + w[1] + w[2] + w[3];
      return false;
    });
    const u64 upto = wave_scan64(s);
    mine = lane64(upto, 63);
    base = lane64(q.before(s, total), 0);
  };
  u64 mine, base, total, whole;
  sums(false, mine, base, total);
  whole = total;
  if (h.r == 0.f) sums(true, mine, base, total);
  const double limit = (double)h.r * (double)total;
  if ((double)base > limit || !((double)(base + mine) > limit)) return;  // another wave's
  u64 sum = base;
  walk(h.r == 0.f, [&](const u64(&w)[4], int i0) {
    const u64 all = w[0] + w[1] + w[2] + w[3], upto = sum + wave_scan64(all);
    const u64 here = __ballot((double)upto > limit);
    if (here == 0) {
      sum = lane64(upto, 63);
      return false;
    }
    if (lane == __ffsll(here) - 1) {
      u64 s = upto - all;
      int c = 0;
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (c == j && !((double)(s += w[j]) > limit)) c = j + 1;
      store(a, b, (uint32_t)(i0 + c), share(h, weigh, row.x[i0 + c], whole));
    }
    return true;
  });
}

// ---- rows and lists in LDS ----------------------------------------------------------------------------

// Tokens in index order, each thread with a run of 4 * quads of them in a row; -inf behind the last one, up to the last
// thread's. Quad s is stored at s ^ (s >> 3 & 7): the quads that neighbouring threads read at a time, `quads` apart, are
// then in different banks. index: the tokens' indexes, or null: first, first + 1, ...
IEK_DEV int stored(int quad) { return quad ^ (quad >> 3 & 7); }
IEK_DEV int quads_of(int n) { return (n + 4 * ST - 1) / (4 * ST); }
struct Tokens {
  const float4* x;
  const uint32_t* index;
  int quads, first;
  IEK_DEV float value(int i) const { return reinterpret_cast<const float*>(x + stored(i >> 2))[i & 3]; }
  IEK_DEV uint32_t at(int i) const { return index ? index[i] : (uint32_t)(first + i); }
  template <int U = 2, class F>
  IEK_DEV void each(F f) const {  // f(value, place)
#pragma unroll U
    for (int j = 0; j < quads; ++j) {
      const int s = (int)threadIdx.x * quads + j;
      const float4 v = x[stored(s)];
      f(v.x, 4 * s);
      f(v.y, 4 * s + 1);
      f(v.z, 4 * s + 2);
      f(v.w, 4 * s + 3);
    }
  }
};

// A thread's tokens that in(value) holds for, as bits.
template <class In>
IEK_DEV uint32_t bits_of(const Tokens& T, In in) {
  uint32_t bits = 0;
#pragma unroll 4
  for (int j = 0; j < T.quads; ++j) {
    const float4 v = T.x[stored((int)threadIdx.x * T.quads + j)];
    bits |= ((in(v.x) ? 1u : 0u) | (in(v.y) ? 2u : 0u) | (in(v.z) ? 4u : 0u) | (in(v.w) ? 8u : 0u)) << 4 * j;
  }
  return bits;
}
// f(value, place) of these
template <class F>
IEK_DEV void each_of(const Tokens& T, uint32_t bits, F f) {
  for (; bits; bits &= bits - 1) {
    const int i = (int)threadIdx.x * 4 * T.quads + __ffs(bits) - 1;
    f(T.value(i), i);
  }
}

// n <= SLICE logits from p on into LDS; returns the largest of those that the thread loaded, +inf for a NaN. (A
// row's address is a multiple of 4 bytes.)
IEK_DEV float load_tokens(float4* to, const float* p, int n) {
  typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int U = SLICE / (4 * ST);
  const int t = threadIdx.x, quads = quads_of(n);
  f4u_t v[U];
  // all loads first, the last quads from where four are left (a row of fewer than four has no vector to load)
#pragma unroll
  for (int q = 0; q < U; ++q) {
    if (q >= quads) break;  // uniform
    if (n >= 4) {
      v[q] = *reinterpret_cast<const f4u_t*>(p + min(4 * (q * ST + t), n - 4));
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[q][c] = p[min(c, n - 1)];
    }
  }
  float most = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int q = 0; q < U; ++q) {
    if (q >= quads) break;
    const int i = 4 * (q * ST + t);
    float x[4] = {v[q][0], v[q][1], v[q][2], v[q][3]};
    if (4 * ST * (q + 1) > n) {  // uniform: the last ones
      const int s = n >= 4 ? max(0, i - (n - 4)) : 0;  // (the loaded ones begin s before i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float y = v[q][c];
#pragma unroll
        for (int d = 1; d < 4; ++d)
          if (s == d) y = v[q][(c + d) & 3];
        x[c] = i + c < n ? y : -INFINITY;
      }
    }
    to[stored(q * ST + t)] = make_float4(x[0], x[1], x[2], x[3]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      nan |= x[c] != x[c];
      most = fmaxf(most, x[c]);
    }
  }
  return nan ? INFINITY : most;
}

IEK_DEV float steps(float x, float top, float scale) { return fminf((top - x) * scale, (float)(BINS - 1)); }
IEK_DEV int bin_of(float x, float top, float scale) { return (int)steps(x, top, scale); }
// Whether a token is less than `far` steps below the top. Where the span is beyond f32, the scale is 0 and the steps of a
// token as far down are NaN: bin_of counts it in the last bin, so it is within every bound.
IEK_DEV bool within(float x, float top, float scale, float far) {
  const float s = (top - x) * scale;
  return x > -INFINITY && (!(s >= far) || far == INFINITY);
}

IEK_DEV void clear_bins(Smem& m, u64* hist) {
#pragma unroll
  for (int i = 0; i < BINS / ST; ++i) hist[threadIdx.x + ST * i] = 0;
  if (threadIdx.x == 0) {
    m.count = 0;
    m.word2 = -1;
  }
  __syncthreads();
}
// The bin in which the tokens stop being kept: keeps(sum before it, the total), but not all of it; -1 if all are kept.
// above: the sum before it.
template <class Keeps>
IEK_DEV int cross(Group& q, const u64* hist, Keeps keeps, u64& above, u64& total) {
  const int t = threadIdx.x;
  Smem& m = q.m;
  const u64 a = hist[2 * t], b = hist[2 * t + 1];
  const u64 before = q.before(a + b, total);
  if (keeps(before, total) && !keeps(before + a + b, total)) {
    const bool first = !keeps(before + a, total);
    m.word = first ? before : before + a;
    m.word2 = 2 * t + (first ? 0 : 1);
  }
  __syncthreads();
  above = m.word;
  return m.word2;
}

// What is kept: the tokens above `over`, and the first `ties` of those that are it.
struct Cut {
  float over;
  int ties;
};

// Ranks n <= NEAR tokens of s.near against each other, with several threads a token (a power of two up to a wave, their
// parts joined over the lanes): to(token, the sum of those before it, how many those are and how many of them equal it, whether
// it is the last), in the first thread of each.
template <class To>
IEK_DEV void rank(const Bins& s, int n, To to) {
  const int t = threadIdx.x, size = n <= 16 ? 16 : 1 << (32 - __clz(n - 1)), each = ST / size, me = t / each;
  u64 sum = 0;
  int count = 0, equal = 0;
  if (me < n) {
    const u64 mine = s.near[me];
#pragma unroll 4
    for (int j = t & (each - 1); j < n; j += each) {
      const u64 o = s.near[j], w = s.near_w[j];
      const bool before = o > mine;
      sum += before ? w : 0;
      count += before;
      equal += before && (uint32_t)(o >> 32) == (uint32_t)(mine >> 32);
    }
  }
  for (int d = 1; d < each; d <<= 1) {
    sum += __shfl_xor(sum, d);
    count += __shfl_xor(count, d);
    equal += __shfl_xor(equal, d);
  }
  if ((t & (each - 1)) == 0 && me < n) to(me, sum, count, equal);
}

// The border among n <= NEAR tokens of a bin: keeps(the sum before a token). m.border, m.ties: the last value that stays
// and how many of it; m.word: the sum up to it; m.word2: whether it is the last of them. kept(token), for those that stay.
template <class Keeps, class Kept>
IEK_DEV void rank_near(Smem& m, const Bins& s, int n, u64 above, Keeps keeps, Kept kept) {
  rank(s, n, [&](int i, u64 sum, int count, int equal) {
    const u64 own = s.near_w[i];
    sum += above;
    if (keeps(sum)) kept(i);
    const bool last = count == n - 1;
    if (keeps(sum) && (last || !keeps(sum + own))) {
      m.border = value_of((uint32_t)(s.near[i] >> 32));
      m.ties = equal + 1;
      m.word = sum + own;
      m.word2 = last;
    }
  });
  __syncthreads();
}

// Adds up weights (or counts) of the tokens above `over` in bins of 1 / scale from the top.
IEK_DEV void fill_bins(const Tokens& T, u64* hist, const Weigh& weigh, bool counts, float top, float scale, float over) {
  // (the last bin, which may have most of the tokens, from a sum of each wave)
  u64 far = 0;
  T.each([&](float x, int) {
    const u64 all = counts ? 1 : weigh(x), w = x > over ? all : 0;
    const int bin = bin_of(x, top, scale);
    const bool last = bin == BINS - 1;
    far += last ? w : 0;
    if (!last) atomicAdd(&hist[bin], w);
  });
  far = wave_scan64(far);
  if ((threadIdx.x & 63) == 63 && far) atomicAdd(&hist[BINS - 1], far);
}
// Puts the tokens above `over` of a bin into s.near, in any order; m.count of them (more than NEAR: not all are there).
IEK_DEV void gather_near(const Tokens& T, Smem& m, Bins& s, const Weigh& weigh, bool counts, float top, float scale, float over, int bin) {
  const uint32_t bits = bits_of(T, [&](float x) { return x > over && bin_of(x, top, scale) == bin; });
  each_of(T, bits, [&](float x, int i) {
    const int at = atomicAdd(&m.count, 1);
    if (at < NEAR) {
      s.near[at] = (u64)key_of(x) << 32 | (uint32_t)~T.at(i);
      s.near_w[at] = counts ? 1 : weigh(x);
    }
  });
  __syncthreads();
}

// Cuts the tokens kept to those that keeps(the sum before them, the total). False: the bin of the border has too many
// tokens. counts: sums are of tokens, not of weights. (Of now.over only now.ties stay.)
template <class Keeps>
IEK_DEV bool cut_at(const Tokens& T, Group& q, Bins& s, const Weigh& weigh, bool counts, float top, float scale, Cut& now, Keeps keeps) {
  Smem& m = q.m;
  clear_bins(m, s.hist);
  fill_bins(T, s.hist, weigh, counts, top, scale, now.over);
  const int tie_bin = now.ties > 0 ? bin_of(now.over, top, scale) : -1;
  const u64 tie_w = now.ties > 0 ? (counts ? 1 : weigh(now.over)) : 0;
  if (threadIdx.x == 0 && now.ties > 0) atomicAdd(&s.hist[tie_bin], tie_w * (u64)now.ties);
  __syncthreads();
  u64 above, total;
  const int bin = cross(q, s.hist, keeps, above, total);
  if (bin < 0) return true;  // all of them
  gather_near(T, m, s, weigh, counts, top, scale, now.over, bin);
  const int n = m.count;
  if (n > NEAR) return false;
  if (threadIdx.x == 0) {
    m.word2 = n == 0;
    m.word = above;
  }
  __syncthreads();
  rank_near(m, s, n, above, [&](u64 v) { return keeps(v, total); }, [](int) {});
  // all of the bin's, and some of the value that was the last one before
  const u64 sum = m.word;
  if (m.word2 && bin == tie_bin && keeps(sum, total)) {
    // (the sums before them are sum + j tie_w)
    int lo = 0, hi = now.ties;  // keeps(lo); not keeps(hi), or hi is all of them
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      (keeps(sum + tie_w * (u64)mid, total) ? lo : hi) = mid;
    }
    now.ties = lo + 1;
  } else {
    now = Cut{m.border, m.ties};
  }
  __syncthreads();
  return true;
}

// How a row's tokens are weighed at the end: those kept, if not below min-p.
struct Final {
  Weigh weigh;
  double least;
  Cut cut;
  u64 tie_w;
  IEK_DEV Final(const Weigh& w, const Head& h, const Cut& c) : weigh(w), least(fminf(h.m, 1.f)), cut(c), tie_w(0) {
    if (c.ties > 0) tie_w = weight(c.over);
  }
  IEK_DEV u64 weight(float x) const {
    const double w = weigh.real(x);
    return w >= least ? weigh.whole(w) : 0;
  }
};

// The thread's sum of kept weights. ties: how many of the value `over` come before its run.
IEK_DEV u64 run_sum(const Tokens& T, Group& q, const Final& f, int& ties) {
  u64 sum = 0;
  int equal = 0;
  for (int j = 0; j < T.quads; ++j) {
    const float4 v = T.x[stored((int)threadIdx.x * T.quads + j)];
    const float x[4] = {v.x, v.y, v.z, v.w};
    const float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if (f.cut.ties > 0) equal += (x[0] == f.cut.over) + (x[1] == f.cut.over) + (x[2] == f.cut.over) + (x[3] == f.cut.over);
    if (!__any(most > f.cut.over)) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const u64 w = f.weight(x[c]);
      sum += x[c] > f.cut.over ? w : 0;
    }
  }
  ties = 0;
  if (f.cut.ties > 0) {
    u64 unused;
    ties = (int)q.before(equal, unused);
    sum += f.tie_w * (u64)max(0, min(f.cut.ties - ties, equal));
  }
  return sum;
}
// Stores the token of T at which the running sum first exceeds the limit: `base` before the thread's run, `sum` in it.
IEK_DEV void pick_in_run(const Tokens& T, const Final& f, u64 base, u64 sum, int ties, double limit, const SampleArgs& a, int b, const Head& h,
                         u64 total) {
  const unsigned long long here = __ballot(!((double)base > limit) && (double)(base + sum) > limit);
  if (here == 0) return;  // another wave's
  // the wave goes through that thread's run, a token a lane
  const int owner = __ffsll(here) - 1, lane = threadIdx.x & 63, per = 4 * T.quads;
  const int i = (((int)threadIdx.x & ~63) + owner) * per + min(lane, per - 1);
  const float x = T.value(i);
  const bool live = lane < per, tie = live && f.cut.ties > 0 && x == f.cut.over;
  const int rank = __builtin_amdgcn_readlane(ties, owner) + __popcll(__ballot(tie) & ((1ull << lane) - 1));
  const u64 w = live && x > f.cut.over ? f.weight(x) : tie && rank < f.cut.ties ? f.tie_w : 0;
  const u64 upto = lane64(base, owner) + wave_scan64(w);
  const unsigned long long past = __ballot(live && (double)upto > limit);
  if (past != 0 && lane == __ffsll(past) - 1) store(a, b, T.at(i), share(h, f.weigh, x, total));
}

// The token of a row, of tokens T cut to `cut`.
IEK_DEV void pick(const Tokens& T, Group& q, const SampleArgs& a, int b, const Head& h, const Weigh& weigh, const Cut& cut) {
  const Final f(weigh, h, cut);
  int ties;
  const u64 sum = run_sum(T, q, f, ties);
  u64 total;
  const u64 base = q.before(sum, total);
  pick_in_run(T, f, base, sum, ties, (double)h.r * (double)total, a, b, h, total);
}

// A list of tokens in LDS, in index order, and its room.
struct List {
  float4* x;
  uint32_t* index;
  IEK_DEV void put(int at, float v, uint32_t i) const {
    reinterpret_cast<float*>(x + stored(at >> 2))[at & 3] = v;
    index[at] = i;
  }
  // the list of n as tokens
  IEK_DEV Tokens tokens(int n) const {
    for (int i = n + (int)threadIdx.x; i < LIST; i += ST) put(i, -INFINITY, 0);
    for (int i = LIST / 4 + (int)threadIdx.x; i < ST; i += ST) x[stored(i)] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    __syncthreads();
    return Tokens{x, index, 1, 0};
  }
};
constexpr int LIST_BYTES = 16 * ST + 4 * LIST;

// The tokens that in(value) holds for, in index order, to put(place, value, index), if there are at most `room`; returns
// how many there are.
template <class In, class Put>
IEK_DEV int compact(const Tokens& T, Group& q, int room, In in, Put put) {
  const uint32_t bits = bits_of(T, in);
  u64 total;
  int at = (int)q.before(__popc(bits), total);
  if ((int)total <= room) each_of(T, bits, [&](float v, int i) { put(at++, v, T.at(i)); });
  return (int)total;
}

// A bound on the distance of the first k tokens, as steps below `far` of 1 / scale from the top. most: the largest of a
// thread's share of the tokens.
IEK_DEV float bound_of_k(Group& q, u64* hist, float most, int k, float top, float& scale) {
  // bins from the largest to the least of the threads' largest
  const float span = q.most(most > -INFINITY ? top - most : 0.f);
  scale = fminf((float)(BINS - 1) / span, 1e30f);  // (a span of 0: 1e30)
  clear_bins(q.m, hist);
  if (most > -INFINITY) atomicAdd(&hist[bin_of(most, top, scale)], 1ull);
  __syncthreads();
  u64 above, all;
  const int bin = cross(q, hist, [&](u64 v, u64) { return v < (u64)k; }, above, all);
  return bin < 0 ? INFINITY : (float)(bin + 1);  // (no bin: fewer than k threads have any)
}

// The token of a row whose n <= NEAR tokens that may be kept are the list: all of them ranked against each other.
IEK_DEV void pick_of_few(const Tokens& T, int n, Group& q, Bins& s, const SampleArgs& a, int b, const Head& h, const Weigh& weigh) {
  const int t = threadIdx.x;
  const bool live = t < n;
  const float x = live ? T.value(t) : -INFINITY;
  const double real = weigh.real(x);
  const u64 w = live ? weigh.whole(real) : 0;
  if (live) {
    s.near[t] = (u64)key_of(x) << 32 | (uint32_t)~T.at(t);
    s.near_w[t] = w;
  }
  __syncthreads();
  rank(s, n, [&](int i, u64 sum, int count, int) {
    s.hist[i] = sum;
    s.hist[NEAR + i] = (u64)count;
  });
  __syncthreads();
  const u64 above = live ? s.hist[t] : 0;
  const bool first = live && (h.k <= 0 || (int)s.hist[NEAR + t] < h.k);
  bool kept = first && real >= fminf(h.m, 1.f);
  if (h.p < 1.f) {
    const u64 all = q.sum(first ? w : 0);
    kept &= above == 0 || (double)above < (double)h.p * (double)all;
  }
  u64 total;
  const u64 base = q.before(kept ? w : 0, total);
  const double limit = (double)h.r * (double)total;
  if (kept && !((double)base > limit) && (double)(base + w) > limit) store(a, b, T.at(t), share(h, weigh, x, total));
}

// What top-k and top-p keep of T. False: it is left to any_row.
IEK_DEV bool filter(const Tokens& T, Group& q, Bins& s, const Head& h, const Weigh& weigh, float k_scale, float p_scale, Cut& cut) {
  if (h.k > 0 && !cut_at(T, q, s, weigh, true, h.top, k_scale, cut, [&](u64 v, u64) { return v < (u64)h.k; })) return false;
  return !(h.p < 1.f) ||
         cut_at(T, q, s, weigh, false, h.top, p_scale, cut, [&](u64 v, u64 all) { return v == 0 || (double)v < (double)h.p * (double)all; });
}

IEK_DEV float list_scale(float span) { return fminf((float)(BINS - 1) / span, 1e30f); }  // (a span of 0: 1e30)
IEK_DEV float weight_scale(const Head& h) { return fminf(64.f * 1.44269504f / h.t, 1e30f); }

// The lowest index of the largest logit, by one thread of the workgroup.
IEK_DEV void store_top(const Tokens& T, Group& q, const SampleArgs& a, int b, float top) {
  int at = INT32_MAX;
  T.each([&](float x, int i) { at = x == top ? min(at, i) : at; });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) at = min(at, __shfl_xor(at, d));
  u64 total;
  const u64 before = q.before((threadIdx.x & 63) == 0 && at != INT32_MAX, total);
  if ((threadIdx.x & 63) == 0 && at != INT32_MAX && before == 0) store(a, b, T.at(at), 1.f);
}

// The token of a row of up to SLICE logits, which are in `data`. False: it is left to any_row. The list takes the
// histogram's place after it, and the bins then the tokens'.
IEK_DEV bool one_row(const SampleArgs& a, int b, const Head& h, Group& q, float4* data, char* more, float most) {
  const Tokens T{data, nullptr, quads_of(a.n), 0};
  const Weigh weigh = weigh_of(h, a.n, q.m.table);
  Bins& bins = *reinterpret_cast<Bins*>(more);
  const List list{reinterpret_cast<float4*>(more), reinterpret_cast<uint32_t*>(more + 16 * ST)};
  Bins& room = *reinterpret_cast<Bins*>(data);
  auto put = [&](int at, float v, uint32_t i) { list.put(at, v, i); };
  Cut cut{-INFINITY, 0};
  float scale = 0.f, far = -1.f;
  if (h.k > 0 && (h.k <= ST || a.n <= LIST)) {
    far = bound_of_k(q, bins.hist, most, min(h.k, ST), h.top, scale);
  } else if (h.k <= 0 && !(h.p < 1.f) && h.m > 0.f) {
    // (a distance that is too large by the roundings at least: min-p itself is looked at later)
    scale = 1.f;
    far = -logf(fminf(h.m, 1.f)) * h.t * 1.0001f + 1e-6f * fabsf(h.top) + 1e-30f;
  }
  if (far >= 0.f) {
    const int n = compact(T, q, LIST, [&](float v) { return within(v, h.top, scale, far); }, put);
    if (n <= LIST) {
      const Tokens L = list.tokens(n);
      if (n <= NEAR) {
        pick_of_few(L, n, q, room, a, b, h, weigh);
        return true;
      }
      if (far < INFINITY) scale = fminf(scale * ((float)BINS / far), 1e30f);
      if (!filter(L, q, room, h, weigh, scale, scale, cut)) return false;
      pick(L, q, a, b, h, weigh, cut);
      return true;
    }
  }
  if (h.k > 0) {
    float span = 0.f;
    T.each([&](float x, int) { span = x > -INFINITY ? fmaxf(span, h.top - x) : span; });
    scale = fminf((float)(BINS - 1) / q.most(span), 1e30f);
  }
  if (!filter(T, q, bins, h, weigh, scale, weight_scale(h), cut)) return false;
  Tokens left = T;
  if (cut.ties > 0) {
    const int n = compact(T, q, LIST, [&](float v) { return v >= cut.over; }, put);
    if (n <= LIST) left = list.tokens(n);
  }
  pick(left, q, a, b, h, weigh, cut);
  return true;
}

// Rows of up to SLICE logits.
__global__ __launch_bounds__(ST) void row_kernel(SampleArgs a) {
  __shared__ Smem m;
  __shared__ float4 data[SLICE / 4];
  __shared__ __align__(16) char more[sizeof(Bins) > LIST_BYTES ? sizeof(Bins) : LIST_BYTES];
  const int b = blockIdx.x;
  const SampleParams o = params_of(a, b);
  Group q(m);
  const float most = load_tokens(data, a.logits + (size_t)b * a.stride, a.n);
  fill_table(m.table);
  const Head h = head_of(o, a.n, q.most(most));
  if (!h.good) {
    if (threadIdx.x == 0) store(a, b, NO_TOKEN, NAN);
  } else if (h.t == 0.f) {
    store_top(Tokens{data, nullptr, quads_of(a.n), 0}, q, a, b, h.top);
  } else if (h.r == 0.f || !one_row(a, b, h, q, data, more, most)) {
    any_row(a, b, h, m, reinterpret_cast<Bins*>(more)->hist);
  }
}

// ---- rows of several slices -----------------------------------------------------------------------------

// Candidates of a slice, slices of a row at most (one a thread of the last launch).
constexpr int SEGMENT = 256, MOST_SLICES = ST;

// A row in slices of `length` logits, and its part of the workspace.
struct Slices {
  int length, count;
  size_t bytes;  // of a row
  char* base;
};
struct RowSpace {
  u64 *hist, *near, *near_w, *sum;   // [BINS], [NEAR], [NEAR], [slices]
  float *most, *least;               // [slices]: the largest logit, and the least of the threads' largest
  int* found;                        // [slices]: candidates; [slices]: tokens of the border's bin
  float* x;                          // [slices][SEGMENT] candidates
  uint32_t* index;
};
IEK_DEV RowSpace space_of(const Slices& z, int b) {
  char* p = z.base + (size_t)b * z.bytes;
  const size_t n = (size_t)z.count;
  RowSpace r;
  r.hist = reinterpret_cast<u64*>(p);
  r.near = r.hist + BINS;
  r.near_w = r.near + NEAR;
  r.sum = r.near_w + NEAR;
  r.most = reinterpret_cast<float*>(r.sum + n);
  r.least = r.most + n;
  r.found = reinterpret_cast<int*>(r.least + n);
  r.x = reinterpret_cast<float*>(r.found + n + 1);
  r.index = reinterpret_cast<uint32_t*>(r.x + n * SEGMENT);
  return r;
}
// Which rows go which way (the others are left to the last launch, to any_row).
IEK_DEV bool by_list(const Head& h) { return h.k > 0 && h.k <= ST; }
IEK_DEV bool by_slices(const Head& h) { return h.good && h.t > 0.f && h.r > 0.f && h.k <= ST; }

// What a workgroup takes of the row's part first, all of it at once and ahead of its logits; from these the row's head and
// the span of the threads' maxima.
struct Early {
  SampleParams o;
  float most, least;
};
IEK_DEV Early early_of(const SampleArgs& a, const Slices& z, int b, const RowSpace& r) {
  const int t = threadIdx.x;
  return Early{params_of(a, b), t < z.count ? r.most[t] : -INFINITY, t < z.count ? r.least[t] : INFINITY};
}
IEK_DEV Head head_of_slices(const SampleArgs& a, const Slices& z, const Early& e, Group& q, float& span) {
  const float top = q.most(e.most);
  span = q.most((int)threadIdx.x < z.count ? top - e.least : 0.f);
  return head_of(e.o, a.n, top);
}
IEK_DEV float load_slice(float4* to, const SampleArgs& a, const Slices& z, int b, int s, Tokens& T) {
  const int first = s * z.length, n = min(z.length, a.n - first);
  T = Tokens{to, nullptr, quads_of(n), first};
  return load_tokens(to, a.logits + (size_t)b * a.stride + first, n);
}

// First launch: the slices' maxima; the row's histogram and counter are cleared.
__global__ __launch_bounds__(ST) void slice_most_kernel(SampleArgs a, Slices z) {
  __shared__ Smem m;
  __shared__ float4 data[SLICE / 4];
  const int b = blockIdx.y, s = blockIdx.x, t = threadIdx.x;
  const RowSpace r = space_of(z, b);
  for (int i = s * ST + t; i < BINS; i += z.count * ST) r.hist[i] = 0;
  if (s == 0 && t == 0) r.found[z.count] = 0;
  Group q(m);
  Tokens T;
  const float most = load_slice(data, a, z, b, s, T), top = q.most(most);
  const float span = q.most(most > -INFINITY ? top - most : 0.f);
  if (t == 0) {
    r.most[s] = top;
    r.least[s] = top > -INFINITY ? top - span : INFINITY;  // (a slice of nothing has no say)
  }
}

// Second: the row's histogram, of the threads' maxima (top-k) or of weights (top-p); or the slice's sum of weights.
__global__ __launch_bounds__(ST) void slice_bins_kernel(SampleArgs a, Slices z) {
  __shared__ Smem m;
  __shared__ float4 data[SLICE / 4];
  __shared__ u64 hist[BINS];
  const int b = blockIdx.y, s = blockIdx.x, t = threadIdx.x;
  const RowSpace r = space_of(z, b);
  const Early e = early_of(a, z, b, r);
  Group q(m);
  Tokens T;
  const float most = load_slice(data, a, z, b, s, T);
  fill_table(m.table);
  float span;
  const Head h = head_of_slices(a, z, e, q, span);
  if (!by_slices(h)) return;
  const Weigh weigh = weigh_of(h, a.n, m.table);
  if (!by_list(h) && !(h.p < 1.f)) {
    int ties;
    const u64 sum = q.sum(run_sum(T, q, Final(weigh, h, Cut{-INFINITY, 0}), ties));
    if (t == 0) r.sum[s] = sum;
    return;
  }
  clear_bins(m, hist);
  if (by_list(h)) {
    if (most > -INFINITY) atomicAdd(&hist[bin_of(most, h.top, list_scale(span))], 1ull);
  } else {
    fill_bins(T, hist, weigh, false, h.top, weight_scale(h), -INFINITY);
  }
  __syncthreads();
  for (int i = t; i < BINS; i += ST)
    if (hist[i]) atomicAdd(&r.hist[i], hist[i]);
}

// The bin of the row's histogram (`bins`: the thread's of it) that the border is in; into m.hist's copy.
constexpr int PER = BINS / ST;
IEK_DEV void bins_of(const RowSpace& r, u64 (&bins)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; ++i) bins[i] = r.hist[threadIdx.x + i * ST];
}
IEK_DEV int cross_row(const Head& h, const u64 (&bins)[PER], Group& q, u64* hist, u64& above, u64& total) {
  clear_bins(q.m, hist);
#pragma unroll
  for (int i = 0; i < PER; ++i) hist[threadIdx.x + i * ST] = bins[i];
  __syncthreads();
  const bool list = by_list(h);
  return cross(q, hist, [&](u64 v, u64 all) { return list ? v < (u64)h.k : v == 0 || (double)v < (double)h.p * (double)all; }, above, total);
}

// Third: the slice's candidates for top-k; or its sum of the weights above top-p's bin, and its tokens in that.
__global__ __launch_bounds__(ST) void slice_cut_kernel(SampleArgs a, Slices z) {
  __shared__ Smem m;
  __shared__ float4 data[SLICE / 4];
  __shared__ Bins bins;
  const int b = blockIdx.y, s = blockIdx.x, t = threadIdx.x;
  const RowSpace r = space_of(z, b);
  const Early e = early_of(a, z, b, r);
  u64 row[PER];
  bins_of(r, row);
  Group q(m);
  Tokens T;
  load_slice(data, a, z, b, s, T);
  fill_table(m.table);
  float span;
  const Head h = head_of_slices(a, z, e, q, span);
  if (!by_slices(h) || (!by_list(h) && !(h.p < 1.f))) return;
  u64 above, total;
  const int bin = cross_row(h, row, q, bins.hist, above, total);
  if (by_list(h)) {
    const float scale = list_scale(span), far = bin < 0 ? INFINITY : (float)(bin + 1);
    float* x = r.x + (size_t)s * SEGMENT;
    uint32_t* index = r.index + (size_t)s * SEGMENT;
    const int n = compact(T, q, SEGMENT, [&](float v) { return within(v, h.top, scale, far); },
                          [&](int at, float v, uint32_t i) {
                            x[at] = v;
                            index[at] = i;
                          });
    if (t == 0) r.found[s] = n;
    return;
  }
  // (top-p below 1: some bin is the border's)
  const Weigh weigh = weigh_of(h, a.n, m.table);
  const Final f(weigh, h, Cut{-INFINITY, 0});
  const float scale = weight_scale(h);
  u64 sum = 0;
  const uint32_t over = bits_of(T, [&](float x) { return x > -INFINITY && bin_of(x, h.top, scale) < bin; });
  each_of(T, over, [&](float x, int) { sum += f.weight(x); });
  sum = q.sum(sum);
  if (t == 0) r.sum[s] = sum;
  const uint32_t at_border = bits_of(T, [&](float x) { return x > -INFINITY && bin_of(x, h.top, scale) == bin; });
  each_of(T, at_border, [&](float x, int i) {
    const int at = atomicAdd(&r.found[z.count], 1);
    if (at < NEAR) {
      r.near[at] = (u64)key_of(x) << 32 | (uint32_t)~T.at(i);
      r.near_w[at] = weigh(x);
    }
  });
}

// The token of a row of slices. False: it is left to any_row.
struct Joined {
  u64 bins[PER], near, near_w, sum;  // (near: of a row that has them; the thread's sum is its slice's)
  int found, border;
};
IEK_DEV bool join_slices(const SampleArgs& a, const Slices& z, int b, const Head& h, const RowSpace& r, const Joined& e, Group& q, float4* data, char* more) {
  const int t = threadIdx.x;
  Smem& m = q.m;
  Bins& bins = *reinterpret_cast<Bins*>(more);
  const Weigh weigh = weigh_of(h, a.n, m.table);
  if (by_list(h)) {
    const List list{reinterpret_cast<float4*>(more), reinterpret_cast<uint32_t*>(more + 16 * ST)};
    Bins& room = *reinterpret_cast<Bins*>(data);
    const int mine = t < z.count ? e.found : 0;
    u64 total, most;
    const int at = (int)q.before(mine, total);
    q.before(mine > SEGMENT, most);
    if (most > 0 || total > LIST) return false;
    // the waves take the segments in turn: their places and counts through LDS
    int2* seg = reinterpret_cast<int2*>(data);
    if (t < z.count) seg[t] = int2{at, mine};
    __syncthreads();
    for (int i = t >> 6; i < z.count; i += NW) {
      const int2 g = seg[i];
      for (int j = t & 63; j < g.y; j += 64) list.put(g.x + j, r.x[(size_t)i * SEGMENT + j], r.index[(size_t)i * SEGMENT + j]);
    }
    __syncthreads();
    const int n = (int)total;
    const Tokens L = list.tokens(n);
    if (n <= NEAR) {
      pick_of_few(L, n, q, room, a, b, h, weigh);
      return true;
    }
    Cut cut{-INFINITY, 0};
    float low = 0.f;
    L.each([&](float x, int) { low = x > -INFINITY ? fmaxf(low, h.top - x) : low; });
    const float scale = list_scale(q.most(low));
    if (!filter(L, q, room, h, weigh, scale, scale, cut)) return false;
    pick(L, q, a, b, h, weigh, cut);
    return true;
  }
  Cut cut{-INFINITY, 0};
  u64 mine = t < z.count ? e.sum : 0;
  const float least = fminf(h.m, 1.f);
  if (h.p < 1.f) {
    u64 above, total;
    cross_row(h, e.bins, q, bins.hist, above, total);
    const int n = e.border;
    if (n > NEAR) return false;
    if (t < n) {
      bins.near[t] = e.near;
      bins.near_w[t] = e.near_w;
    }
    u64* add = bins.hist;  // (of each slice, the kept ones of these)
    __syncthreads();
    add[t] = 0;
    __syncthreads();
    rank_near(m, bins, n, above, [&](u64 v) { return v == 0 || (double)v < (double)h.p * (double)total; }, [&](int i) {
      if (weigh.real(value_of((uint32_t)(bins.near[i] >> 32))) >= least)
        atomicAdd(&add[~(uint32_t)bins.near[i] / (uint32_t)z.length], bins.near_w[i]);
    });
    cut = Cut{m.border, m.ties};
    mine += add[t];
  }
  // the slice that has the token
  u64 total;
  const u64 base = q.before(mine, total);
  const double limit = (double)h.r * (double)total;
  if (!((double)base > limit) && (double)(base + mine) > limit) {
    m.word = base;
    m.word2 = t;
  }
  __syncthreads();
  const u64 from = m.word;
  const int s = m.word2;
  if (cut.ties > 0) {  // the kept ties before it
    const uint32_t index = t < e.border ? ~(uint32_t)bins.near[t] : 0xFFFFFFFFu;
    const bool tie = t < e.border && value_of((uint32_t)(bins.near[t] >> 32)) == cut.over && index < (uint32_t)(s * z.length);
    cut.ties = max(0, cut.ties - (int)q.sum(tie));
  }
  Tokens T;
  load_slice(data, a, z, b, s, T);
  __syncthreads();
  const Final f(weigh, h, cut);
  int ties;
  const u64 sum = run_sum(T, q, f, ties);
  u64 unused;
  const u64 before = from + q.before(sum, unused);
  pick_in_run(T, f, before, sum, ties, limit, a, b, h, total);
  return true;
}

// Fourth: a workgroup a row.
__global__ __launch_bounds__(ST) void slice_join_kernel(SampleArgs a, Slices z) {
  __shared__ Smem m;
  __shared__ float4 data[SLICE / 4];
  __shared__ __align__(16) char more[sizeof(Bins) > LIST_BYTES ? sizeof(Bins) : LIST_BYTES];
  const int b = blockIdx.x;
  const RowSpace r = space_of(z, b);
  // (what a row has no use for, or what nobody wrote, is not looked at)
  const int t = threadIdx.x, c = min(t, z.count - 1), near = min(t, NEAR - 1);
  const Early first = early_of(a, z, b, r);
  Joined e;
  bins_of(r, e.bins);
  e.near = r.near[near];
  e.near_w = r.near_w[near];
  e.sum = r.sum[c];
  e.found = r.found[c];
  e.border = r.found[z.count];
  Group q(m);
  fill_table(m.table);
  float span;
  const Head h = head_of_slices(a, z, first, q, span);
  if (!h.good) {
    if (threadIdx.x == 0) store(a, b, NO_TOKEN, NAN);
  } else if (h.t == 0.f) {
    // the first slice that has the maximum
    u64 total;
    const bool has = t < z.count && first.most == h.top;
    if (q.before(has, total) == 0 && has) m.word2 = t;
    __syncthreads();
    Tokens T;
    load_slice(data, a, z, b, m.word2, T);
    __syncthreads();
    store_top(T, q, a, b, h.top);
  } else if (!by_slices(h) || !join_slices(a, z, b, h, r, e, q, data, more)) {
    any_row(a, b, h, m, reinterpret_cast<Bins*>(more)->hist);
  }
}

}  // namespace

void check_sample_params(const SampleParams& p) {
  if (!std::isfinite(p.temperature) || p.temperature < 0.0f)
    fail(ST_SAMPLING, "temperature must not be negative, got " + std::to_string(p.temperature));
  if (!(p.r >= 0.0f && p.r < 1.0f)) fail(ST_OP, "sample: the uniform draw must be in [0, 1)");
  if (std::isnan(p.top_p) || std::isnan(p.min_p)) fail(ST_OP, "sample: a filter is NaN");
}

// Slices of a row: as many workgroups as fill the chip, of whole quads of all threads. (8 rows of 262144: slices of 8192.)
static Slices slices_of(size_t rows, size_t n) {
  constexpr size_t unit = 4 * ST;
  Slices z{};
  if (n <= SLICE) return z;
  const size_t fill = (n * rows / 256 + unit - 1) / unit * unit, least = (n / MOST_SLICES + unit) / unit * unit;
  z.length = (int)std::min<size_t>(SLICE, std::max({fill, least, 2 * unit}));
  z.count = (int)((n + z.length - 1) / z.length);
  z.bytes = (8 * (BINS + 2 * NEAR + (size_t)z.count) + 8 * (size_t)z.count + 4 * ((size_t)z.count + 1) + 8 * (size_t)SEGMENT * z.count + 15) / 16 * 16;
  return z;
}

size_t sample_workspace(size_t rows, size_t n) {
  if (n == 0) fail(ST_SAMPLING, "logits slice is empty");
  if (n > (size_t)SLICE * MOST_SLICES || rows > (1u << 21)) fail(ST_OP, "sample: dims too large");
  const Slices z = slices_of(rows, n);
  return rows * z.bytes;
}

void launch_sample(const SampleArgs& a, int rows, void* ws, hipStream_t st) {
  Slices z = slices_of((size_t)rows, (size_t)a.n);
  if (z.count == 0) {
    hipLaunchKernelGGL(row_kernel, dim3((unsigned)rows), dim3(ST), 0, st, a);
    return;
  }
  z.base = static_cast<char*>(ws);
  // (a grid's second dimension has 65535 at most)
  for (int b = 0; b < rows; b += 65535) {
    const int some = std::min(rows - b, 65535);
    SampleArgs x = a;
    x.logits += (size_t)b * a.stride;
    x.index += b;
    if (x.prob) x.prob += b;
    for (const float** p : {&x.temperature, &x.top_p, &x.min_p, &x.r})
      if (*p) *p += b;
    if (x.top_k) x.top_k += b;
    const dim3 grid((unsigned)z.count, (unsigned)some);
    hipLaunchKernelGGL(slice_most_kernel, grid, dim3(ST), 0, st, x, z);
    hipLaunchKernelGGL(slice_bins_kernel, grid, dim3(ST), 0, st, x, z);
    hipLaunchKernelGGL(slice_cut_kernel, grid, dim3(ST), 0, st, x, z);
    hipLaunchKernelGGL(slice_join_kernel, dim3((unsigned)some), dim3(ST), 0, st, x, z);
    z.base += (size_t)some * z.bytes;
  }
}

}  // namespace iek
