// Sampling with temperature, top-k, top-p and min-p, a row of logits per sequence (iek_dev_sample).
//
// Of a row with maximum M, token i has the weight w_i = exp((l_i - M) / T). The filters keep a prefix of the tokens
// in descending order (equal ones: the lower index first):
//   top-k: the first k;  top-p: of those the ones before which the sum of weights is below p times their total;
//   min-p: the ones with w_i >= min_p (M's token has 1).
// The pick is the first token in index order up to which the kept weights sum to more than r times their total.
//
// Weights are summed as integers, w 2^S rounded, with S as large as n of them allow in 64 bits: sums do not depend on
// their order, so atomics on histograms and any split give the same token every time, and a weight is off by 2^-S-1
// of the largest (2^-48 at 32000 tokens), where f32 sums would move the borders of tokens by 1e-7 of the total.
// A prefix is found by a radix selection on the logits' bits as ordered integers, 11, 11 and 10 bits at a time, of
// counts (top-k) or of weights (top-p).
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

// Weights of a row: w 2^S as an integer.
struct Weigh {
  double top, inv, one;  // one = 2^S
  IEK_DEV double real(float x) const { return exp(((double)x - top) * inv); }
  IEK_DEV u64 operator()(float x) const { return (u64)(real(x) * one + 0.5); }
};

IEK_DEV u64 wave_sum64(u64 v) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) v += __shfl_xor(v, s);
  return v;
}
// Inclusive prefix sum over the lanes.
IEK_DEV u64 wave_scan64(u64 v) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const u64 up = __shfl_up(v, s);
    if ((int)(threadIdx.x & 63) >= s) v += up;
  }
  return v;
}

struct Smem {
  u64 hist[BINS];
  u64 part[NW];
  u64 word;
  int word2;
};

// The bin, from the top, in which the running sum of the histogram passes `need`, and the sum above it: the first
// with above + hist > need (strictly) if STRICT, else >= need. (Some bin does.)
template <class Passes>
IEK_DEV int pick_bin(Smem& m, Passes passes, u64& above) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // thread t: bins BINS - 1 - 2 t and the next below
  const u64 a = m.hist[BINS - 1 - 2 * t], b = m.hist[BINS - 2 - 2 * t];
  const u64 incl = wave_scan64(a + b);
  if (lane == 63) m.part[wave] = incl;
  __syncthreads();
  u64 base = 0;
  for (int w = 0; w < wave; ++w) base += m.part[w];
  const u64 before = base + incl - a - b;
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

// What a row keeps: the keys above `key` and the first `ties` of those that are it.
struct Kept {
  uint32_t key;
  int ties;
};

// A wave's run of the row: Q groups of 256 logits, four a lane.
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
IEK_DEV Kept select(const Row& row, Smem& m, const Kept& now, const Weigh& weigh, Passes passes, u64& above) {
  uint32_t prefix = 0;
  u64 sum = 0;
  const uint32_t shifts[3] = {21, 10, 0};
  for (int d = 0; d < 3; ++d) {
    const uint32_t shift = shifts[d], bits = d == 2 ? 10 : 11;
    for (int i = threadIdx.x; i < BINS; i += ST) m.hist[i] = 0;
    __syncthreads();
    row.each([&](float x, int) {
      const uint32_t k = key_of(x);
      if (k <= now.key || (d > 0 && (k >> (shift + bits)) != prefix)) return;
      atomicAdd(&m.hist[(k >> shift) & ((1u << bits) - 1)], WEIGHTS ? weigh(x) : 1ull);
    });
    // of the last key kept so far only its first ones
    if (threadIdx.x == 0 && (d == 0 || (now.key >> (shift + bits)) == prefix) && now.ties > 0)
      atomicAdd(&m.hist[(now.key >> shift) & ((1u << bits) - 1)], (u64)now.ties * (WEIGHTS ? weigh(value_of(now.key)) : 1ull));
    __syncthreads();
    u64 up;
    const int bin = pick_bin(m, [&](u64 s) { return passes(sum + s); }, up);
    sum += up;
    prefix = prefix << bits | (uint32_t)bin;
  }
  above = sum;
  return Kept{prefix, 0};
}

__global__ __launch_bounds__(ST) void sample_kernel(SampleArgs a) {
  __shared__ Smem m;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, b = blockIdx.x;
  Row row{a.logits + (size_t)b * a.stride, a.n, 0, 0};
  row.groups = ((a.n + 255) / 256 + NW - 1) / NW;
  row.first = wave * row.groups * 256;
  SampleParams o = a.one;
  if (a.temperature) o = {a.temperature[b], a.top_p ? a.top_p[b] : 1.f, a.min_p ? a.min_p[b] : 0.f, a.r[b], a.top_k ? a.top_k[b] : 0};
  const float temp = o.temperature, r = o.r, p = o.top_p;
  const int k = o.top_k;
  // the largest logit and its lowest index; a NaN counts as the largest
  u64 best = 0;
  row.each([&](float x, int i) {
    const u64 v = (u64)(x != x ? 0xFFFFFFFFu : key_of(x)) << 32 | (uint32_t)~i;
    best = best > v ? best : v;
  });
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const u64 o = __shfl_xor(best, s);
    best = best > o ? best : o;
  }
  if (lane == 0) m.part[wave] = best;
  __syncthreads();
  for (int w = 0; w < NW; ++w) best = best > m.part[w] ? best : m.part[w];
  __syncthreads();
  const uint32_t top_key = (uint32_t)(best >> 32);
  const float top = value_of(top_key);
  // (a NaN parameter fails its comparison)
  const bool good = top_key != 0xFFFFFFFFu && fabsf(top) < INFINITY && temp >= 0.f && temp < INFINITY && r >= 0.f && r < 1.f &&
                    p == p && o.min_p == o.min_p;
  if (!good || temp == 0.f) {
    if (t == 0) {
      a.index[b] = good ? ~(uint32_t)best : NO_TOKEN;
      if (a.prob) a.prob[b] = good ? 1.f : NAN;
    }
    return;
  }
  const Weigh weigh{(double)top, 1.0 / (double)temp, (double)(1ull << (32 + __clz(a.n)))};
  Kept kept{0, 0};
  if (k > 0 && k < a.n) {
    u64 above;
    kept = select<false>(row, m, kept, weigh, [&](u64 s) { return s >= (u64)k; }, above);
    kept.ties = k - (int)above;
  }
  if (p < 1.f) {
    u64 total = 0;
    row.each([&](float x, int) {
      if (key_of(x) > kept.key) total += weigh(x);
    });
    total = wave_sum64(total);
    if (lane == 0) m.part[wave] = total;
    __syncthreads();
    total = (u64)kept.ties * weigh(value_of(kept.key));
    for (int w = 0; w < NW; ++w) total += m.part[w];
    __syncthreads();
    const double limit = (double)p * (double)total;
    u64 above;
    // (of p <= 0 the first token stays)
    const Kept next = select<true>(row, m, kept, weigh, [&](u64 s) { return s > 0 && !((double)s < limit); }, above);
    const double w = (double)weigh(value_of(next.key));
    const double fit = ceil((limit - (double)above) / w);
    const int ties = fit < 1 ? 1 : fit > (double)a.n ? a.n : (int)fit;
    kept.ties = next.key == kept.key ? min(kept.ties, ties) : ties;
    kept.key = next.key;
  }
  // in index order: each wave's ties, then its sum of kept weights
  int equal = 0;
  row.each([&](float x, int) { equal += kept.ties > 0 && key_of(x) == kept.key; });
  equal = (int)wave_sum64(equal);
  if (lane == 0) m.part[wave] = equal;
  __syncthreads();
  int seen = 0;  // ties before the wave's run
  for (int w = 0; w < wave; ++w) seen += (int)m.part[w];
  __syncthreads();
  const double floor_w = fminf(o.min_p, 1.f);
  // of a draw of 0, which takes the first token of any weight, all of them have one here
  auto weight = [&](float x, bool tie_kept, bool any) -> u64 {
    const uint32_t key = key_of(x);
    if (!(key > kept.key || (tie_kept && key == kept.key))) return 0;
    const double w = weigh.real(x);
    return !(w >= floor_w) ? 0 : any ? w > 0 : (u64)(w * weigh.one + 0.5);
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
  u64 mine = 0;
  walk(false, [&](const u64(&w)[4], int) {
    mine += w[0] + w[1] + w[2] + w[3];
    return false;
  });
  mine = wave_sum64(mine);
  if (lane == 0) m.part[wave] = mine;
  __syncthreads();
  u64 total = 0, base = 0;
  for (int w = 0; w < NW; ++w) {
    if (w == wave) base = total;
    total += m.part[w];
  }
  const u64 all_of_it = total;
  if (r == 0.f) {
    mine = 0;
    walk(true, [&](const u64(&w)[4], int) {
      mine += w[0] + w[1] + w[2] + w[3];
      return false;
    });
    mine = wave_sum64(mine);
    __syncthreads();
    if (lane == 0) m.part[wave] = mine;
    __syncthreads();
    total = base = 0;
    for (int w = 0; w < NW; ++w) {
      if (w == wave) base = total;
      total += m.part[w];
    }
  }
  const double limit = (double)r * (double)total;
  if ((double)base > limit || !((double)(base + mine) > limit)) return;  // another wave's
  u64 sum = base;
  walk(r == 0.f, [&](const u64(&w)[4], int i0) {
    const u64 all = w[0] + w[1] + w[2] + w[3], upto = sum + wave_scan64(all);
    const u64 here = __ballot((double)upto > limit);
    if (here == 0) {
      sum = __shfl(upto, 63);
      return false;
    }
    if (lane == __ffsll(here) - 1) {
      u64 s = upto - all;
      int c = 0;
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (c == j && !((double)(s += w[j]) > limit)) c = j + 1;
      a.index[b] = (uint32_t)(i0 + c);
      if (a.prob) a.prob[b] = (float)(weigh.real(row.x[i0 + c]) / ((double)all_of_it / weigh.one));
    }
    return true;
  });
}

}  // namespace

void check_sample_params(const SampleParams& p) {
  if (!std::isfinite(p.temperature) || p.temperature < 0.0f)
    fail(ST_SAMPLING, "temperature must not be negative, got " + std::to_string(p.temperature));
  if (!(p.r >= 0.0f && p.r < 1.0f)) fail(ST_OP, "sample: the uniform draw must be in [0, 1)");
  if (std::isnan(p.top_p) || std::isnan(p.min_p)) fail(ST_OP, "sample: a filter is NaN");
}

size_t sample_workspace(size_t rows, size_t n) { return 0; }

void launch_sample(const SampleArgs& a, int rows, void* ws, hipStream_t st) {
  hipLaunchKernelGGL(sample_kernel, dim3((unsigned)rows), dim3(ST), 0, st, a);
}

}  // namespace iek
