// Attention of one or several new tokens per sequence over the paged KV cache (paged.h), the entries that the
// batch shares read once for all.
//
// Column (b * n_q + t) * G + g of a KV head is query token t of sequence b, query head g of its group of G. It
// sees the entries [lo, hi): hi = len[b] - (n_q - 1 - t), lo = hi - window with a window, else 0. The entries
// [0, shared) are the same ones for every sequence and are found by one list of pages; so there are two kinds of
// job: all columns over a chunk of the shared entries, and a sequence's columns over a chunk of its own. With
// scores s in base 2, out = (sum 2^(s - m) v) / (sum 2^(s - m)); a job leaves (m, sum, o), a second launch joins.
//
// Both products run on the matrix cores with 16 columns a product:
//   S^T[slot][column] = K q: K's rows as they lie, a lane 16 bytes of one;
//   O^T[dim][column] += V^T P: P comes out of the first product in the layout that the second one takes.
// f32 pages: mfma_f32_16x16x4_f32, a tile of 16 slots, operands straight from the loads (V's four dims of a lane
// go to four products). fp16 pages: mfma_f32_16x16x32_f16, a tile of 32 slots; K and V are exact, q and P are fp16
// (hi, lo) pairs of 22 bits, two products each; V's rows are transposed in registers, 2 x 2 values at a time.
// q is scaled by a power of two into fp16's range, P to at most 2^15.
#include <type_traits>

#include "common.cuh"
#include "paged.h"

namespace iek {

namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr int MAX_SPLIT = 256;
constexpr int SHARED_BATCH = 64;
constexpr int TURN = 256;        // workgroups: one a CU
constexpr int JOIN_WAVES = 512;  // columns from which the join gives each to one wave

// The running maximum is only a reference: it moves when a tile's is more than 2^LAG above it. For fp16 pages P is held
// at 2^UP times its share, at most 2^15, so that what fp16 cuts off at its lower end, 2^-25, is 2^-38 of the largest.
template <bool F16>
constexpr float LAG = F16 ? 2.f : 8.f;
template <bool F16>
constexpr float UP = F16 ? 8192.f : 1.f;

// A wave takes DIMS of a row; of wider rows two or four waves take 128 each of one tile and exchange their parts
// of the scores through LDS.
constexpr int dims_of(int hd) { return hd < 128 ? hd : 128; }
constexpr int sets_of(int hd) { return WAVES * dims_of(hd) / hd; }  // sets of waves that have a row between them
template <bool F16>
constexpr int tile_of() { return F16 ? 32 : 16; }

struct Plan {
  int group, cols;           // query heads of a KV head, columns of a sequence
  int all;                   // columns of the batch
  bool own_wide, pre_wide;   // the sets of waves split the columns, not the tiles
  int own_blocks, pre_blocks;  // workgroups that the columns of a job are spread over
  int share;                 // own chunks of a KV head to aim at; 0: sequences are cut by `tiles`
  int tiles, nsplit;         // share 0: tiles a chunk, chunks a sequence at most; else the smallest chunk
  int chunks;                // own chunks of a KV head at most
  int pre_chunks;            // chunks of the shared entries at most (0: nothing is shared)
  int pre_tiles;             // the smallest of them
  bool direct;               // nothing is shared and every sequence is one chunk
  float *ml, *o;             // own: [chunks][n_kv][cols] pairs (m, sum), [chunks][n_kv][cols][hd]
  float *pml, *po;           // shared: [pre_chunks][n_kv][all] pairs, [pre_chunks][n_kv][all][hd]
};

// Constant while the kernel runs: read through the scalar cache.
IEK_DEV int scalar(const int* p, size_t i) {
  return ((const __attribute__((address_space(4))) int*)p)[i];
}
IEK_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
IEK_DEV int col_hi(const PagedAttn& a, int n, int t) { return n - (a.n_q - 1 - t); }
IEK_DEV int col_lo(const PagedAttn& a, int hi) { return a.window > 0 ? max(0, hi - a.window) : 0; }
IEK_DEV int bounded(int n, int most) { return max(0, min(n, most)); }
IEK_DEV int shared_entries(const PagedAttn& a) { return a.max_shared > 0 ? bounded(uniform(scalar(a.shared, 0)), a.max_shared) : 0; }
// The tiles [t0, t1) of a sequence's own entries that any of its columns sees.
template <int TILE>
IEK_DEV void own_range(const PagedAttn& a, int n, int shared, int& t0, int& t1) {
  t0 = max(shared, col_lo(a, max(0, col_hi(a, n, 0)))) / TILE;
  t1 = n > shared ? max(t0, (n + TILE - 1) / TILE) : t0;
}
// (tiles of a sequence: below 2^23, so that the product with the reciprocal is off by less than one)
IEK_DEV int ceil_div(int a, int b) {
  const int up = a + b - 1, q = (int)((float)up * __builtin_amdgcn_rcpf((float)b)), r = up - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}
IEK_DEV int scan(int v) {
  auto up = [](auto ctrl, auto rows, int x) {
    return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  using std::integral_constant;
  v += up(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{}, v);  // row_shr 1, 2, 4, 8
  v += up(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{}, v);
  v += up(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{}, v);
  v += up(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{}, v);
  v += up(integral_constant<int, DPP_BCAST15>{}, integral_constant<int, 0xA>{}, v);
  return v + up(integral_constant<int, DPP_BCAST31>{}, integral_constant<int, 0xC>{}, v);
}

// Own chunk x of a KV head (FIND), or the chunks of sequence b: its length, tiles a chunk, number of chunks
// (0 with FIND: there is no chunk x) and first chunk. Up to SHARED_BATCH sequences the chunk's size is found from
// the lengths themselves: their total by the chunks that fill the chip, each sequence evenly into as many as that
// takes. Larger batches are cut by max_len.
struct Cut {
  int b, n, tiles, count, first;
};
template <bool FIND, int TILE, int STEP>
IEK_DEV Cut cut(const Paged& c, const PagedAttn& a, const Plan& p, int shared, int x, int b) {
  Cut r{b, 0, p.tiles, 0, 0};
  int t0, t1;
  const int least = p.direct ? 1 : 0;  // (a sequence without entries: its zeros are written)
  if (p.share == 0 || c.batch == 1) {
    if (FIND) r.b = c.batch == 1 ? 0 : min(x / p.nsplit, c.batch - 1);
    r.n = uniform(bounded(scalar(a.len, r.b), a.max_len));
    own_range<TILE>(a, r.n, shared, t0, t1);
    if (p.share != 0) r.tiles = max(p.tiles, ceil_div(ceil_div(t1 - t0, min(p.share, MAX_SPLIT)), STEP) * STEP);
    r.tiles = uniform(r.tiles);
    r.count = max(least, uniform(ceil_div(t1 - t0, r.tiles)));
    r.first = r.b * p.nsplit;
    if (FIND && x - r.first >= r.count) r.count = 0;
    return r;
  }
  const int lane = threadIdx.x & 63;
  const int n = lane < c.batch ? bounded(a.len[lane], a.max_len) : 0;
  own_range<TILE>(a, n, shared, t0, t1);
  const int each = lane < c.batch ? t1 - t0 : 0;
  const int total = __builtin_amdgcn_readlane(scan(each), 63);
  const int most = (int)wave_max((float)each);
  const int aim = max(p.share - c.batch / 2, (p.share + 1) / 2);
  const int size = max(p.tiles, ceil_div(max((int)(((unsigned)total + aim - 1) / (unsigned)aim), ceil_div(most, MAX_SPLIT)), STEP) * STEP);
  const int even = max(p.tiles, ceil_div(ceil_div(each, max(1, ceil_div(each, size))), STEP) * STEP);
  const int mine = lane < c.batch ? max(least, ceil_div(each, even)) : 0, upto = scan(mine);
  if (FIND) {
    const unsigned long long here = __ballot(upto > x && upto - mine <= x);
    if (here == 0) return r;
    r.b = __ffsll(here) - 1;
  }
  r.n = __builtin_amdgcn_readlane(n, r.b);
  r.tiles = __builtin_amdgcn_readlane(even, r.b);
  r.count = __builtin_amdgcn_readlane(mine, r.b);
  r.first = __builtin_amdgcn_readlane(upto, r.b) - r.count;
  return r;
}

// The shared entries' tiles [t0, t1) that any column sees, cut into `count` chunks of `tiles`.
struct PreCut {
  int t0, t1, tiles, count;
};
template <int TILE>
IEK_DEV PreCut pre_cut(const Paged& c, const PagedAttn& a, const Plan& p, int shared) {
  PreCut r{0, (shared + TILE - 1) / TILE, 1, 0};
  if (a.window > 0) {  // from the shortest sequence's window on
    int least = INT32_MAX;
    for (int b = threadIdx.x & 63; b < c.batch; b += 64) {
      const int n = bounded(a.len[b], a.max_len);
      if (n > 0) least = min(least, col_lo(a, max(0, col_hi(a, n, 0))));
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) least = min(least, __shfl_xor(least, s));
    r.t0 = min(uniform(least) / TILE, r.t1);
  }
  r.tiles = max(p.pre_tiles, uniform(ceil_div(r.t1 - r.t0, max(1, p.pre_chunks))));
  r.count = uniform(ceil_div(r.t1 - r.t0, r.tiles));
  return r;
}

// v over the wave's four groups of 16 lanes
IEK_DEV float groups_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
IEK_DEV float groups_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

IEK_DEV f4_t mfma(u4_t a, u4_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
}
IEK_DEV f4_t mfma(float a, float b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Where 16 slots lie: the pages of a job, and the numbers of a tile's.
struct Pages {
  const int* list;
  int end;  // entries
};
template <bool F16>
struct Ids {
  int id[F16 ? 2 : 1];
};
template <bool F16>
IEK_DEV Ids<F16> ids_of(const Paged& c, const Pages& g, int tile) {
  Ids<F16> r;
#pragma unroll
  for (int x = 0; x < (F16 ? 2 : 1); ++x) {
    const int j = tile * tile_of<F16>() + 16 * x;
    r.id[x] = uniform(j < g.end ? scalar(g.list, j >> c.shift) : -1);
    if ((unsigned)r.id[x] >= (unsigned)c.n_pages) r.id[x] = -1;
  }
  return r;
}

// Buffer accesses end at the last live row of the 16, and at none where there is no page: the rows behind it read
// as zeros, whatever they hold (a NaN would reach O through a weight of 0).
template <int HD, bool F16>
IEK_DEV __amdgpu_buffer_rsrc_t rows_rsrc(const Paged& c, const void* pool, int h, int id, int j, int end) {
  const size_t row = (((size_t)max(id, 0) * c.n_kv + h) << c.shift) + (j & ((1 << c.shift) - 1));
  const int live = uniform(id < 0 ? 0 : max(0, min(16, end - j)));  // (a median of three is a vector instruction)
  const char* base = static_cast<const char*>(pool) + row * (HD * (F16 ? 2 : 4));
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, live * HD * (F16 ? 2 : 4), 0x00020000);
}

// A wave's part of a tile: lane (r = lane & 15, kg = lane >> 4). sum: o[x]'s V^T, of 1 in place of every infinity of the sign
// and NaN and 0 for the rest, times weights (for the rare tiles with a V that is not finite).
template <int DIMS, bool HALVES>
struct Tile;
template <int DIMS>
struct Tile<DIMS, false> {
  f4_t k[DIMS / 16];     // K[r][16 i + 4 kg + e]
  f4_t v[4][DIMS / 64];  // V[4 kg + i][64 u + 4 r + e]
  template <bool>
  IEK_DEV bool not_finite() const {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4 * (DIMS / 64) * 4; ++i) top = max(top, __float_as_uint(v[i & 3][i >> 4][i >> 2 & 3]) & 0x7FFFFFFFu);
    return top >= 0x7F800000u;
  }
  template <bool>
  IEK_DEV void drop() {
#pragma unroll
    for (int i = 0; i < 4 * (DIMS / 64) * 4; ++i) {
      float x = v[i & 3][i >> 4][i >> 2 & 3];
      asm volatile("" : "+v"(x));
      v[i & 3][i >> 4][i >> 2 & 3] = (__float_as_uint(x) & 0x7FFFFFFFu) >= 0x7F800000u ? 0.f : x;
    }
  }
  template <bool>
  IEK_DEV f4_t sum(int x, const float (&w)[4], bool minus) const {
    f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y = v[i][x >> 2][x & 3];
      asm volatile("" : "+v"(y));  // (nothing of this is to be kept for another column, in registers of the common path)
      o = mfma(y == (minus ? -INFINITY : INFINITY) || y != y ? 1.f : 0.f, w[i], o);
    }
    return o;
  }
};
// (fp16, or with F16 false bf16)
template <int DIMS>
struct Tile<DIMS, true> {
  static constexpr int VW = DIMS / 32;
  u4_t k[2][VW];         // K[16 s + r][32 i + 8 kg + (0 .. 7)]
  uint32_t v[8][VW];     // V[16 (j >> 2) + 4 kg + (j & 3)][DIMS / 16 * r + ...]
  template <bool F16>
  static constexpr uint32_t INF = F16 ? 0x7C00u : 0x7F80u;
  template <bool F16>
  IEK_DEV bool not_finite() const {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 8 * VW; ++i) {
      lo = max(lo, v[i & 7][i >> 3] & 0x7FFFu);
      hi = max(hi, v[i & 7][i >> 3] & 0x7FFF0000u);
    }
    return lo >= INF<F16> || hi >= INF<F16> << 16;
  }
  template <bool F16>
  IEK_DEV void drop() {
#pragma unroll
    for (int i = 0; i < 8 * VW; ++i) {
      uint32_t x = v[i & 7][i >> 3];
      asm volatile("" : "+v"(x));
      x = (x & 0x7FFFu) >= INF<F16> ? x & 0xFFFF0000u : x;
      x = (x & 0x7FFF0000u) >= INF<F16> << 16 ? x & 0x0000FFFFu : x;
      v[i & 7][i >> 3] = x;
    }
  }
  // V^T's operand for the dims 2 w + e
  IEK_DEV u4_t operand(int w, int e) const {
    u4_t r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], e ? 0x07060302u : 0x05040100u);
    return r;
  }
  template <bool F16>
  IEK_DEV f4_t sum(int x, const float (&w)[8], bool minus) const {
    u4_t y = operand(x >> 1, x & 1), z;
    asm volatile("" : "+v"(y));  // (nothing of this is to be kept for another column, in registers of the common path)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      auto flag = [&](uint32_t half) -> uint32_t {  // 1 in fp16
        const uint32_t size = half & 0x7FFFu;
        return size > INF<F16> || (size == INF<F16> && (half >> 15 & 1) == (minus ? 1u : 0u)) ? 0x3C00u : 0u;
      };
      const uint32_t both = y[j];  // (bit_cast of an element of a vector takes the vector's first)
      y[j] = flag(both) | flag(both >> 16) << 16;
      z[j] = __builtin_bit_cast(uint32_t, h2_t{(_Float16)w[2 * j], (_Float16)w[2 * j + 1]});
    }
    return mfma(y, z, f4_t{0.f, 0.f, 0.f, 0.f});
  }
};

template <int HD, int DIMS, bool F16>
IEK_DEV void load_k(Tile<DIMS, F16>& T, const Paged& c, int h, const Ids<F16>& id, int tile, int end, int dim0, int lane) {
  if constexpr (F16) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const auto rs = rows_rsrc<HD, true>(c, c.k, h, id.id[s], 32 * tile + 16 * s, end);
#pragma unroll
      for (int i = 0; i < DIMS / 32; ++i)
        T.k[s][i] = __builtin_amdgcn_raw_buffer_load_b128(rs, 2 * ((lane & 15) * HD + 8 * (lane >> 4)), 2 * (dim0 + 32 * i), 0);
    }
  } else {
    const auto rs = rows_rsrc<HD, false>(c, c.k, h, id.id[0], 16 * tile, end);
#pragma unroll
    for (int i = 0; i < DIMS / 16; ++i)
      T.k[i] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, 4 * ((lane & 15) * HD + 4 * (lane >> 4)),
                                                                              4 * (dim0 + 16 * i), 0));
  }
}

template <int HD, int DIMS, bool F16>
IEK_DEV void load_v(Tile<DIMS, F16>& T, const Paged& c, int h, const Ids<F16>& id, int tile, int end, int dim0, int lane) {
  if constexpr (F16) {
    const int off = 2 * (4 * (lane >> 4) * HD + DIMS / 16 * (lane & 15));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const auto rs = rows_rsrc<HD, true>(c, c.v, h, id.id[s], 32 * tile + 16 * s, end);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DIMS == 64) {
          const auto x = __builtin_amdgcn_raw_buffer_load_b64(rs, off, 2 * (dim0 + j * HD), 0);
          T.v[4 * s + j][0] = x[0];
          T.v[4 * s + j][1] = x[1];
        } else {
          const auto x = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 2 * (dim0 + j * HD), 0);
#pragma unroll
          for (int w = 0; w < 4; ++w) T.v[4 * s + j][w] = x[w];
        }
      }
    }
  } else {
    const int off = 4 * (4 * (lane >> 4) * HD + 4 * (lane & 15));
    const auto rs = rows_rsrc<HD, false>(c, c.v, h, id.id[0], 16 * tile, end);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int u = 0; u < DIMS / 64; ++u)
        T.v[i][u] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 4 * (dim0 + i * HD + 64 * u), 0));
  }
}

// The dim (of the wave's) that element r of o[x] of lane group kg is.
template <int DIMS, bool F16>
IEK_DEV int dim_at(int x, int kg, int r) {
  return F16 ? DIMS / 16 * (4 * kg + r) + x : 64 * (x >> 2) + 4 * (4 * kg + r) + (x & 3);
}

template <int DIMS, bool F16, int CG>
struct Query;
template <int DIMS, int CG>
struct Query<DIMS, false, CG> {
  f4_t q[CG][DIMS / 16];
};
template <int DIMS, int CG>
struct Query<DIMS, true, CG> {
  u4_t hi[CG][DIMS / 32], lo[CG][DIMS / 32];
};

// A column's scores of a tile, base 2, to shares of its running maximum m; l their sum, o what is scaled along.
template <bool F16, int NX, int ND>
IEK_DEV void weigh_tile(float (&s)[NX], float& m, float& l, f4_t (&o)[ND]) {
  float top = s[0];
#pragma unroll
  for (int i = 1; i < NX; ++i) top = fmaxf(top, s[i]);
  top = groups_max(top);
  if (__any(top > m + LAG<F16> || (m == -INFINITY && top > m))) {
    const bool up = top > m + LAG<F16> || m == -INFINITY;
    const float corr = up && m != -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 1.f;  // (all is 0 before)
    if (up) m = top;
    l *= corr;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] *= corr;
  }
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
    l += s[i];
  }
}

// What a job's columns and entries are.
struct Job {
  int h;
  int col0, cols;  // the batch's columns [col0, col0 + cols)
  int block;       // of the workgroups that these are spread over
  Pages pages;
  int begin;       // entries [begin, pages.end)
  int t0, t1;      // this chunk's tiles
  float *ml, *o;   // the partial results of column col0, or, if null, the output is written
};

template <int HD, bool F16>
struct Shared {
  static constexpr int SETS = sets_of(HD), DW = WAVES / SETS;
  f4_t parts[DW > 1 ? 2 : 1][DW > 1 ? WAVES : 1][2][F16 ? 2 : 1][64];
  float m[SETS][16], l[SETS][16];
  float o[SETS][16][HD + 4 * DW];
};

// Four dims of column cc of the job, or of the output.
template <int HD>
IEK_DEV void put_dims(const PagedAttn& a, const Plan& p, const Job& J, int cc, int dim, f4_t y, float sum) {
  if (J.o) {
    *reinterpret_cast<f4_t*>(J.o + (size_t)cc * HD + dim) = y;
  } else {
    const int col = J.col0 + cc, b = col / p.cols, t = (col - b * p.cols) / p.group, g = col - b * p.cols - t * p.group;
    float* out = a.out + (((size_t)b * a.n_q + t) * a.n_heads + J.h * p.group + g) * HD + dim;
    *reinterpret_cast<f4_t*>(out) = sum == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : y / sum;
  }
}
IEK_DEV void put_sums(const Job& J, int cc, float m, float l) {
  if (!J.ml) return;
  J.ml[2 * cc] = isnan(l) ? l : m;  // (a NaN: the maxima pass it over)
  J.ml[2 * cc + 1] = l;
}
// A wave's 16 columns from cc0 on, DIMS of them from dim0 on: turned through LDS of its own (`room`), since a lane holds
// pieces of 16 or 32 bytes of a column. (64 sequences over 16384 shared fp16 entries: 77 us, written as they are held 86.)
constexpr int turn_row(int dims) { return dims + 4; }
template <int HD, int DIMS, bool HALVES, int ND>
IEK_DEV void put_columns(const PagedAttn& a, const Plan& p, const Job& J, float* room, int cc0, int dim0, float m, float l, const f4_t (&o)[ND], float scale) {
  constexpr int ROW = turn_row(DIMS), PER = DIMS / 4;
  const int lane = threadIdx.x & 63, kg = lane >> 4, cl = lane & 15;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < ND; i += 4)
      *reinterpret_cast<f4_t*>(room + cl * ROW + dim_at<DIMS, HALVES>(i, kg, r)) = f4_t{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]} * scale;
  if (kg == 0) room[cl * ROW + DIMS] = l;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int i = 0; i < 16 * PER / 64; ++i) {
    const int at = 64 * i + lane, col = at / PER, dim = 4 * (at % PER);
    if (cc0 + col < J.cols) put_dims<HD>(a, p, J, cc0 + col, dim0 + dim, *reinterpret_cast<const f4_t*>(room + col * ROW + dim), room[col * ROW + DIMS]);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (dim0 == 0 && kg == 0 && cc0 + cl < J.cols) put_sums(J, cc0 + cl, m, l);
}

template <int HD, bool F16, bool WIDE, int CG>
IEK_DEV void run_job(const Paged& c, const PagedAttn& a, const Plan& p, const Job& J, Shared<HD, F16>& L) {
  constexpr int DIMS = dims_of(HD), SETS = sets_of(HD), DW = WAVES / SETS, TILE = tile_of<F16>();
  constexpr int STEP = WIDE ? 1 : SETS, NH = F16 ? 2 : 1, NX = 4 * NH, ND = DIMS / 16;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int kg = lane >> 4, cl = lane & 15;
  const int set = wave / DW, dim0 = (wave % DW) * DIMS;
  const int col_base = WIDE ? (J.block * SETS + set) * CG * 16 : J.block * CG * 16;
  const float ks = a.scale * 1.44269504088896340736f;
  const int G = p.group;
  int tile = uniform(J.t0 + (WIDE ? 0 : set));
  // Loads are issued without conditions, those past the chunk's last entry of nothing. (The compiler moves the first ones behind
  // q's conversion, V before K for fp16, so its wait at the loop's head, for both ways into it, is one for all loads in
  // flight: a tile's K products wait for its V too.)
  const Pages pages{J.pages.list, min(J.pages.end, J.t1 * TILE)};
  Ids<F16> id = ids_of<F16>(c, pages, tile), next = ids_of<F16>(c, pages, tile + STEP);
  Tile<DIMS, F16> T;
  // this lane's columns
  int hi[CG], lo[CG];
  float qs[CG];
  Query<DIMS, F16, CG> Q;
  const float* rows[CG];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    const int col = J.col0 + min(col_base + 16 * u + cl, J.cols - 1);
    const int b = col / p.cols, t = (col - b * p.cols) / G, g = col - b * p.cols - t * G;
    hi[u] = col_hi(a, bounded(a.len[b], a.max_len), t);
    lo[u] = max(col_lo(a, hi[u]), J.begin);
    hi[u] = min(hi[u], J.pages.end);
    rows[u] = a.q + ((size_t)b * a.n_q + t) * a.q_stride + (size_t)(J.h * G + g) * HD + dim0;
  }
  f4_t raw[F16 ? CG : 1][F16 ? DIMS / 16 : 1];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    if constexpr (F16) {
#pragma unroll
      for (int i = 0; i < DIMS / 32; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) raw[u][2 * i + e] = *reinterpret_cast<const f4_t*>(rows[u] + 32 * i + 8 * kg + 4 * e);
    } else {
#pragma unroll
      for (int i = 0; i < DIMS / 16; ++i) Q.q[u][i] = *reinterpret_cast<const f4_t*>(rows[u] + 16 * i + 4 * kg);
    }
  }
  load_k<HD>(T, c, J.h, id, tile, pages.end, dim0, lane);
  load_v<HD>(T, c, J.h, id, tile, pages.end, dim0, lane);
  int lo_max = 0, hi_min = INT32_MAX;
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    qs[u] = ks;
    if constexpr (F16) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < DIMS / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(raw[u][i][e]));
      top = groups_max(top);
      // into [2^13, 2^14) by a power of two (an infinity or NaN, or a row of zeros, stays what it is)
      int ex = (int)(__float_as_uint(top) >> 23) - 127;
      ex = ex == 128 ? 0 : min(13 - ex, 126);
      const float up = __builtin_amdgcn_ldexpf(1.f, ex);
      qs[u] = __builtin_amdgcn_ldexpf(ks, -ex);
#pragma unroll
      for (int i = 0; i < DIMS / 32; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f4_t v = raw[u][2 * i + (e >> 1)];
          const float y0 = v[2 * (e & 1)] * up, y1 = v[2 * (e & 1) + 1] * up;
          const h2_t w = {(_Float16)y0, (_Float16)y1};
          const h2_t z = {(_Float16)(y0 - (float)w[0]), (_Float16)(y1 - (float)w[1])};
          Q.hi[u][i][e] = __builtin_bit_cast(uint32_t, w);
          Q.lo[u][i][e] = __builtin_bit_cast(uint32_t, z);
        }
    }
    lo_max = max(lo_max, lo[u]);
    hi_min = min(hi_min, hi[u]);
  }
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) {
    lo_max = max(lo_max, __shfl_xor(lo_max, s));
    hi_min = min(hi_min, __shfl_xor(hi_min, s));
  }
  lo_max = uniform(lo_max);
  hi_min = uniform(hi_min);
  float m[CG], l[CG];
  f4_t o[CG][ND];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[u][i] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  const int span = J.t1 - J.t0;
  const int t_end = DW > 1 ? J.t0 + (span + STEP - 1) / STEP * STEP : J.t1;  // (all waves go through the barriers, some with no tile)
  for (int turn = 0; tile < t_end; tile = uniform(tile + STEP), turn ^= 1) {
    float s[CG][NX];
    const Ids<F16> after = ids_of<F16>(c, pages, tile + 2 * STEP);
    {
      f4_t d[CG][NH];
#pragma unroll
      for (int u = 0; u < CG; ++u)
#pragma unroll
        for (int x = 0; x < NH; ++x) d[u][x] = f4_t{0.f, 0.f, 0.f, 0.f};
      if constexpr (F16) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int i = 0; i < DIMS / 32; ++i)
#pragma unroll
            for (int u = 0; u < CG; ++u) {
              d[u][x] = mfma(T.k[x][i], Q.hi[u][i], d[u][x]);
              d[u][x] = mfma(T.k[x][i], Q.lo[u][i], d[u][x]);
            }
      } else {
        // (several sums of a quarter or half of the dims: one of all of them rounds up to 128 times in a row)
        constexpr int N = 4 / CG;
        f4_t z[CG][N];
#pragma unroll
        for (int u = 0; u < CG; ++u)
#pragma unroll
          for (int x = 0; x < N; ++x) z[u][x] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < DIMS / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int u = 0; u < CG; ++u) z[u][e % N] = mfma(T.k[i][e], Q.q[u][i][e], z[u][e % N]);
#pragma unroll
        for (int u = 0; u < CG; ++u) d[u][0] = N == 4 ? (z[u][0] + z[u][1]) + (z[u][2 % N] + z[u][3 % N]) : z[u][0] + z[u][1 % N];
      }
      load_k<HD>(T, c, J.h, next, tile + STEP, pages.end, dim0, lane);
#pragma unroll
      for (int u = 0; u < CG; ++u)
#pragma unroll
        for (int x = 0; x < NH; ++x) {
          d[u][x] *= qs[u];
          if constexpr (DW > 1) L.parts[turn][wave][u][x][lane] = d[u][x];
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][4 * x + i] = d[u][x][i];
        }
    }
    if constexpr (DW > 1) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < CG; ++u)
#pragma unroll
        for (int x = 0; x < NH; ++x) {
          f4_t y = L.parts[turn][set * DW][u][x][lane];
#pragma unroll
          for (int w = 1; w < DW; ++w) y += L.parts[turn][set * DW + w][u][x][lane];  // (the same order in every wave)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][4 * x + i] = y[i];
        }
    }
    const bool inner = tile * TILE >= lo_max && (tile + 1) * TILE <= hi_min && id.id[0] >= 0 && id.id[NH - 1] >= 0;
#pragma unroll
    for (int u = 0; u < CG; ++u) {
      if (!inner) {
#pragma unroll
        for (int i = 0; i < NX; ++i) {
          const int j = tile * TILE + 16 * (i >> 2) + 4 * kg + (i & 3);
          if (j < lo[u] || j >= hi[u] || id.id[i >> 2] < 0) s[u][i] = -INFINITY;
        }
      }
      weigh_tile<F16>(s[u], m[u], l[u], o[u]);
    }
    if (!inner && __any(T.template not_finite<F16>())) {
      // V that is not finite, in entries that some columns may not see: taken out of the product (where a weight of 0
      // would make NaN of it), and given as infinities of the same sign (both for NaN) to the columns that do see it
#pragma unroll
      for (int u = 0; u < CG; ++u) {
        float sees[NX];
#pragma unroll
        for (int i = 0; i < NX; ++i) {
          const int j = tile * TILE + 16 * (i >> 2) + 4 * kg + (i & 3);
          sees[i] = j < lo[u] || j >= hi[u] || id.id[i >> 2] < 0 ? 0.f : 1.f;
        }
#pragma unroll
        for (int x = 0; x < ND; ++x) {
          const f4_t up = T.template sum<F16>(x, sees, false), down = T.template sum<F16>(x, sees, true);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[u][x][r] += (up[r] > 0.f ? INFINITY : 0.f) + (down[r] > 0.f ? -INFINITY : 0.f);
        }
      }
      T.template drop<F16>();
    }
    if constexpr (F16) {
      u4_t ph[CG], pl[CG];
#pragma unroll
      for (int u = 0; u < CG; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y0 = s[u][2 * i] * UP<F16>, y1 = s[u][2 * i + 1] * UP<F16>;
          const h2_t w = {(_Float16)y0, (_Float16)y1};
          const h2_t z = {(_Float16)(y0 - (float)w[0]), (_Float16)(y1 - (float)w[1])};
          ph[u][i] = __builtin_bit_cast(uint32_t, w);
          pl[u][i] = __builtin_bit_cast(uint32_t, z);
        }
#pragma unroll
      for (int w = 0; w < DIMS / 32; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u4_t v = T.operand(w, e);
#pragma unroll
          for (int u = 0; u < CG; ++u) {
            o[u][2 * w + e] = mfma(v, ph[u], o[u][2 * w + e]);
            o[u][2 * w + e] = mfma(v, pl[u], o[u][2 * w + e]);
          }
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < ND; ++x)
#pragma unroll
          for (int u = 0; u < CG; ++u) o[u][x] = mfma(T.v[i][x >> 2][x & 3], s[u][i], o[u][x]);
    }
    load_v<HD>(T, c, J.h, next, tile + STEP, pages.end, dim0, lane);
    id = next;
    next = after;
  }

  constexpr float DOWN = 1.f / UP<F16>;
  if constexpr (WIDE) {
#pragma unroll
    for (int u = 0; u < CG; ++u) {
      l[u] = groups_sum(l[u]);
      put_columns<HD, DIMS, F16>(a, p, J, &L.o[0][0][0] + wave * 16 * turn_row(DIMS), col_base + 16 * u, dim0, m[u], l[u], o[u], DOWN);
    }
  } else {
    // the sets' parts: to a common maximum, then summed through LDS
#pragma unroll
    for (int u = 0; u < CG; ++u) {
      if (u > 0) __syncthreads();
      l[u] = groups_sum(l[u]);
      if (kg == 0 && dim0 == 0) {
        L.m[set][cl] = m[u];
        L.l[set][cl] = l[u];
      }
      __syncthreads();
      float top = L.m[0][cl];
#pragma unroll
      for (int w = 1; w < SETS; ++w) top = fmaxf(top, L.m[w][cl]);
      const float mine = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - top) * DOWN;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < ND; i += 4)
          *reinterpret_cast<f4_t*>(&L.o[set][cl][dim0 + dim_at<DIMS, F16>(i, kg, r)]) =
              f4_t{o[u][i][r], o[u][i + 1][r], o[u][i + 2][r], o[u][i + 3][r]} * mine;
      __syncthreads();
      for (int i = threadIdx.x; i < 16 * HD / 4; i += 64 * WAVES) {
        const int col = i / (HD / 4), dim = 4 * (i % (HD / 4)), cc = col_base + 16 * u + col;
        if (cc >= J.cols) continue;
        f4_t y = *reinterpret_cast<const f4_t*>(&L.o[0][col][dim]);
#pragma unroll
        for (int w = 1; w < SETS; ++w) y += *reinterpret_cast<const f4_t*>(&L.o[w][col][dim]);
        float mm = L.m[0][col], ll = 0.f;
#pragma unroll
        for (int w = 1; w < SETS; ++w) mm = fmaxf(mm, L.m[w][col]);
#pragma unroll
        for (int w = 0; w < SETS; ++w)
          ll += L.l[w][col] * (L.m[w][col] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(L.m[w][col] - mm));
        put_dims<HD>(a, p, J, cc, dim, y, ll);
        if (dim == 0) put_sums(J, cc, mm, ll);
      }
    }
  }
}

// ---- many columns: tiles in LDS -----------------------------------------------------------------------
// For rows of up to 128 the four waves split the columns of a job and share its tiles of 32 slots, which lie in LDS. Both
// products are mfma_f32_16x16x32 ones. fp16 pages: a ring of four tiles, filled by copies without registers three tiles
// ahead (of head_dim 128 one tile's time ahead: the 13 or 26 registers that spill are read back in the block for values that are not
// finite, and for these the compiler waits at every tile for all that is in flight, the copies just issued among them);
// 32 columns a wave, K and V one plane, q and P pairs (as above). f32 pages: one tile, each thread 16-byte pieces of
// rows, the next tile's in flight in registers meanwhile; 16 columns a wave, every operand as three bf16 numbers that sum
// to it exactly (8 bits each, the first one cut off, the others rounded), six products: of the parts' orders those up to the
// third; what is left out is below 2^-22 of a product. (mfma_f32_16x16x4_f32, exact, takes 32 cycles for 4 of the 32 terms.)
// 32 heads of 128, part launch: 16384 shared fp16 entries, 64 sequences 65 us (with each wave's tiles in its registers 113),
// 4096 f32 ones, 32 sequences 28 us (42). The matrix cores are busy for 14 and 10 us of these, a SIMD issues for half of the time: it waits for copies and for
// its two waves' softmax, and the first tile, the results and the own chunks' one turn take 15 to 20.
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
IEK_DEV f4_t mfma_b(u4_t a, u4_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
// Two numbers as three pairs of bf16.
IEK_DEV void three(float x, float y, uint32_t& a, uint32_t& b, uint32_t& c) {
  const uint32_t xa = __float_as_uint(x) & 0xFFFF0000u, ya = __float_as_uint(y) & 0xFFFF0000u;
  a = __builtin_amdgcn_perm(ya, xa, 0x07060302u);
  const float xr = x - __uint_as_float(xa), yr = y - __uint_as_float(ya);
  b = __builtin_bit_cast(uint32_t, b2_t{(__bf16)xr, (__bf16)yr});
  const float xs = xr - __uint_as_float(b << 16), ys = yr - __uint_as_float(b & 0xFFFF0000u);
  c = __builtin_bit_cast(uint32_t, b2_t{(__bf16)xs, (__bf16)ys});
}

template <int HD, bool F16>
struct Staged {
  static constexpr int NP = F16 ? 1 : 3, PIECES = HD / 8;  // planes; pieces of eight numbers a row
  static constexpr int CG = F16 ? 2 : 1;                   // groups of 16 columns a wave
  static constexpr int RING = F16 ? 4 : 1;                 // tiles
  struct One {
    u4_t k[NP][32 * PIECES], v[NP][32 * PIECES];
  } ring[RING];
  // K's pieces are permuted within rows, so that 16 rows' pieces of the same dims are in different banks
  static IEK_DEV int turned(int row) { return HD == 128 ? row & 15 : row >> 1 & 7; }
  static IEK_DEV int k_at(int row, int piece) { return row * PIECES + (piece ^ turned(row)); }
};

// 16 bytes a lane from memory to 1024 in a row in LDS, without registers. (The waits for it are the caller's; the one between
// the write of m0, where LDS is written, and the copy is here: the compiler puts none into inline assembly.)
IEK_DEV void copy16(const void* lds, const char* from, uint32_t offset) {
  const uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds;
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(__builtin_amdgcn_readfirstlane(at)), "v"(offset), "s"(from) : "memory");
}
template <int N>
IEK_DEV void copies_left() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// fp16 tiles into LDS, 64 pieces a copy. Rows behind the last live one are that one again, and
// those without a page any row: such a tile is not an inner one, where values out of sight are looked at.
template <int HD>
struct Copies {
  using S = Staged<HD, true>;
  static constexpr int N = S::PIECES / 8;  // copies of K, and of V, a wave and tile
  uint32_t row, k_at, v_at;  // this lane's of 16 rows, and its pieces' places
  IEK_DEV Copies() {
    const int at = (threadIdx.x & 63) + 64 * (int)(threadIdx.x >> 6);
    row = at / S::PIECES & 15;
    k_at = 16 * (at % S::PIECES ^ S::turned(at / S::PIECES));
    v_at = 16 * (at % S::PIECES);
  }
  IEK_DEV void tile(typename S::One& to, const Paged& c, int h, const Ids<true>& id, int tile, int end) const {
    const int wave = uniform(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int piece = (i * WAVES + wave) * 64, half = N == 2 ? i : wave >> 1, j = 32 * tile + 16 * half;
      const int page = max(half ? id.id[1] : id.id[0], 0);
      const size_t first = ((((size_t)(uint32_t)page * (uint32_t)c.n_kv + h) << c.shift) + (j & ((1 << c.shift) - 1))) * (2 * HD);
      uint32_t from = row;
      if (end - j < 16) from = min(from, (uint32_t)max(0, end - j - 1));  // (uniform)
      from *= 2 * HD;
      copy16(&to.k[0][piece], static_cast<const char*>(c.k) + first, from + k_at);
      copy16(&to.v[0][piece], static_cast<const char*>(c.v) + first, from + v_at);
    }
  }
};

// A thread's pieces of an f32 tile on their way: piece t % PIECES of the rows t / PIECES, ...
template <int HD>
struct Way {
  using S = Staged<HD, false>;
  static constexpr int PIECES = HD / 8, RPP = 64 * WAVES / PIECES, NPASS = 32 / RPP;
  u4_t k[NPASS][2], v[NPASS][2];
  IEK_DEV void load(const Paged& c, int h, const Ids<true>& id, int tile, int end) {
    const int t = threadIdx.x, wave = uniform(t >> 6);
#pragma unroll
    for (int p = 0; p < NPASS; ++p) {
      // (a wave's rows of a pass are in one half of the tile)
      const int half = (p * RPP + wave * 64 / PIECES) >> 4, row = (p * RPP + t / PIECES) & 15;
      const int off = (row * HD + 8 * (t % PIECES)) * 4;
      const auto rk = rows_rsrc<HD, false>(c, c.k, h, half ? id.id[1] : id.id[0], 32 * tile + 16 * half, end);
      const auto rv = rows_rsrc<HD, false>(c, c.v, h, half ? id.id[1] : id.id[0], 32 * tile + 16 * half, end);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        k[p][n] = __builtin_amdgcn_raw_buffer_load_b128(rk, off, 16 * n, 0);
        v[p][n] = __builtin_amdgcn_raw_buffer_load_b128(rv, off, 16 * n, 0);
      }
    }
  }
  IEK_DEV void store(typename S::One& L) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int p = 0; p < NPASS; ++p) {
      const int row = p * RPP + t / PIECES, piece = t % PIECES;
      u4_t x[3], y[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t q[3];
        const u4_t kk = k[p][e >> 1], vv = v[p][e >> 1];
        three(__uint_as_float(kk[2 * (e & 1)]), __uint_as_float(kk[2 * (e & 1) + 1]), q[0], q[1], q[2]);
        x[0][e] = q[0], x[1][e] = q[1], x[2][e] = q[2];
        // (a signalling NaN made a quiet one: the first part, cut off, may be an infinity otherwise)
        three(__builtin_canonicalizef(__uint_as_float(vv[2 * (e & 1)])), __builtin_canonicalizef(__uint_as_float(vv[2 * (e & 1) + 1])), q[0], q[1],
              q[2]);
        y[0][e] = q[0], y[1][e] = q[1], y[2][e] = q[2];
      }
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        L.k[n][S::k_at(row, piece)] = x[n];
        L.v[n][row * PIECES + piece] = y[n];
      }
    }
  }
};

template <int HD, bool F16>
IEK_DEV void run_wide(const Paged& c, const PagedAttn& a, const Plan& p, const Job& J, Staged<HD, F16>& R) {
  using S = Staged<HD, F16>;
  constexpr int CG = S::CG, NP = S::NP, PIECES = S::PIECES, KS = HD / 32, ND = HD / 16, TILE = 32, DW2 = HD / 32;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kg = lane >> 4, cl = lane & 15, G = p.group;
  const int col_base = (J.block * WAVES + wave) * CG * 16;
  const bool idle = col_base >= J.cols;  // (such a wave takes part in the staging alone)
  const Pages pages{J.pages.list, min(J.pages.end, J.t1 * TILE)};
  // f32: the tile after the present one is under way to registers; fp16: up to three are to LDS
  constexpr int AHEAD = S::RING - 1, COPIES = S::PIECES / 4;  // (copies a wave and tile)
  Ids<true> id[F16 ? AHEAD + 2 : 3];
#pragma unroll
  for (int i = 0; i < (F16 ? AHEAD + 2 : 3); ++i) id[i] = ids_of<true>(c, pages, J.t0 + i);
  Way<HD> way;
  const Copies<HD> copies;
  if constexpr (F16) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (J.t0 + i < J.t1) copies.tile(R.ring[i], c, J.h, id[i], J.t0 + i, pages.end);
  } else {
    way.load(c, J.h, id[0], J.t0, pages.end);
  }
  int hi[CG], lo[CG], lo_max = 0, hi_min = INT32_MAX;
  float qs[CG], m[CG], l[CG];
  u4_t q[CG][KS][F16 ? 2 : 3];
  f4_t o[CG][ND];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    const int col = J.col0 + min(col_base + 16 * u + cl, J.cols - 1);
    const int b = col / p.cols, t = (col - b * p.cols) / G, g = col - b * p.cols - t * G;
    hi[u] = col_hi(a, bounded(a.len[b], a.max_len), t);
    lo[u] = max(col_lo(a, hi[u]), J.begin);
    hi[u] = min(hi[u], J.pages.end);
    lo_max = max(lo_max, lo[u]);
    hi_min = min(hi_min, hi[u]);
    const float* row = a.q + ((size_t)b * a.n_q + t) * a.q_stride + (size_t)(J.h * G + g) * HD + 8 * kg;
    f4_t raw[2 * KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      raw[2 * i] = *reinterpret_cast<const f4_t*>(row + 32 * i);
      raw[2 * i + 1] = *reinterpret_cast<const f4_t*>(row + 32 * i + 4);
    }
    qs[u] = a.scale * 1.44269504088896340736f;
    float up = 1.f;
    if constexpr (F16) {  // into [2^13, 2^14) by a power of two (an infinity or NaN, or a row of zeros, stays what it is)
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(raw[i][e]));
      top = groups_max(top);
      int ex = (int)(__float_as_uint(top) >> 23) - 127;
      ex = ex == 128 ? 0 : min(13 - ex, 126);
      up = __builtin_amdgcn_ldexpf(1.f, ex);
      qs[u] = __builtin_amdgcn_ldexpf(qs[u], -ex);
    }
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y0 = raw[2 * i + (e >> 1)][2 * (e & 1)] * up, y1 = raw[2 * i + (e >> 1)][2 * (e & 1) + 1] * up;
        if constexpr (F16) {
          const h2_t w = {(_Float16)y0, (_Float16)y1};
          const h2_t z = {(_Float16)(y0 - (float)w[0]), (_Float16)(y1 - (float)w[1])};
          q[u][i][0][e] = __builtin_bit_cast(uint32_t, w);
          q[u][i][1][e] = __builtin_bit_cast(uint32_t, z);
        } else {
          uint32_t x, y, z;
          three(y0, y1, x, y, z);
          q[u][i][0][e] = x;
          q[u][i][1][e] = y;
          q[u][i][2][e] = z;
        }
      }
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[u][i] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) {
    lo_max = max(lo_max, __shfl_xor(lo_max, x));
    hi_min = min(hi_min, __shfl_xor(hi_min, x));
  }
  lo_max = uniform(lo_max);
  hi_min = uniform(hi_min);
  for (int tile = J.t0; tile < J.t1; tile = uniform(tile + 1)) {
    const Ids<true> more = ids_of<true>(c, pages, tile + (F16 ? AHEAD + 2 : 3));
    typename S::One& L = R.ring[F16 ? (tile - J.t0) & AHEAD : 0];
    if constexpr (F16) {
      // this tile's copies are there, the wave's by the wait and the others' by the barrier; that also frees the tile before
      if (tile + 2 < J.t1) copies_left<2 * COPIES>();
      else if (tile + 1 < J.t1) copies_left<COPIES>();
      else copies_left<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (tile + AHEAD < J.t1) copies.tile(R.ring[(tile - J.t0 + AHEAD) & AHEAD], c, J.h, id[AHEAD], tile + AHEAD, pages.end);
    } else {
      __syncthreads();  // (all waves have read the tile before)
      way.store(L);
      way.load(c, J.h, id[1], tile + 1, pages.end);
      __syncthreads();
    }
    if (!idle) {
      f4_t d[CG][2];
#pragma unroll
      for (int u = 0; u < CG; ++u) d[u][0] = d[u][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int at = S::k_at(16 * x + cl, 4 * i + kg);
          if constexpr (F16) {
            const u4_t k = L.k[0][at];
#pragma unroll
            for (int z = 1; z >= 0; --z)
#pragma unroll
              for (int u = 0; u < CG; ++u) d[u][x] = mfma(k, q[u][i][z], d[u][x]);
          } else {
            const u4_t k0 = L.k[0][at], k1 = L.k[1][at], k2 = L.k[2][at];
#pragma unroll
            for (int u = 0; u < CG; ++u) {
              d[u][x] = mfma_b(k2, q[u][i][0], d[u][x]);
              d[u][x] = mfma_b(k0, q[u][i][2], d[u][x]);
              d[u][x] = mfma_b(k1, q[u][i][1], d[u][x]);
              d[u][x] = mfma_b(k1, q[u][i][0], d[u][x]);
              d[u][x] = mfma_b(k0, q[u][i][1], d[u][x]);
              d[u][x] = mfma_b(k0, q[u][i][0], d[u][x]);
            }
          }
        }
      const bool inner = tile * TILE >= lo_max && (tile + 1) * TILE <= hi_min && id[0].id[0] >= 0 && id[0].id[1] >= 0;
      u4_t w[CG][F16 ? 2 : 3];
#pragma unroll
      for (int u = 0; u < CG; ++u) {
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = d[u][i >> 2][i & 3] * qs[u];
        if (!inner) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = tile * TILE + 16 * (i >> 2) + 4 * kg + (i & 3);
            if (j < lo[u] || j >= hi[u] || id[0].id[i >> 2] < 0) s[i] = -INFINITY;
          }
        }
        weigh_tile<F16>(s, m[u], l[u], o[u]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y0 = s[2 * i] * UP<F16>, y1 = s[2 * i + 1] * UP<F16>;
          if constexpr (F16) {
            const h2_t x = {(_Float16)y0, (_Float16)y1};
            const h2_t z = {(_Float16)(y0 - (float)x[0]), (_Float16)(y1 - (float)x[1])};
            w[u][0][i] = __builtin_bit_cast(uint32_t, x);
            w[u][1][i] = __builtin_bit_cast(uint32_t, z);
          } else {
            uint32_t x, y, z;
            three(y0, y1, x, y, z);
            w[u][0][i] = x;
            w[u][1][i] = y;
            w[u][2][i] = z;
          }
        }
      }
#pragma unroll
      for (int n = NP - 1; n >= 0; --n) {
        Tile<HD, true> T;  // (the plane's part of this lane, as fp16 pages' tiles are held)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int row = 16 * (j >> 2) + 4 * kg + (j & 3);
          if constexpr (HD == 128) {
            const u4_t x = L.v[n][row * PIECES + cl];
#pragma unroll
            for (int e = 0; e < 4; ++e) T.v[j][e] = x[e];
          } else {
            const uint2 x = *(reinterpret_cast<const uint2*>(&L.v[n][row * PIECES]) + cl);
            T.v[j][0] = x.x;
            T.v[j][1] = x.y;
          }
        }
        if (!inner && __any(T.template not_finite<F16>())) {
          // (as in run_job; a number that is not finite is so in its first part, and its other parts are dropped too)
          if (n == 0) {
#pragma unroll
            for (int u = 0; u < CG; ++u) {
              float sees[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int j = tile * TILE + 16 * (i >> 2) + 4 * kg + (i & 3);
                sees[i] = j < lo[u] || j >= hi[u] || id[0].id[i >> 2] < 0 ? 0.f : 1.f;
              }
#pragma unroll
              for (int x = 0; x < ND; ++x) {
                const f4_t plus = T.template sum<F16>(x, sees, false), minus = T.template sum<F16>(x, sees, true);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[u][x][r] += (plus[r] > 0.f ? INFINITY : 0.f) + (minus[r] > 0.f ? -INFINITY : 0.f);
              }
            }
          }
          T.template drop<F16>();
        }
#pragma unroll
        for (int y = 0; y < DW2; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u4_t v = T.operand(y, e);
            if constexpr (F16) {
#pragma unroll
              for (int z = 1; z >= 0; --z)
#pragma unroll
                for (int u = 0; u < CG; ++u) o[u][2 * y + e] = mfma(v, w[u][z], o[u][2 * y + e]);
              continue;
            }
#pragma unroll
            for (int u = 0; u < CG; ++u) {
              f4_t& to = o[u][2 * y + e];
              if constexpr (!F16) {
                if (n == 0) to = mfma_b(v, w[u][2], to);
                if (n <= 1) to = mfma_b(v, w[u][1], to);
                to = mfma_b(v, w[u][0], to);
              }
            }
          }
      }
    }
#pragma unroll
    for (int i = 0; i + 1 < (F16 ? AHEAD + 2 : 3); ++i) id[i] = id[i + 1];
    id[(F16 ? AHEAD + 2 : 3) - 1] = more;
  }
  __syncthreads();  // (all waves have read the last tile)
  static_assert(sizeof(float) * WAVES * 16 * turn_row(HD) <= sizeof(S), "");
  float* room = reinterpret_cast<float*>(&R) + wave * 16 * turn_row(HD);
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    l[u] = groups_sum(l[u]);
    put_columns<HD, HD, true>(a, p, J, room, col_base + 16 * u, 0, m[u], l[u], o[u], 1.f / UP<F16>);
  }
}

// Columns of a workgroup of a job of many, and the slots of its tiles.
constexpr bool staged(int hd) { return hd <= 128; }
constexpr int wide_groups(int hd, bool f16) { return f16 ? (staged(hd) ? 2 : 1) : staged(hd) ? 1 : 2; }  // of 16, a wave
constexpr int wide_columns(int hd, bool f16) { return 16 * sets_of(hd) * wide_groups(hd, f16); }
constexpr int wide_tile(int hd, bool f16) { return f16 || staged(hd) ? 32 : 16; }
template <int HD, bool F16>
union Room {
  Shared<HD, F16> narrow;
  Staged<staged(HD) ? HD : 64, F16> wide;
};
template <int HD, bool F16, bool WIDE>
IEK_DEV void run(const Paged& c, const PagedAttn& a, const Plan& p, const Job& J, Room<HD, F16>& L) {
  if constexpr (!WIDE) run_job<HD, F16, false, 1>(c, a, p, J, L.narrow);
  else if constexpr (staged(HD)) run_wide<HD, F16>(c, a, p, J, L.wide);
  else run_job<HD, F16, true, wide_groups(HD, F16)>(c, a, p, J, L.narrow);
}
template <int HD, bool F16, bool WIDE>
constexpr int TILE_OF = WIDE ? wide_tile(HD, F16) : tile_of<F16>();

// Workgroups: first the shared entries' ([chunk][column block][head]), then the own ones'. The chunks that do not
// exist are the last of their kind.
template <int HD, bool F16, bool PRE_WIDE, bool OWN_WIDE>
__global__ __launch_bounds__(64 * WAVES, 2) void part_kernel(Paged c, PagedAttn a, Plan p, int pre_groups) {
  __shared__ __align__(16) char room[PRE_WIDE ? sizeof(Room<HD, F16>) : sizeof(Shared<HD, F16>)];
  Room<HD, F16>& L = *reinterpret_cast<Room<HD, F16>*>(room);
  const int shared = shared_entries(a);
  Job J;
  // The shared chunks, which the matrix cores bound, and the own ones, which the memory bounds, take turns in runs of one
  // workgroup a CU, so that most CUs have one of each (32 sequences, 4096 shared f32 entries and up to 714 own ones: 49 us, with
  // the shared ones first 52).
  const int own_groups = gridDim.x - pre_groups, both = min(pre_groups, own_groups) / TURN * TURN;
  int id = blockIdx.x;
  bool pre = id < 2 * both ? id / TURN % 2 == 0 : id < both + pre_groups;
  if (id < 2 * both) id = id / (2 * TURN) * TURN + id % TURN;
  else id -= pre ? both : pre_groups;
  if (pre) {
    J.h = id % c.n_kv;
    id /= c.n_kv;
    J.block = id % p.pre_blocks;
    const int x = id / p.pre_blocks;
    const PreCut pc = pre_cut<TILE_OF<HD, F16, PRE_WIDE>>(c, a, p, shared);
    if (x >= pc.count) return;
    J.col0 = 0;
    J.cols = p.all;
    J.pages = Pages{a.shared_pages, shared};
    J.begin = 0;
    J.t0 = pc.t0 + x * pc.tiles;
    J.t1 = min(pc.t1, J.t0 + pc.tiles);
    const size_t row = ((size_t)x * c.n_kv + J.h) * p.all;
    J.ml = p.pml + 2 * row;
    J.o = p.po + row * HD;
    run<HD, F16, PRE_WIDE>(c, a, p, J, L);
    return;
  }
  J.h = id % c.n_kv;
  id /= c.n_kv;
  J.block = id % p.own_blocks;
  const int x = id / p.own_blocks;
  constexpr int TILE = TILE_OF<HD, F16, OWN_WIDE>;
  const Cut ct = cut<true, TILE, OWN_WIDE ? 1 : sets_of(HD)>(c, a, p, shared, x, 0);
  if (ct.count == 0) return;  // uniform
  J.col0 = ct.b * p.cols;
  J.cols = p.cols;
  J.pages = Pages{c.table + (size_t)ct.b * c.max_pages, ct.n};
  J.begin = shared;
  int t0, t1;
  own_range<TILE>(a, ct.n, shared, t0, t1);
  J.t0 = t0 + (x - ct.first) * ct.tiles;
  J.t1 = min(t1, J.t0 + ct.tiles);
  const size_t row = ((size_t)x * c.n_kv + J.h) * p.cols;
  J.ml = p.direct ? nullptr : p.ml + 2 * row;
  J.o = p.direct ? nullptr : p.o + row * HD;
  run<HD, F16, OWN_WIDE>(c, a, p, J, L);
}

// The join: 64 dims of a column of a KV head a workgroup, sixteen partial results at a time.
template <int HD, bool F16, bool PRE_WIDE, bool OWN_WIDE>
__global__ __launch_bounds__(256) void join_kernel(Paged c, PagedAttn a, Plan p) {
  constexpr int SD = 64, TPR = SD / 4, GRP = 256 / TPR, EARLY = 4;
  __shared__ float w[2 * MAX_SPLIT];
  __shared__ float red[2][4];
  __shared__ __align__(16) f4_t acc[GRP][TPR];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int slice = blockIdx.x % (HD / SD), hc = blockIdx.x / (HD / SD), h = hc / p.all, col = hc - h * p.all;
  const int b = col / p.cols, cc = col - b * p.cols;
  const int shared = shared_entries(a);
  const int pre = p.pre_chunks > 0 ? pre_cut<TILE_OF<HD, F16, PRE_WIDE>>(c, a, p, shared).count : 0;
  const Cut ct = cut<false, TILE_OF<HD, F16, OWN_WIDE>, OWN_WIDE ? 1 : sets_of(HD)>(c, a, p, shared, 0, b);
  const int live = pre + ct.count;
  const size_t pstep = (size_t)c.n_kv * p.all, ostep = (size_t)c.n_kv * p.cols;
  const size_t prow = (size_t)h * p.all + col, orow = (size_t)ct.first * ostep + (size_t)h * p.cols + cc;
  const int g = t / TPR, d = slice * SD + 4 * (t % TPR);
  auto part = [&](int i) {
    const float* o = i < pre ? p.po + (prow + i * pstep) * HD : p.o + (orow + (i - pre) * ostep) * HD;
    return *reinterpret_cast<const f4_t*>(o + d);
  };
  // the first ones are under way while their weights are made
  f4_t early[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) early[i] = g + i * GRP < live ? part(g + i * GRP) : f4_t{0.f, 0.f, 0.f, 0.f};
  float m[2], l[2], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int k = t + 256 * i;
    m[i] = -INFINITY;
    l[i] = 0.f;
    if (k < live) {
      const float* ml = k < pre ? p.pml + 2 * (prow + k * pstep) : p.ml + 2 * (orow + (k - pre) * ostep);
      m[i] = ml[0];
      l[i] = ml[1];
    }
    top = fmaxf(top, m[i]);
  }
  top = wave_max(top);
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float f = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - top);
    if (t + 256 * i < live) w[t + 256 * i] = f;
    sum += l[i] * f;
  }
  sum = wave_sum(sum);
  if (lane == 0) red[1][wave] = sum;
  __syncthreads();
  sum = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  f4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    if (g + i * GRP < live) y += early[i] * w[g + i * GRP];
#pragma unroll 4
  for (int i = g + EARLY * GRP; i < live; i += GRP) y += part(i) * w[i];
  acc[g][t % TPR] = y;
  __syncthreads();
  if (t < TPR) {
#pragma unroll
    for (int i = 1; i < GRP; ++i) y += acc[i][t];
    const int tq = cc / p.group;
    float* out = a.out + (((size_t)b * a.n_q + tq) * a.n_heads + h * p.group + cc - tq * p.group) * HD + d;
    *reinterpret_cast<f4_t*>(out) = sum == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : y / sum;
  }
}

// The same for many columns (2048 of 128 dims with one or two partial results 4.3 us, above 10; 512 of two or three 4.8 and
// 5.2; 256 of 64 5.0 and 4.8; 32 of 64 7.8 and 4.8): one a wave, and no barrier. A row takes HD / 4 lanes, so a wave sums 256 / HD partial results
// at a time (a lane has two pieces of a row of 512); 64 of the pairs are read at once and go to the lanes that need them.
template <int HD, bool F16, bool PRE_WIDE, bool OWN_WIDE>
__global__ __launch_bounds__(256) void join_columns_kernel(Paged c, PagedAttn a, Plan p) {
  constexpr int TPR = HD < 256 ? HD / 4 : 64, GRP = 64 / TPR, V = HD / 4 / TPR, EARLY = 4;
  const int lane = threadIdx.x & 63, hc = uniform(blockIdx.x * 4 + (threadIdx.x >> 6)), h = hc / p.all, col = hc - h * p.all;
  if (h >= c.n_kv) return;
  const int b = col / p.cols, cc = col - b * p.cols;
  const int shared = shared_entries(a);
  const int pre = p.pre_chunks > 0 ? pre_cut<TILE_OF<HD, F16, PRE_WIDE>>(c, a, p, shared).count : 0;
  const Cut ct = cut<false, TILE_OF<HD, F16, OWN_WIDE>, OWN_WIDE ? 1 : sets_of(HD)>(c, a, p, shared, 0, b);
  const int live = uniform(pre + ct.count);
  const size_t pstep = (size_t)c.n_kv * p.all, ostep = (size_t)c.n_kv * p.cols;
  const size_t prow = (size_t)h * p.all + col, orow = (size_t)ct.first * ostep + (size_t)h * p.cols + cc;
  const int g = lane / TPR, d = 4 * (lane % TPR);
  f4_t y[V];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) y[v] = f4_t{0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < live; first += 64) {
    const int n = min(64, live - first);
    float m = -INFINITY, l = 0.f;
    if (lane < n) {
      const int k = first + lane;
      const float* ml = k < pre ? p.pml + 2 * (prow + k * pstep) : p.ml + 2 * (orow + (k - pre) * ostep);
      m = ml[0];
      l = ml[1];
    }
    auto part = [&](int i, int v) {
      const int k = first + min(i, n - 1);
      const float* o = k < pre ? p.po + (prow + k * pstep) * HD : p.o + (orow + (k - pre) * ostep) * HD;
      return *reinterpret_cast<const f4_t*>(o + d + 256 * v);
    };
    f4_t x[EARLY][V];  // (under way while the weights are made)
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) x[i][v] = part(i * GRP + g, v);
    const float old = top;
    top = fmaxf(top, wave_max(m));
    const float down = old == top ? 1.f : __builtin_amdgcn_exp2f(old - top);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    sum = sum * down + wave_sum(l * f);
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] *= down;
    for (int i = 0; i < n; i += EARLY * GRP) {
#pragma unroll
      for (int e = 0; e < EARLY; ++e) {
        const int at = i + e * GRP + g;
        const float w = __shfl(f, min(at, 63));
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (at < n) y[v] += x[e][v] * w;
          x[e][v] = part(at + EARLY * GRP, v);
        }
      }
    }
  }
#pragma unroll
  for (int s = TPR; s < 64; s <<= 1)
#pragma unroll
    for (int r = 0; r < 4; ++r) y[0][r] += __shfl_xor(y[0][r], s);
  if (g == 0) {
    const int tq = cc / p.group;
    float* out = a.out + (((size_t)b * a.n_q + tq) * a.n_heads + h * p.group + cc - tq * p.group) * HD + d;
#pragma unroll
    for (int v = 0; v < V; ++v) *reinterpret_cast<f4_t*>(out + 256 * v) = sum == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : y[v] / sum;
  }
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }
int tile_of_kind(const Paged& c, bool wide) { return wide ? wide_tile(c.hd, c.f16) : c.f16 ? 32 : 16; }
int blocks_of(const Paged& c, long long cols, bool wide) {
  const int per = wide ? wide_columns(c.hd, c.f16) : 16;
  return (int)((cols + per - 1) / per);
}

// The plan for own parts of at most `own` entries (which may begin inside a tile: `edge`) and `shared` shared ones;
// more of them never need less.
Plan make_plan(const Paged& c, int n_heads, int n_q, int own, int shared, bool edge) {
  Plan p{};
  const int sets = sets_of(c.hd);
  p.group = n_heads / c.n_kv;
  p.cols = p.group * n_q;
  p.all = p.cols * c.batch;
  // Up to 32 columns a sequence take one or two workgroups, each with its tiles in registers. (Part launch, 16 sequences up to
  // 2048 of 8 KV heads of 128, 20 columns: fp16 21.5 us, as many columns 30; f32 43.5 and 42.5; one sequence of 500 10.7 us
  // without a join, as many columns 11.0 and one. With 64 columns in four workgroups f32 takes 80 us, as many columns 48.)
  p.own_wide = p.cols > 32;
  p.pre_wide = p.own_wide || (shared > 0 && p.all > 16);
  const int tile = tile_of_kind(c, p.own_wide), pre_tile = tile_of_kind(c, p.pre_wide);
  p.own_blocks = blocks_of(c, p.cols, p.own_wide);
  p.pre_blocks = blocks_of(c, p.all, p.pre_wide);
  constexpr int target = 512;  // workgroups that fill the chip once, two a CU
  const int tiles = (own + tile - 1) / tile + (edge ? 1 : 0);
  const int step = p.own_wide ? 1 : sets;
  // Up to so many tiles a sequence is one chunk and has no join, a launch of 4 us: a further tile of each set takes 0.7 to
  // 1.2 us (one sequence of 250 f32 entries, 32 heads of 128: one chunk 11.2 us, two 12.9; 500 fp16 ones 9.8 and 12.2).
  // Where there is a join anyway, chunks are as small as they come as long as the chip is not full: 531 entries of one
  // sequence 7.2 us, with two tiles a set 8.5; a window of 512 over 64 columns of 256 dims 13.4, with four tiles 20.
  const int whole = p.own_wide ? 4 : 4 * step;
  p.direct = shared == 0 && tiles <= whole;
  p.tiles = p.direct ? whole : p.own_wide && staged(c.hd) ? 2 : step;
  if (c.batch <= SHARED_BATCH) {
    p.share = std::max(1, target / (c.n_kv * p.own_blocks));
    p.nsplit = 0;
    // (sum of ceil(tiles / size) <= total / size + batch, size >= total / share)
    p.chunks = (int)std::min<long long>(p.share + c.batch, (long long)c.batch * std::max(1, (tiles + p.tiles - 1) / p.tiles));
  } else {
    const long long units = (long long)c.batch * c.n_kv * p.own_blocks;
    const int want = (int)std::max<long long>(1, std::min<long long>(MAX_SPLIT, 2 * target / units));
    p.nsplit = std::max(1, std::min(want, (tiles + p.tiles - 1) / p.tiles));
    p.tiles = std::max(p.tiles, ((tiles + p.nsplit - 1) / p.nsplit + step - 1) / step * step);
    p.chunks = c.batch * p.nsplit;
    p.direct = shared == 0 && p.nsplit == 1;
  }
  if (shared > 0) {
    const int pt = (shared + pre_tile - 1) / pre_tile;
    p.pre_tiles = !p.pre_wide ? sets : staged(c.hd) ? 2 : 1;
    p.pre_chunks = std::max(1, std::min({MAX_SPLIT, (pt + p.pre_tiles - 1) / p.pre_tiles, (int)(target / ((long long)c.n_kv * p.pre_blocks))}));
  }
  return p;
}

struct Sizes {
  size_t ml, o, pml, po;
  size_t all() const { return ml + o + pml + po; }
};
Sizes sizes(const Paged& c, const Plan& p) {
  const size_t own = p.direct ? 0 : (size_t)p.chunks * c.n_kv * p.cols, pre = (size_t)p.pre_chunks * c.n_kv * p.all;
  return {up256(own * 8), up256(own * c.hd * 4), up256(pre * 8), up256(pre * c.hd * 4)};
}

// Workgroups of the shared entries, of the own ones and of the join.
struct Grid {
  int pre, own, join;
};
Grid grid_of(const Paged& c, const Plan& p) {
  const long long pre = (long long)p.pre_chunks * p.pre_blocks * c.n_kv, own = (long long)p.chunks * p.own_blocks * c.n_kv;
  const long long join = p.direct ? 0 : (long long)c.n_kv * p.all * (c.hd / 64);
  if (pre + own >= 1 << 24 || join >= 1 << 24) fail(ST_OP, "paged: dims too large");  // (2^32 threads)
  return {(int)pre, (int)own, (int)join};
}

template <int HD, bool F16>
void launch_hd(const Paged& c, const PagedAttn& a, const Plan& p, hipStream_t st) {
  const Grid g = grid_of(c, p);
  auto go = [&](auto pre, auto own) {
    constexpr bool PRE = decltype(pre)::value, OWN = decltype(own)::value;
    hipLaunchKernelGGL((part_kernel<HD, F16, PRE, OWN>), dim3((unsigned)(g.pre + g.own)), dim3(64 * WAVES), 0, st, c, a, p, g.pre);
    if (g.join == 0) return;
    const int columns = c.n_kv * p.all;
    if (columns < JOIN_WAVES) hipLaunchKernelGGL((join_kernel<HD, F16, PRE, OWN>), dim3((unsigned)g.join), dim3(256), 0, st, c, a, p);
    else hipLaunchKernelGGL((join_columns_kernel<HD, F16, PRE, OWN>), dim3((unsigned)(columns + 3) / 4), dim3(256), 0, st, c, a, p);
  };
  // (own_wide: pre_wide, too)
  if (p.own_wide) go(std::true_type{}, std::true_type{});
  else if (p.pre_wide) go(std::true_type{}, std::false_type{});
  else go(std::false_type{}, std::false_type{});
}

}  // namespace

size_t paged_attention_workspace(const Paged& c, int n_heads, int n_q, int max_len, int max_shared) {
  if (c.batch == 0 || n_q == 0) return 0;
  const Plan p = make_plan(c, n_heads, n_q, max_len, max_shared, true);
  grid_of(c, p);  // (refuses)
  return sizes(c, p).all();
}

void launch_paged_attention(const Paged& c, const PagedAttn& a, void* ws, hipStream_t st) {
  // the entries that a sequence's columns see at most, wherever they begin in their tile
  const long long span = a.window > 0 ? std::min<long long>(a.max_len, (long long)a.window + a.n_q - 1) : a.max_len;
  Plan p = make_plan(c, a.n_heads, a.n_q, (int)span, a.max_shared, span < a.max_len);
  const Sizes z = sizes(c, p);
  if (p.pre_wide && !p.own_wide) {
    // Two workgroups a CU read the shared entries; if the own ones are twice their tiles or more, and so the longer work,
    // one does, and own ones take the other place: half the partial results. (Part and join, one and two: 4096 shared f32
    // entries and up to 714 own ones of 32 sequences 47 and 55 us, fp16 33 and 41; 16384 shared fp16 entries of 64 sequences
    // with up to 2616 own ones 111 and 132, with up to 616, on the other side of the rule, 91 and 85.)
    const long long mine = a.window > 0 ? span : std::max(0, a.max_len - a.max_shared);
    const long long own = (long long)c.batch * p.own_blocks * (mine / tile_of_kind(c, false));
    const long long shared = (long long)p.pre_blocks * (a.max_shared / tile_of_kind(c, true));
    if (own >= 2 * shared) p.pre_chunks = std::min(p.pre_chunks, std::max(1, (int)(256 / ((long long)c.n_kv * p.pre_blocks))));
  }
  char* base = static_cast<char*>(ws);
  p.ml = reinterpret_cast<float*>(base);
  p.o = reinterpret_cast<float*>(base + z.ml);
  p.pml = reinterpret_cast<float*>(base + z.ml + z.o);
  p.po = reinterpret_cast<float*>(base + z.ml + z.o + z.pml);
  auto go = [&](auto f) {
    constexpr bool F16 = decltype(f)::value;
    switch (c.hd) {
      case 64: launch_hd<64, F16>(c, a, p, st); break;
      case 128: launch_hd<128, F16>(c, a, p, st); break;
      case 256: launch_hd<256, F16>(c, a, p, st); break;
      default: launch_hd<512, F16>(c, a, p, st); break;
    }
  };
  if (c.f16) go(std::true_type{});
  else go(std::false_type{});
}

}  // namespace iek
