// Attention of one or several new tokens per sequence over the 8-bit KV cache (kv8.h).
//
// Column c = t * G + g of a KV head is query token t, query head g of its group of G. It sees the
// entries [lo, hi): hi = len - (n_q - 1 - t), lo = hi - window with a window, else 0. With scores s in
// base 2, out = (sum 2^(s - m) v) / (sum 2^(s - m)).
//
// The work is reading the codes once. A wave takes 32 slots (one block, one scale) at a time, both
// products on the matrix cores in fp16, which holds every code exactly, with 16 columns a product: eight
// query columns, each as two halves of an fp16 (hi, lo) pair that carries 22 bits (the sums are f32).
//   S^T[slot][column] = K q: K's bytes are a lane's own row, converted in registers;
//   O^T[dim][column] += V^T P: P comes out of the first product in the layout the second one takes
//     (slots 4 kg .. 4 kg + 3 of both halves of the block are the eight terms of lane group kg), V's bytes
//     are loaded as rows and transposed in registers, 2 x 2 values at a time.
// Nothing is staged in LDS before the end of a chunk. q is scaled by a power of two into fp16's range,
// P by 2^14 relative to its block's largest score of the column, so that neither can leave it: the
// factor between the block's and the running maximum, and V's scale, are applied to the f32 products.
#include <cfloat>

#include "common.cuh"
#include "kv8.h"
#include "kv8_codes.cuh"

namespace iek {

namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr int TILE = KV8_BLOCK;
constexpr int WAVES = 4;
constexpr int MAX_SPLIT = 256;

// A wave takes DIMS of a row: up to head_dim 128 all of them, and the four waves four tiles at a time;
// of wider rows two or four waves take 128 each of one tile, so that a tile's work, and the registers of q
// and o, are no larger (one wave a row had 256 accumulators and more at 512: 8223 keys of one KV head
// 26 us, so 13.8).
constexpr int dims_of(int hd) { return hd < 128 ? hd : 128; }
constexpr int tile_waves(int hd) { return WAVES * dims_of(hd) / hd; }

// A sequence's tiles are cut into chunks, whole rounds of a workgroup's waves, one workgroup and one
// partial result each. Up to SHARED_BATCH sequences the chunk's size is found on the device from the
// lengths themselves (a launch is sized for max_len, and may be a captured one): the total over the
// sequences by the chunks that fill the chip (half of one a sequence is lost to its last chunk), then
// each sequence evenly into as many as that takes: a batch of ragged lengths is spread evenly, and a
// short sequence in a large cache finely (16 sequences up to 8223 keys, cut by max_len 48 us, so 36). A
// chunk's number is its place in the running sum of the sequences' counts; a sequence without entries has
// one chunk, which writes zeros. Larger batches are cut by max_len.
constexpr int SHARED_BATCH = 64;

struct Plan {
  int group, cols, cblocks;  // query heads and columns of a KV head, workgroups the columns are spread over
  int groups;                // of eight columns a workgroup
  int share;                 // chunks of a KV head to aim at; 0: sequences are cut by `tiles`
  int tiles, nsplit;         // share 0: tiles a chunk, chunks a sequence at most; else the smallest chunk
  int chunks;                // of a KV head at most
  bool direct;               // every sequence is one chunk
  int spad;                  // stored scores a column
  float* ml;                 // [chunks][n_kv][cols] pairs (m, l)
  float* o;                  // [chunks][n_kv][cols][hd]
  float* s;                  // [batch][n_kv][cols][spad], base 2, or null
};

// The slots that the columns of query token t see, and the tile range [t0, t1) that any column sees.
IEK_DEV int col_hi(const Kv8Attn& a, int n, int t) { return n - (a.n_q - 1 - t); }
IEK_DEV int col_lo(const Kv8Attn& a, int hi) { return a.window > 0 ? max(0, hi - a.window) : 0; }
IEK_DEV int entries(const Kv8Attn& a, int b) { return max(0, min(a.len[b], a.max_len)); }
IEK_DEV void tile_range(const Kv8Attn& a, int n, int& t0, int& t1) {
  t0 = col_lo(a, max(0, col_hi(a, n, 0))) / TILE;
  t1 = (n + TILE - 1) / TILE;
}

// Chunk x of a KV head (FIND), or the chunks of sequence b: its entries n, tiles a chunk, number of
// chunks (0 with FIND: there is no chunk x) and first chunk.
struct Cut {
  int b, n, tiles, count, first;
};
IEK_DEV int ceil_div(int a, int b) { return (int)(((unsigned)a + b - 1) / (unsigned)b); }
// the same for tiles of one sequence (below 2^22, so that the product with the reciprocal is off by less than one)
IEK_DEV int ceil_div_tiles(int a, int b) {
  const int up = a + b - 1, q = (int)((float)up * __builtin_amdgcn_rcpf((float)b)), r = up - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}
IEK_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <bool FIND, int HD>
IEK_DEV Cut cut(const Kv8& c, const Kv8Attn& a, const Plan& p, int x, int b) {
  constexpr int TW = tile_waves(HD);
  Cut r{b, 0, p.tiles, 0, 0};
  int t0, t1;
  if (p.share == 0 || c.batch == 1) {
    if (FIND) r.b = c.batch == 1 ? 0 : min(x / p.nsplit, c.batch - 1);  // (the grid may be rounded up)
    r.n = entries(a, r.b);
    tile_range(a, r.n, t0, t1);
    if (p.share != 0)
      r.tiles = max(p.tiles, ceil_div(uniform(ceil_div_tiles(t1 - t0, min(p.share, MAX_SPLIT))), TW) * TW);
    r.count = max(1, uniform(ceil_div_tiles(t1 - t0, r.tiles)));
    r.first = r.b * p.nsplit;
    if (FIND && x - r.first >= r.count) r.count = 0;
    return r;
  }
  const int lane = threadIdx.x & 63;
  const int n = lane < c.batch ? entries(a, lane) : 0;
  tile_range(a, n, t0, t1);
  const int each = lane < c.batch ? t1 - t0 : 0;
  const int total = __builtin_amdgcn_readlane(wave_scan(each), 63);
  const int most = (int)wave_max((float)each);  // (exact: a sequence has at most 2^21 tiles)
  const int aim = max(p.share - c.batch / 2, (p.share + 1) / 2);
  const int size = max(p.tiles, ceil_div(max(ceil_div(total, aim), ceil_div(most, MAX_SPLIT)), TW) * TW);
  const int even = max(p.tiles, ceil_div(ceil_div_tiles(each, max(1, ceil_div_tiles(each, size))), TW) * TW);
  const int mine = lane < c.batch ? max(1, ceil_div_tiles(each, even)) : 0, upto = wave_scan(mine);
  if (FIND) r.b = __popcll(__ballot(lane < c.batch && upto - mine <= x)) - 1;
  r.n = __builtin_amdgcn_readlane(n, r.b);
  r.tiles = __builtin_amdgcn_readlane(even, r.b);
  r.count = __builtin_amdgcn_readlane(mine, r.b);
  r.first = __builtin_amdgcn_readlane(upto, r.b) - r.count;
  if (FIND && x - r.first >= r.count) r.count = 0;
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
// v plus the value of the lane eight further in its row of 16: the hi and lo columns
IEK_DEV float pair_sum(float v) { return v + dpp_f<0x128>(0.f, v); }  // row_ror:8

// Four codes as fp16: pairs (0, 1) and (2, 3). int8: as 1024 + (code + 128), whose fp16 bits are
// 0x6400 | byte, minus 1152.
template <bool E4M3>
IEK_DEV void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
  } else {
    w ^= 0x80808080u;
    const h2_t k = {(_Float16)-1152.f, (_Float16)-1152.f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + k);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + k);
  }
}

IEK_DEV f4_t mfma(u4_t a, u4_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
}

// Raw bytes of a wave's part of a tile: K, two sets of 16 rows, 16 bytes per 64 dims; V, eight rows of
// DIMS / 16 bytes.
template <int DIMS>
struct Tile {
  static constexpr int KC = DIMS / 64, VW = DIMS / 64;  // 16-byte pieces of K a row, dwords of V a row
  u4_t k[2][KC];
  uint32_t v[8][VW];
  float ks, vs;
};

// Buffer accesses end at the last live row of the tile: the rows behind it read as zero codes, whatever
// they hold (a NaN code would reach O through a weight of 0).
template <int HD>
IEK_DEV __amdgpu_buffer_rsrc_t tile_rsrc(const uint8_t* codes, int tile, int n) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(codes) + (size_t)tile * (TILE * HD), (short)0,
                                           min(TILE, n - tile * TILE) * HD, 0x00020000);
}

// (dim0: the wave's first dim)
template <int HD, int DIMS>
IEK_DEV void load_k(Tile<DIMS>& T, const uint8_t* codes, const float* ks, int tile, int n, int dim0, int lane) {
  const auto rs = tile_rsrc<HD>(codes, tile, n);
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < Tile<DIMS>::KC; ++i)
      T.k[s][i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (lane & 15) * HD + 16 * (lane >> 4),
                                                        dim0 + 16 * s * HD + 64 * i, 0);
  T.ks = ks[tile];
}

template <int HD, int DIMS>
IEK_DEV void load_v(Tile<DIMS>& T, const uint8_t* codes, const float* vs, int tile, int n, int dim0, int lane) {
  constexpr int VW = Tile<DIMS>::VW;
  static_assert(VW == 1 || VW == 2, "dims of a lane");
  const auto rs = tile_rsrc<HD>(codes, tile, n);
  const int off = 4 * (lane >> 4) * HD + (DIMS / 16) * (lane & 15);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = dim0 + (16 * (j >> 2) + (j & 3)) * HD;
    if constexpr (VW == 1) {
      T.v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, row, 0);
    } else {
      const auto x = __builtin_amdgcn_raw_buffer_load_b64(rs, off, row, 0);
      T.v[j][0] = x[0];
      T.v[j][1] = x[1];
    }
  }
  T.vs = vs[tile];
}

// One workgroup: CG * 8 columns of a KV head over a chunk.
template <int HD, bool E4M3, int CG>
__global__ __launch_bounds__(64 * WAVES, 2) void part_kernel(Kv8 c, Kv8Attn a, Plan p) {
  constexpr int DIMS = dims_of(HD), TW = tile_waves(HD), DW = WAVES / TW;
  constexpr int NS = DIMS / 32;  // steps of the first product
  constexpr int ND = DIMS / 16;  // dims of a lane in the second: ND r + i of row r
  constexpr int VW = Tile<DIMS>::VW;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = lane >> 4, c8 = lane & 7;
  const bool lo_half = lane & 8;
  const int tw = wave / DW, dim0 = (wave % DW) * DIMS;
  // The chunks that do not exist are the last workgroups, so that the others spread evenly over the CUs (between
  // them they left some with three and some with one: 16 x 4096 keys of 8 heads 34 us instead of 29).
  int h = blockIdx.x, x = blockIdx.y, cb = 0;
  if (p.cblocks > 1) {  // the workgroups of a chunk's columns on one XCD: consecutive ones go to the eight in turn
    const int unit = (h >> 3) / p.cblocks * 8 + (h & 7);
    cb = (h >> 3) % p.cblocks;
    x = unit / c.n_kv;
    h = unit - x * c.n_kv;
  }
  // (a single sequence's queries are under way before its length is there)
  Cut ct{};
  if (c.batch != 1) ct = cut<true, HD>(c, a, p, x, 0);
  const int b = ct.b, bh = b * c.n_kv + h, G = p.group;
  // this lane's columns, and its part of their q: dims 64 i + 16 kg + [0, 16) as steps 2 i and 2 i + 1
  f4_t qr[CG][DIMS / 16];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    const int cc = min((cb * CG + u) * 8 + c8, p.cols - 1), t = a.n_q == 1 ? 0 : cc / G;
    const float* row = a.q + ((size_t)b * a.n_q + t) * a.q_stride + (size_t)(h * G + cc - t * G) * HD + dim0 + 16 * kg;
#pragma unroll
    for (int i = 0; i < DIMS / 64; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) qr[u][4 * i + e] = *reinterpret_cast<const f4_t*>(row + 64 * i + 4 * e);
  }
  if (c.batch == 1) ct = cut<true, HD>(c, a, p, x, 0);
  if (ct.count == 0) return;  // uniform
  const int n = ct.n;
  int t0, t1;
  tile_range(a, n, t0, t1);
  t0 += (x - ct.first) * ct.tiles;
  t1 = min(t1, t0 + ct.tiles);
  const uint8_t* K = c.k + (size_t)bh * c.cap * HD;
  const uint8_t* V = c.v + (size_t)bh * c.cap * HD;
  const float* KS = c.ks + (size_t)bh * c.nblk;
  const float* VS = c.vs + (size_t)bh * c.nblk;
  Tile<DIMS> T;
  int tile = t0 + tw;
  if (tile < t1) {
    load_k<HD>(T, K, KS, tile, n, dim0, lane);
    load_v<HD>(T, V, VS, tile, n, dim0, lane);
  }
  u4_t q[CG][NS];
  const float less = lo_half ? -1.f : 0.f;
  float qs[CG];
  int hi[CG], lo[CG];
  int lo_max = 0, hi_min = n;
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    const int cc = min((cb * CG + u) * 8 + c8, p.cols - 1);
    hi[u] = col_hi(a, n, a.n_q == 1 ? 0 : cc / G);
    lo[u] = col_lo(a, hi[u]);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < DIMS / 16; ++i)
#pragma unroll
      for (int f = 0; f < 4; ++f) top = fmaxf(top, fabsf(qr[u][i][f]));
    top = groups_max(top);
    // into [2^13, 2^14) by a power of two (an infinity or NaN, or a row of zeros, stays what it is)
    int ex = (int)(__float_as_uint(top) >> 23) - 127;
    ex = ex == 128 ? 0 : min(13 - ex, 126);
    const float up = __builtin_amdgcn_ldexpf(1.f, ex);
    qs[u] = __builtin_amdgcn_ldexpf(a.scale * 1.44269504088896340736f, -ex);
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f4_t v = qr[u][2 * i + (e >> 1)];
        const float y0 = v[2 * (e & 1)] * up, y1 = v[2 * (e & 1) + 1] * up;
        const h2_t w = {(_Float16)y0, (_Float16)y1};  // hi, or what that rounds off
        const h2_t z = {(_Float16)fmaf((float)w[0], less, y0), (_Float16)fmaf((float)w[1], less, y1)};
        q[u][i][e] = __builtin_bit_cast(uint32_t, z);
      }
    lo_max = max(lo_max, lo[u]);
    hi_min = min(hi_min, hi[u]);
  }
  // (over the workgroup's columns, which are in ascending order of t)
  lo_max = __builtin_amdgcn_readlane(lo_max, 7);
  hi_min = __builtin_amdgcn_readlane(hi_min, 0);
  float m[CG], l[CG];
  f4_t o[CG][ND];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[u][i] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  // P's column of this lane: e's fp16, or 2^11 times what that rounds off (taken back from o at the end)
  const float rest = lo_half ? -2048.f : 0.f, keep = lo_half ? 2048.f : 1.f;

  __shared__ __align__(16) f4_t parts[DW > 1 ? 2 : 1][DW > 1 ? WAVES : 1][CG][64];  // a tile's scores from each wave's dims
  const int t_end = DW > 1 ? t0 + ceil_div(t1 - t0, TW) * TW : t1;  // (all waves go through the barriers)
  for (int turn = 0; tile < t_end; tile = __builtin_amdgcn_readfirstlane(tile + TW), turn ^= 1) {
    const bool have = DW == 1 || tile < t1;
    const bool inner = tile * TILE >= lo_max && (tile + 1) * TILE <= hi_min;  // every column sees all of it
    const bool more = tile + TW < t1;
    float s[CG][8], ks = 0.f;
    if (have) {
      f4_t d[CG][2];
#pragma unroll
      for (int u = 0; u < CG; ++u) d[u][0] = d[u][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          u4_t k;
          uint32_t y, z;
          codes_f16<E4M3>(T.k[r][i >> 1][2 * (i & 1)], y, z);
          k[0] = y;
          k[1] = z;
          codes_f16<E4M3>(T.k[r][i >> 1][2 * (i & 1) + 1], y, z);
          k[2] = y;
          k[3] = z;
#pragma unroll
          for (int u = 0; u < CG; ++u) d[u][r] = mfma(k, q[u][i], d[u][r]);
        }
      ks = T.ks;
      if (more) load_k<HD>(T, K, KS, tile + TW, n, dim0, lane);
#pragma unroll
      for (int u = 0; u < CG; ++u) {
        const float f = DW == 1 ? qs[u] * ks : qs[u];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[u][i] = pair_sum(d[u][i >> 2][i & 3]) * f;
        if (DW > 1)  // both halves of a row of lanes have all eight: four each
          parts[turn][wave][u][lane] =
              lo_half ? f4_t{s[u][4], s[u][5], s[u][6], s[u][7]} : f4_t{s[u][0], s[u][1], s[u][2], s[u][3]};
      }
    }
    if constexpr (DW > 1) {
      __syncthreads();
      if (!have) continue;
#pragma unroll
      for (int u = 0; u < CG; ++u) {
        f4_t y = parts[turn][tw * DW][u][lane & ~8], z = parts[turn][tw * DW][u][lane | 8];
#pragma unroll
        for (int w = 1; w < DW; ++w) {  // (in the same order in every wave: their maxima are the same)
          y += parts[turn][tw * DW + w][u][lane & ~8];
          z += parts[turn][tw * DW + w][u][lane | 8];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[u][i] = y[i] * ks;
          s[u][4 + i] = z[i] * ks;
        }
      }
    }
    u4_t pr[CG];
    float fac[CG];
#pragma unroll
    for (int u = 0; u < CG; ++u) {
      if (!inner) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = tile * TILE + 16 * (i >> 2) + 4 * kg + (i & 3);
          if (j < lo[u] || j >= hi[u]) s[u][i] = -INFINITY;
        }
      }
      if (p.s && dim0 == 0) {
        const int col = (cb * CG + u) * 8 + c8;
        float* to = p.s + ((size_t)bh * p.cols + col) * p.spad + tile * TILE + 4 * kg + (lo_half ? 16 : 0);
        const f4_t v = lo_half ? f4_t{s[u][4], s[u][5], s[u][6], s[u][7]} : f4_t{s[u][0], s[u][1], s[u][2], s[u][3]};
        if (col < p.cols) *reinterpret_cast<f4_t*>(to) = v;
      }
      float top = s[u][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[u][i]);
      top = groups_max(top);
      // The running maximum is only a reference: it moves when a block's is more than 2^8 above it.
      if (__any(top > m[u] + 8.f || (m[u] == -INFINITY && top > m[u]))) {
        const bool up = top > m[u] + 8.f || m[u] == -INFINITY;
        const float corr = up && m[u] != -INFINITY ? __builtin_amdgcn_exp2f(m[u] - top) : 1.f;  // (all is 0 before)
        if (up) m[u] = top;
        l[u] *= corr;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[u][i] *= corr;
      }
      const float ref = top == -INFINITY ? 0.f : top;
      fac[u] = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - m[u] - 14.f);
      float sum = 0.f, x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(s[u][i] - ref + 14.f);
        sum += x[i];
      }
      l[u] += sum * fac[u];  // (NaN with a NaN among the scores, also if the largest of the others is -inf)
      fac[u] = top == -INFINITY ? 0.f : fac[u] * T.vs;  // (a column that sees none of the block takes no NaN from it)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h2_t e = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
        const h2_t f = {(_Float16)fmaf((float)e[0], rest, x[2 * i] * keep),
                        (_Float16)fmaf((float)e[1], rest, x[2 * i + 1] * keep)};
        pr[u][i] = __builtin_bit_cast(uint32_t, f);
      }
    }
    // Codes of a block with a NaN scale may be NaN (e4m3), times a weight of 0 too: the scale alone is to tell.
    if (E4M3 && isnan(__uint_as_float(uniform(__float_as_uint(T.vs))))) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) T.v[j][w] = 0;
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      uint32_t x[8][2];
#pragma unroll
      for (int j = 0; j < 8; ++j) codes_f16<E4M3>(T.v[j][w], x[j][0], x[j][1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = __builtin_amdgcn_perm(x[2 * j + 1][e >> 1], x[2 * j][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int u = 0; u < CG; ++u) {
          const f4_t t = mfma(v, pr[u], f4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) o[u][4 * w + e][r] += t[r] * fac[u];
        }
      }
    }
    if (more) load_v<HD>(T, V, VS, tile + TW, n, dim0, lane);
  }

  // The waves' parts: to a common maximum, then summed through LDS, one wave after the other's columns.
  __shared__ float sm[TW][8 * CG], sl[TW][8 * CG];
  __shared__ __align__(16) float so[TW][8][HD];
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    l[u] = groups_sum(l[u]);
    if (lane < 8 && dim0 == 0) {
      sm[tw][8 * u + lane] = m[u];
      sl[tw][8 * u + lane] = l[u];
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < CG; ++u) {
    float top = sm[0][8 * u + c8];
#pragma unroll
    for (int w = 1; w < TW; ++w) top = fmaxf(top, sm[w][8 * u + c8]);
    const float mine = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - top - (lo_half ? 11.f : 0.f));
    if (u > 0) __syncthreads();
    // dims dim0 + ND (4 kg + r) + i: for each r the lane has ND of them in a row, stored by the hi lanes for
    // r = 0, 1 and the lo lanes for r = 2, 3
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float y[ND];
#pragma unroll
      for (int i = 0; i < ND; ++i) y[i] = pair_sum(o[u][i][r] * mine);
      if (lo_half == (r >= 2)) {
#pragma unroll
        for (int i = 0; i < ND; i += 4)
          *reinterpret_cast<f4_t*>(&so[tw][c8][dim0 + ND * (4 * kg + r) + i]) = f4_t{y[i], y[i + 1], y[i + 2], y[i + 3]};
      }
    }
    __syncthreads();
    const int c0 = (cb * CG + u) * 8;
    for (int i = threadIdx.x; i < 8 * HD / 4; i += 64 * WAVES) {
      const int col = i / (HD / 4), dim = 4 * (i % (HD / 4));
      if (c0 + col >= p.cols) continue;
      f4_t y = *reinterpret_cast<const f4_t*>(&so[0][col][dim]);
#pragma unroll
      for (int w = 1; w < TW; ++w) y += *reinterpret_cast<const f4_t*>(&so[w][col][dim]);
      float mm = sm[0][8 * u + col];
#pragma unroll
      for (int w = 1; w < TW; ++w) mm = fmaxf(mm, sm[w][8 * u + col]);
      float ll = 0.f;
#pragma unroll
      for (int w = 0; w < TW; ++w)
        ll += sl[w][8 * u + col] * (sm[w][8 * u + col] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sm[w][8 * u + col] - mm));
      const size_t row = ((size_t)x * c.n_kv + h) * p.cols + c0 + col;
      if (p.direct) {
        const int t = (c0 + col) / G, g = (c0 + col) - t * G;
        float* out = a.out + (((size_t)b * a.n_q + t) * a.n_heads + h * G + g) * HD + dim;
        *reinterpret_cast<f4_t*>(out) = ll == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : y / ll;
      } else {
        *reinterpret_cast<f4_t*>(p.o + row * HD + dim) = y;
      }
      if (dim == 0) {
        p.ml[2 * row] = isnan(ll) ? ll : mm;  // (a NaN: the maxima pass it over)
        p.ml[2 * row + 1] = ll;
      }
    }
  }
}

// Largest m and sum of l 2^(m - top) over the chunks of a column, by one wave: ml the first chunk's pair, `step`
// columns apart. m and l are left in the lanes, chunk lane + 64 i.
IEK_DEV void column_sum(const float* ml, size_t step, int count, float (&m)[MAX_SPLIT / 64], float& top, float& sum) {
  const int lane = threadIdx.x & 63;
  float l[MAX_SPLIT / 64];
  top = -INFINITY;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < MAX_SPLIT / 64; ++i) {
    const int k = lane + 64 * i;
    m[i] = -INFINITY;
    l[i] = 0.f;
    if (64 * i < count && k < count) {
      m[i] = ml[2 * k * step];
      l[i] = ml[2 * k * step + 1];
    }
  }
#pragma unroll
  for (int i = 0; i < MAX_SPLIT / 64; ++i) top = fmaxf(top, m[i]);
  top = wave_max(top);
#pragma unroll
  for (int i = 0; i < MAX_SPLIT / 64; ++i) sum += m[i] == -INFINITY ? 0.f : l[i] * __builtin_amdgcn_exp2f(m[i] - top);
  sum = wave_sum(sum);
}

// A column's largest score and sum as m and r, with which an entry's weight is 2^(score - m) r. Out of the column's
// sight scores are -inf and weights 0; a NaN sum makes NaN (infinity times 0) of all others and of them nothing.
IEK_DEV void share_terms(float top, float sum, float& m, float& r) {
  m = isnan(sum) ? -FLT_MAX : top == -INFINITY ? 0.f : top;
  r = isnan(sum) || sum == 0.f ? 0.f : 1.f / sum;
}

// The join. Workgroups [0, ncol), unless the chunks have written the output themselves: 64 dims of a
// column, sixteen chunks at a time; those behind them: the weights of 1024 entries of a KV head. MANY
// (several query tokens: many columns of few chunks, where workgroups are what costs): 64 dims of four
// columns, a wave each; the weights of 256 entries, a quarter of the columns a wave (22 sequences up to
// 451 keys of 512, eleven tokens: 69 us without it, 40 so).
template <int HD, bool MANY>
__global__ __launch_bounds__(256) void join_kernel(Kv8 c, Kv8Attn a, Plan p, int ncol, int wblocks) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, G = p.group;
  constexpr int SD = 64, TPR = SD / 4, GRP = 256 / TPR;
  if (MANY && (int)blockIdx.x < ncol) {
    __shared__ float wc[4][MAX_SPLIT];
    const int quads = (p.cols + 3) / 4, id = blockIdx.x / (HD / SD), bh = id / quads;
    const int col = (id - bh * quads) * 4 + wave, b = bh / c.n_kv, h = bh - b * c.n_kv;
    if (col >= p.cols) return;  // (uniform in the wave; there is no barrier)
    const Cut ct = cut<false, HD>(c, a, p, 0, b);
    const int d = (blockIdx.x % (HD / SD)) * SD + 4 * (lane & 15);
    const size_t step = (size_t)c.n_kv * p.cols, row = (size_t)ct.first * step + (size_t)h * p.cols + col;
    float m[MAX_SPLIT / 64], top, sum;
    column_sum(p.ml + 2 * row, step, ct.count, m, top, sum);
#pragma unroll
    for (int i = 0; i < MAX_SPLIT / 64; ++i)
      if (64 * i < ct.count) wc[wave][lane + 64 * i] = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - top);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = lane >> 4; i < ct.count; i += 4)
      y += *reinterpret_cast<const f4_t*>(p.o + (row + i * step) * HD + d) * wc[wave][i];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = groups_sum(y[i]);
    const int tq = col / G;
    float* out = a.out + (((size_t)b * a.n_q + tq) * a.n_heads + h * G + col - tq * G) * HD + d;
    if (lane < 16) *reinterpret_cast<f4_t*>(out) = sum == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : y / sum;
    return;
  }
  if (!MANY && (int)blockIdx.x < ncol) {
    __shared__ float w[MAX_SPLIT];
    __shared__ float red[2][4];
    __shared__ __align__(16) float acc[GRP][SD];
    const int bc = blockIdx.x / (HD / SD), bh = bc / p.cols, col = bc - bh * p.cols, b = bh / c.n_kv, h = bh - b * c.n_kv;
    // of a single sequence the first parts, without waiting for its length
    constexpr int PRE = 4;
    const size_t step = (size_t)c.n_kv * p.cols;
    const int g = t / TPR, ds = 4 * (t % TPR), d = (blockIdx.x % (HD / SD)) * SD + ds;
    f4_t pre[PRE];
    if (c.batch == 1) {
#pragma unroll
      for (int k = 0; k < PRE; ++k)
        pre[k] = *reinterpret_cast<const f4_t*>(p.o + (min(g + GRP * k, p.chunks - 1) * step + bc) * HD + d);
    }
    const Cut ct = cut<false, HD>(c, a, p, 0, b);
    const int live = ct.count;
    const size_t row = (size_t)ct.first * step + (size_t)h * p.cols + col;
    float m = -INFINITY, l = 0.f;
    if (t < live) {
      m = p.ml[2 * (row + t * step)];
      l = p.ml[2 * (row + t * step) + 1];
    }
    float top = wave_max(m);
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    if (t < live) w[t] = f;
    l = wave_sum(l * f);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    f4_t y = {0.f, 0.f, 0.f, 0.f};
    int i0 = g;
    if (c.batch == 1) {
#pragma unroll
      for (int k = 0; k < PRE; ++k, i0 += GRP)
        if (i0 < live) y += pre[k] * w[i0];
    }
#pragma unroll 4
    for (int i = i0; i < live; i += GRP) y += *reinterpret_cast<const f4_t*>(p.o + (row + i * step) * HD + d) * w[i];
    *reinterpret_cast<f4_t*>(&acc[g][ds]) = y;
    __syncthreads();
    if (t < TPR) {
#pragma unroll
      for (int i = 1; i < GRP; ++i) y += *reinterpret_cast<const f4_t*>(&acc[i][ds]);
      const int tq = col / G;
      float* out = a.out + (((size_t)b * a.n_q + tq) * a.n_heads + h * G + col - tq * G) * HD + d;
      *reinterpret_cast<f4_t*>(out) = l == 0.f ? f4_t{0.f, 0.f, 0.f, 0.f} : y / l;
    }
    return;
  }
  constexpr int COLS = 64 * 8;  // n_q <= 64, groups of at most 8
  __shared__ float cm[COLS], cl[COLS];
  const int id = blockIdx.x - ncol, bh = id / wblocks, b = bh / c.n_kv, h = bh - b * c.n_kv;
  const int j0 = (id - bh * wblocks) * (MANY ? 256 : 1024), j = j0 + 4 * (MANY ? lane : t);
  // what does not wait for the lengths: the first columns' scores (`spad` of them are there) and the old sums
  constexpr int PRE = 8, CS = MANY ? 4 : 1;  // (column c0 + CS k)
  const int c0 = MANY ? wave : 0;
  const float* s = p.s + (size_t)bh * p.cols * p.spad + min(j, p.spad - 4);
  const size_t at = (size_t)bh * c.cap + j;
  f4_t v[PRE], w = {0.f, 0.f, 0.f, 0.f}, old = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int col = 0; col < PRE; ++col) v[col] = *reinterpret_cast<const f4_t*>(s + (size_t)min(c0 + CS * col, p.cols - 1) * p.spad);
  if (a.w_in) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < a.max_len) old[i] = a.w_in[at + i];
  }
  const Cut ct = cut<false, HD>(c, a, p, 0, b);
  const int n = ct.n;
  if (j0 >= n) return;  // uniform
  int t0, t1;
  tile_range(a, n, t0, t1);
  const size_t step = (size_t)c.n_kv * p.cols;
  // a wave a column, or, of many columns with few chunks, a thread
  const float* ml0 = p.ml + 2 * ((size_t)ct.first * step + (size_t)h * p.cols);
  if (!MANY || p.cols <= ct.count) {
    for (int col = wave; col < p.cols; col += 4) {
      float m[MAX_SPLIT / 64], top, sum;
      column_sum(ml0 + 2 * col, step, ct.count, m, top, sum);
      if (lane == 0) share_terms(top, sum, cm[col], cl[col]);
    }
  } else {
    for (int col = t; col < p.cols; col += 256) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll 4
      for (int k = 0; k < ct.count; ++k) top = fmaxf(top, ml0[2 * (k * step + col)]);
#pragma unroll 4
      for (int k = 0; k < ct.count; ++k) {
        const float m = ml0[2 * (k * step + col)], l = ml0[2 * (k * step + col) + 1];
        sum += m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f(m - top);
      }
      share_terms(top, sum, cm[col], cl[col]);
    }
  }
  __syncthreads();
  if (!MANY && j >= n) return;
  if (j < n && j >= t0 * TILE) {
#pragma unroll
    for (int k = 0; k < PRE; ++k) {
      const int col = c0 + CS * k;
      if (col >= p.cols) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(v[k][i] - cm[col]) * cl[col];
    }
#pragma unroll 8
    for (int col = c0 + CS * PRE; col < p.cols; col += CS) {
      const f4_t z = *reinterpret_cast<const f4_t*>(s + (size_t)col * p.spad);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(z[i] - cm[col]) * cl[col];
    }
  }
  if constexpr (MANY) {
    __shared__ f4_t part[4][64];
    part[wave][lane] = w;
    __syncthreads();
    if (wave != 0 || j >= n) return;
    w = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (j + i < n) a.w_out[at + i] = old[i] + w[i];
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Column groups of eight per workgroup. Two share the reading and the conversion of the codes, and take twice
// the registers and twice as long over a tile: they pay where the workgroups of one group each would go
// through more than ten times the chip (five tokens, 8 sequences of 4000 keys of 8 heads of 128: 38 us against 41;
// sixteen, 16 of 4000 of 256: 69 against 96; but five, 4 of 3001 of 64: 12.0 against 10.8).
int col_groups(const Kv8& c, int cols, int tiles) {
  const int tw = tile_waves(c.hd);
  const long long turns = (long long)c.batch * c.n_kv * ((cols + 7) / 8) * ((tiles + tw - 1) / tw);
  return cols > 8 && turns > 10 * 512 ? 2 : 1;
}

// The plan for sequences whose columns see at most `tiles` tiles; more of them never need less.
Plan make_plan(const Kv8& c, int n_heads, int n_q, int tiles) {
  Plan p{};
  p.group = n_heads / c.n_kv;
  p.cols = p.group * n_q;
  p.groups = col_groups(c, p.cols, tiles);
  const int per = 8 * p.groups, tw = tile_waves(c.hd);
  p.cblocks = (p.cols + per - 1) / per;
  // Chunks that fill the chip once, two workgroups a CU. Up to two rounds of the waves the second one costs
  // less than the joining of two chunks.
  constexpr int target = 512;
  p.tiles = tiles <= 2 * tw ? 2 * tw : tw;
  p.direct = tiles <= p.tiles;
  if (c.batch <= SHARED_BATCH) {
    p.share = std::max(1, target / (c.n_kv * p.cblocks));
    p.nsplit = 0;
    // (sum of ceil(tiles / size) <= total / size + batch, size >= total / share)
    p.chunks = (int)std::min<long long>(p.share + c.batch, (long long)c.batch * std::max(1, (tiles + p.tiles - 1) / p.tiles));
  } else {
    const long long units = (long long)c.batch * c.n_kv * p.cblocks;
    const int want = (int)std::max<long long>(1, std::min<long long>(MAX_SPLIT, 2 * target / units));
    p.nsplit = std::max(1, std::min(want, (tiles + p.tiles - 1) / p.tiles));
    p.tiles = std::max(p.tiles, ((tiles + p.nsplit - 1) / p.nsplit + tw - 1) / tw * tw);
    p.chunks = c.batch * p.nsplit;
    p.direct = p.nsplit == 1;
  }
  return p;
}

struct Sizes {
  size_t ml, o, s;
};
Sizes sizes(const Kv8& c, const Plan& p, int spad, bool weights) {
  const size_t rows = (size_t)p.chunks * c.n_kv * p.cols;
  return {up256(rows * 8), p.direct ? 0 : up256(rows * c.hd * 4),
          weights ? up256((size_t)c.batch * c.n_kv * p.cols * spad * 4) : 0};
}

// Workgroups of the join: `ncol` for columns, then `wblocks` a KV head for weights.
struct JoinGrid {
  int ncol, wblocks, all;
};
JoinGrid join_grid(const Kv8& c, const Plan& p, int max_len, bool weights) {
  const bool many = p.cols > 8;
  const long long heads = (long long)c.batch * c.n_kv;
  const long long ncol = p.direct ? 0 : heads * (c.hd / 64) * (many ? (p.cols + 3) / 4 : p.cols);
  const int wblocks = weights ? (max_len + (many ? 255 : 1023)) / (many ? 256 : 1024) : 0;
  const long long all = ncol + heads * wblocks;
  if (all >= 1 << 24) fail(ST_OP, "kv8: dims too large");  // (2^32 threads)
  return {(int)ncol, wblocks, (int)all};
}

template <int HD, int CG>
void launch_cg(const Kv8& c, const Kv8Attn& a, const Plan& p, hipStream_t st) {
  // (at most 65535 KV heads of 64 workgroups' columns each, or chunks that fill the chip: below 2^24 workgroups)
  const long long part = ((long long)p.chunks * c.n_kv + 7) / 8 * 8 * p.cblocks;
  const dim3 grid = p.cblocks == 1 ? dim3((unsigned)c.n_kv, (unsigned)p.chunks) : dim3((unsigned)part);
  const bool many = p.cols > 8;
  const JoinGrid join = join_grid(c, p, a.max_len, a.w_out != nullptr);
  auto fn = c.e4m3 ? part_kernel<HD, true, CG> : part_kernel<HD, false, CG>;
  hipLaunchKernelGGL(fn, grid, dim3(64 * WAVES), 0, st, c, a, p);
  if (join.all)
    hipLaunchKernelGGL((many ? join_kernel<HD, true> : join_kernel<HD, false>), dim3((unsigned)join.all), dim3(256), 0, st, c, a, p,
                       join.ncol, join.wblocks);
}

}  // namespace

// For any window: fewer tiles do not take more chunks, nor do smaller column groups; nor more workgroups in the join.
size_t kv8_attention_workspace(const Kv8& c, int n_heads, int n_q, int max_len, bool weights) {
  if (c.batch == 0 || n_q == 0) return 0;
  const int tiles = (max_len + TILE - 1) / TILE;
  Plan p = make_plan(c, n_heads, n_q, tiles);
  join_grid(c, p, max_len, weights);  // (refuses)
  const Sizes z = sizes(c, p, tiles * TILE, weights);
  return z.ml + z.o + z.s;
}

void launch_kv8_attention(const Kv8& c, const Kv8Attn& a, void* ws, hipStream_t st) {
  // the slots that a sequence's columns see at most, wherever they begin in their tile
  const long long span = a.window > 0 ? std::min<long long>(a.max_len, (long long)a.window + a.n_q + TILE - 2) : a.max_len;
  Plan p = make_plan(c, a.n_heads, a.n_q, (int)((span + TILE - 1) / TILE));
  p.spad = (a.max_len + TILE - 1) / TILE * TILE;
  const Sizes z = sizes(c, p, p.spad, a.w_out != nullptr);
  char* base = static_cast<char*>(ws);
  p.ml = reinterpret_cast<float*>(base);
  p.o = reinterpret_cast<float*>(base + z.ml);
  p.s = a.w_out ? reinterpret_cast<float*>(base + z.ml + z.o) : nullptr;
  const bool two = p.groups == 2;
  switch (c.hd) {
    case 64: two ? launch_cg<64, 2>(c, a, p, st) : launch_cg<64, 1>(c, a, p, st); break;
    case 128: two ? launch_cg<128, 2>(c, a, p, st) : launch_cg<128, 1>(c, a, p, st); break;
    case 256: two ? launch_cg<256, 2>(c, a, p, st) : launch_cg<256, 1>(c, a, p, st); break;
    default: two ? launch_cg<512, 2>(c, a, p, st) : launch_cg<512, 1>(c, a, p, st); break;
  }
}

}  // namespace iek
