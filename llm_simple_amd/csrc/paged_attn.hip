// Attention of new tokens over a cache in pages, gfx950: a batch of sequences of their own lengths, each with one new token or many, over
// all keys up to a token or over a sliding window of them and the first `sinks` keys.
//
//   out[t][h] = sum_c softmax_c(q[t][h] . K[c][h / g] / sqrt(128)) V[c][h / g],   c <= p, and c > p - window or c < sinks
//
// with p the position of token t (paged.hpp).  Query rows of a kv head are (token, head of its g) pairs, token-major, so that K and V of
// a kv head are read for all g heads at once.  Two kinds of workgroups, of four waves each:
//
//  * few rows: a sequence with at most 16 rows.  A stream of K and V through the chip: the rows are the 16 columns of mfma 16x16x32, a wave
//    takes every fourth piece of 32 keys, which it stages in LDS of its own (flash_decode.hip has the layout and why), and keeps its own
//    running maximum, sum and O; the four are merged at the end.
//  * tiles: 128 rows, 32 to a wave (wave_attn.hpp), over tiles of 64 keys in LDS, two of them, so that a tile is on its way while
//    the one before it is worked on.
//
// 8-bit rows become rows of the storage type on their way into LDS: each is widened once for all rows that use it, by a conversion
// that takes the row's power of two along, and everything after is the same code.
//
// Which sequence a workgroup is for is found on the device (lengths may change between replays of a graph): a wave looks at 64 sequences
// at a time.  The keys of a sequence are dealt to as many workgroups as there are pieces of `chunk` units in what its rows see, up to the
// launch's number of splits; then each leaves an fp32 partial, and a second launch folds them.  A unit is 128 keys (few rows) or 64.
//
// Keys that a row must not see: their scores become -inf, so their K does not matter, but a weight of 0 times a V that is not finite
// would be NaN.  Rows behind the last key, and pages that are not there, are zeros (the loads' descriptors end before them).  V of keys
// that only some rows see is what it is: a row whose result is not finite is computed again key by key (exact_row), from the
// keys that it sees alone.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "paged.hpp"
#include "wave_attn.hpp"

namespace llmhip {

constexpr int kFewCols = 16;     // rows of a few-rows workgroup
constexpr int kFewUnit = 128;    // keys of a unit, 32 to a wave
constexpr int kTileRows = 128;   // rows of a tile
constexpr int kTileUnit = 64;    // keys of a unit
constexpr int kUnitBytes = kTileUnit * kRowBytes;
constexpr int kWaveStage = 32 * kRowBytes;  // staging of a few-rows wave, for K and for V
constexpr int kPagedLds = 64 * 1024;

struct PagedAttn {
  PagedBatch batch;
  char *out;
  const char *q, *k, *v;
  float *few_o, *few_ml, *tile_o, *tile_ml;  // [tile][kv head][split][row][128], and [2]: maximum (times scale and log2 e), sum
  int H, Hkv, g;
  FastDiv g_div, Hkv_div, few_splits_div, tile_splits_div;
  int window, sinks;  // window 0: none
  int max_q_len;
  int few_rows;  // sequences of up to so many rows are few-rows ones; 0: none is
  int few_blocks;  // workgroups of the first kind in a launch of both
  int few_splits, few_chunk, tile_splits, tile_chunk;
};

// What a workgroup works on: `rows` rows from row `row0` of a sequence on
struct PagedTile {
  int b, start, m, len, row0, rows;
};

// Inclusive sum over the lanes of a wave
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15, into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31, into rows 2 and 3
  return x;
}

// Tile `w` of all tiles of one kind, a sequence's last (longest) one first.  False: there are not so many.
template <bool FEW> __device__ __forceinline__ bool find_tile(const PagedAttn &p, int w, int lane, PagedTile &t) {
  for (int base = 0; base < p.batch.batch; base += 64) {
    const int i = min(base + lane, p.batch.batch - 1);
    const int start = p.batch.q_starts[i], end = p.batch.q_starts[i + 1], len = p.batch.kv_lens[i];
    const bool valid = base + lane < p.batch.batch && sequence_ok(p.batch, start, end, len) && end - start <= p.max_q_len;
    const int m = valid ? end - start : 0, rows = m * p.g;
    const int mine = FEW ? (m > 0 && rows <= p.few_rows ? 1 : 0) : rows <= p.few_rows ? 0 : (rows + kTileRows - 1) / kTileRows;
    const int upto = wave_prefix(mine), all = __builtin_amdgcn_readlane(upto, 63);
    if (w >= all) {
      w -= all;
      continue;
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > w));
    t.b = base + l;
    t.start = __builtin_amdgcn_readlane(start, l);
    t.m = __builtin_amdgcn_readlane(m, l);
    t.len = __builtin_amdgcn_readlane(len, l);
    // 0 for the last tile (a few-rows sequence has one)
    const int at = w - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
    t.row0 = FEW ? 0 : (__builtin_amdgcn_readlane(mine, l) - 1 - at) * kTileRows;
    t.rows = min(t.m * p.g - t.row0, FEW ? kFewCols : kTileRows);
    return true;
  }
  return false;
}

// The keys that rows at positions p0 .. p1 see, in units of UNIT keys: the first `sink_units` of them are keys 0 .. sink_end, the rest
// begin at key `first`, a multiple of 16, and end at `end`.
struct PagedKeys {
  int sink_units, sink_end, first, end, units;
  __device__ __forceinline__ int base(int unit, int size) const { return unit < sink_units ? unit * size : first + (unit - sink_units) * size; }
  __device__ __forceinline__ int limit(int unit) const { return unit < sink_units ? sink_end : end; }
};
template <int UNIT> __device__ __forceinline__ PagedKeys keys_seen(const PagedAttn &p, int p0, int p1, int len) {
  PagedKeys k;
  k.end = max(min(p1 + 1, len), 0);
  k.first = p.window > 0 ? min(max(p0 - p.window + 1, 0), k.end) & ~(kPageGroup - 1) : 0;
  k.sink_end = min(p.sinks, k.first);
  if (p.window <= 0) k.sink_end = 0;
  k.sink_units = (k.sink_end + UNIT - 1) / UNIT;
  k.units = k.sink_units + (k.end - k.first + UNIT - 1) / UNIT;
  return k;
}

// Units u0 .. u1 of a split, and how many splits there are
struct PagedSplit {
  int count, u0, u1;
};
__device__ __forceinline__ PagedSplit split_of(int units, int split, int splits, int chunk) {
  PagedSplit s = {1, 0, units};
  if (splits > 1 && units > chunk) {
    const int want = min(splits, (units + chunk - 1) / chunk), each = (units + want - 1) / want;
    s.count = (units + each - 1) / each;
    s.u0 = min(split * each, units);
    s.u1 = min(s.u0 + each, units);
  }
  return s;
}

// Places of 64 groups of 16 keys, one to a lane
struct GroupPlaces {
  int page, row;
  __device__ __forceinline__ void look(const PagedAttn &p, int b, int key) {
    const PagePlace at = page_place(p.batch, b, key);
    page = at.page;
    row = at.row;
  }
};
// One group of 16 keys of a kv head
struct Group {
  int64_t page_at;  // bytes from the pool's base to the page
  int row;          // row among the page's rows of all kv heads
  int have;         // rows that are there
};
__device__ __forceinline__ Group group_of(const PagedAttn &p, const GroupPlaces &places, int lane, int kvh, int key, int limit) {
  Group g;
  const int page = __builtin_amdgcn_readlane(places.page, lane);
  g.page_at = (int64_t)page * p.batch.page_stride;
  g.row = kvh * (int)p.batch.page_size.d + __builtin_amdgcn_readlane(places.row, lane);
  g.have = page < 0 ? 0 : min(max(limit - key, 0), kPageGroup);
  if (g.have == 0) g.page_at = g.row = 0;
  return g;
}
template <bool EIGHT> __device__ __forceinline__ __amdgpu_buffer_rsrc_t group_buffer(const char *pool, const Group &g) {
  return byte_buffer(pool + g.page_at + (size_t)g.row * cached_row_bytes(EIGHT), g.have * cached_row_bytes(EIGHT));
}
// The same descriptor of a 16-bit group as words, for assembly
__device__ __forceinline__ u32x4_t group_words(const char *pool, const Group &g) {
  const uint64_t at = reinterpret_cast<uintptr_t>(pool + g.page_at + (size_t)g.row * kRowBytes);
  return u32x4_t{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, (uint32_t)(g.have * kRowBytes), 0x00020000u};
}
// Address of the exponent byte of a group's first row
__device__ __forceinline__ const uint8_t *group_exponents(const PagedAttn &p, const char *pool, const Group &g) {
  return reinterpret_cast<const uint8_t *>(pool + g.page_at + (size_t)p.Hkv * p.batch.page_size.d * kHeadDim + g.row);
}

__device__ __forceinline__ bool sees(const PagedAttn &p, int pos, int key) {
  return key <= pos && (p.window <= 0 || key > pos - p.window || key < p.sinks);
}

// One row by G lanes, from the keys that it sees alone; see the header.  dims G * i .. of lane i's: 128 / G of them from 128 / G * i on.
// M is in units of score times log2 e.
template <typename T, bool EIGHT, int G, int UNIT>
__device__ __forceinline__ void exact_row(const PagedAttn &p, int b, int kvh, const char *q_row, int pos, PagedKeys keys, int u0, int u1,
                                                    float &M, float &L, float (&o)[kHeadDim / G]) {
  constexpr int D = kHeadDim / G, W = cached_row_bytes(EIGHT);
  const int lane = threadIdx.x & (G - 1);
  const size_t exponents = (size_t)p.Hkv * p.batch.page_size.d * kHeadDim;
  M = -INFINITY;
  L = 0.0f;
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = 0.0f;
  for (int u = u0; u < u1; ++u)
    for (int k0 = 0; k0 < UNIT; k0 += G) {
      const int key = keys.base(u, UNIT) + k0 + lane;
      PagePlace at = {-1, 0};
      if (key < keys.limit(u) && sees(p, pos, key)) at = page_place(p.batch, b, key);
      const bool visible = at.page >= 0;
      const int64_t page_at = visible ? (int64_t)at.page * p.batch.page_stride : 0;
      const int row = visible ? kvh * (int)p.batch.page_size.d + at.row : 0;
      float s = -INFINITY;
      if (visible) {
        const char *k_row = p.k + page_at + (size_t)row * W;
        const float scale = EIGHT ? power_of_two((uint8_t)p.k[page_at + exponents + row]) : 1.0f;
        s = 0.0f;
        for (int c = 0; c < kHeadDim; c += 8) {
          const u32x4_t qv = global_load_b128(q_row + c * 2);
          u32x4_t kv;
          if constexpr (EIGHT) {
            const u32x2_t w = *reinterpret_cast<const u32x2_t *>(k_row + c);
            kv = widen8<T>(w[0], w[1], scale);
          } else {
            kv = global_load_b128(k_row + c * 2);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            s += Elem<T>::widen((uint16_t)(qv[i >> 1] >> ((i & 1) * 16))) * Elem<T>::widen((uint16_t)(kv[i >> 1] >> ((i & 1) * 16)));
        }
        s *= kScaleLog2e;
      }
      float most = s;
      for (int x = 1; x < G; x *= 2) most = fmaxf(most, __shfl_xor(most, x, G));
      const float m_new = fmaxf(M, most), m_use = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = fast_exp2(M - m_use), weight = visible ? fast_exp2(s - m_use) : 0.0f;
      M = m_new;
      L = L * alpha + weight;
#pragma unroll
      for (int d = 0; d < D; ++d) o[d] *= alpha;
      for (int i = 0; i < G; ++i) {
        const float w = __shfl(weight, i, G);
        const int at_page = __shfl(at.page, i, G), at_row = __shfl(row, i, G);
        if (at_page < 0) continue;
        const char *v_row = p.v + (int64_t)at_page * p.batch.page_stride + (size_t)at_row * W;
        const float scale = EIGHT ? power_of_two((uint8_t)p.v[(int64_t)at_page * p.batch.page_stride + exponents + at_row]) : 1.0f;
#pragma unroll
        for (int d = 0; d < D; d += 2) {
          uint32_t pair;
          if constexpr (EIGHT)
            pair = widen_pair<T, false>(*reinterpret_cast<const uint16_t *>(v_row + D * lane + d), scale);
          else
            pair = *reinterpret_cast<const uint32_t *>(v_row + (D * lane + d) * 2);
          o[d] += w * Elem<T>::widen((uint16_t)pair);
          o[d + 1] += w * Elem<T>::widen((uint16_t)(pair >> 16));
        }
      }
    }
  for (int x = 1; x < G; x *= 2) L += __shfl_xor(L, x, G);
}

// ---- few rows ----

template <typename T, bool EIGHT> __device__ __forceinline__ void few_rows(const PagedAttn &p, int unit, char *lds) {
  using E = Elem<T>;
  constexpr int kLoads = EIGHT ? 4 : 8;  // of 1 KiB, for 32 rows
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, cg = lane >> 4;
  const int rest = (int)fast_div(unit, p.Hkv_div), kvh = unit - rest * p.Hkv;
  const int tile = (int)fast_div(rest, p.few_splits_div), split = rest - tile * p.few_splits;
  PagedTile t;
  if (!find_tile<true>(p, tile, lane, t)) return;
  const int p0 = t.len - t.m, p1 = t.len - 1;
  const PagedKeys keys = keys_seen<kFewUnit>(p, p0, p1, t.len);
  const PagedSplit part = split_of(keys.units, split, p.few_splits, p.few_chunk);
  if (split >= part.count) return;

  const bool col_valid = col < t.rows;
  const int c_tok = col_valid ? (int)fast_div(col, p.g_div) : 0, c_head = kvh * p.g + (col_valid ? col - c_tok * p.g : 0);
  const int c_pos = p0 + c_tok;
  u32x4_t qf[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) qf[kk] = u32x4_t{0u, 0u, 0u, 0u};
  if (col_valid) {
    const char *qp = p.q + ((size_t)(t.start + c_tok) * p.H + c_head) * kRowBytes + cg * 16;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[kk] = global_load_b128(qp + kk * 64);
  }

  char *vl = lds + wave * kWaveStage, *kl = lds + (4 + wave) * kWaveStage;
  u32x4_t kn[kLoads], vn[kLoads];
  int exps = 0;  // 8 bits: of K's 32 rows in the lower lanes, of V's in the upper ones
  GroupPlaces places = {-1, 0};
  const int iters = part.u1 - part.u0;
  auto piece = [&](int it) { return keys.base(part.u0 + it, kFewUnit) + 32 * wave; };
  auto look = [&](int it) {  // 32 steps, two groups each
    const int i = it + (lane >> 1), u = part.u0 + i, key = keys.base(u, kFewUnit) + 32 * wave + 16 * (lane & 1);
    places.page = -1;
    if (i < iters && key < keys.limit(u)) places.look(p, t.b, key);
  };
  auto group = [&](int it, int half) {
    return group_of(p, places, (it & 31) * 2 + half, kvh, piece(it) + 16 * half, keys.limit(part.u0 + it));
  };
  auto issue = [&](const char *pool, u32x4_t (&to)[kLoads], const Group (&g)[2]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const __amdgpu_buffer_rsrc_t r = group_buffer<EIGHT>(pool, g[half]);
#pragma unroll
      for (int i = 0; i < kLoads / 2; ++i) to[half * (kLoads / 2) + i] = stream_load(r, i * 1024 + lane * 16);
    }
  };
  auto issue_exponents = [&](const Group (&g)[2]) {
    if constexpr (EIGHT) {
      const char *pool = lane < 32 ? p.k : p.v;
      const bool second = lane & 16;
      exps = 127;
      if ((lane & 15) < (second ? g[1].have : g[0].have))
        exps = *((second ? group_exponents(p, pool, g[1]) : group_exponents(p, pool, g[0])) + (lane & 15));
    }
  };
  // Row of a piece that load i of this lane belongs to, and where its 16 bytes (or what 16 e4m3 become) go
  auto stage = [&](char *to, const u32x4_t (&from)[kLoads], int which, auto place) {
    if constexpr (EIGHT) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = 8 * i + (lane >> 3), granule = 2 * (lane & 7);
        const float scale = power_of_two(__builtin_amdgcn_ds_bpermute(4 * (row + 32 * which), exps));
        lds_write_b128(to, place(row, granule), widen8<T>(from[i][0], from[i][1], scale));
        lds_write_b128(to, place(row, granule + 1), widen8<T>(from[i][2], from[i][3], scale));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_write_b128(to, place(4 * i + cg, col), from[i]);
    }
  };

  f32x4_t o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.0f;
  Group now[2];
  if (iters > 0) {
    look(0);
    now[0] = group(0, 0);
    now[1] = group(0, 1);
    issue(p.k, kn, now);
    issue(p.v, vn, now);
    issue_exponents(now);
  }
  for (int it = 0; it < iters; ++it) {
    const int base = piece(it), limit = keys.limit(part.u0 + it);
    const bool whole = now[0].have == kPageGroup && now[1].have == kPageGroup;
    const bool any = now[0].have + now[1].have > 0;
    if (any) {
      __builtin_amdgcn_wave_barrier();
      stage(kl, kn, 0, [](int row, int granule) { return k_swizzle_off(row, granule); });
      stage(vl, vn, 1, [](int row, int granule) { return v_swizzle32_off(row, granule); });
      __builtin_amdgcn_wave_barrier();
    }
    const bool there[2] = {now[0].have > 0, now[1].have > 0};
    if (it + 1 < iters) {
      if (((it + 1) & 31) == 0) look(it + 1);
      now[0] = group(it + 1, 0);
      now[1] = group(it + 1, 1);
      issue(p.k, kn, now);
      issue(p.v, vn, now);
      issue_exponents(now);
    }
    if (!any) continue;
    f32x4_t s[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      s[blk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) s[blk] = E::mfma16(lds_read_b128(kl, k_swizzle_off(blk * 16 + col, 4 * kk + cg)), qf[kk], s[blk]);
    }
    if (!whole || base + 31 > p0 || (p.window > 0 && base <= p1 - p.window && base + 31 >= p.sinks)) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = base + blk * 16 + 4 * cg + i;
          if (!there[blk] || key >= limit || !sees(p, c_pos, key)) s[blk][i] = -INFINITY;
        }
    }
    float mloc = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mloc = quad_max(mloc);
    const float m_new = fmaxf(m_run, mloc * kScaleLog2e);
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
    if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {
      const float alpha = fast_exp2(m_run - m_use);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
      m_run = m_new;
    }
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[blk][i] = fast_exp2(__builtin_fmaf(s[blk][i], kScaleLog2e, -m_use));
    // The weights are rounded to the storage type for the matrix product; the sum takes the rounded ones, so that numerator and
    // denominator carry the same rounding.
    const u32x4_t pf = {E::pack2(s[0][0], s[0][1]), E::pack2(s[0][2], s[0][3]), E::pack2(s[1][0], s[1][1]), E::pack2(s[1][2], s[1][3])};
    l_run += dot2_ones<T>(pf[3], dot2_ones<T>(pf[2], dot2_ones<T>(pf[1], dot2_ones<T>(pf[0], 0.0f))));
    const int vr = 4 * cg + (col >> 2), sub = (col & 1) * 8;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int gran = 2 * d + ((col & 3) >> 1);
      const u32x2_t lo = lds_read_tr16(vl, v_swizzle32_off(vr, gran) + sub);
      const u32x2_t hi = lds_read_tr16(vl, v_swizzle32_off(vr + 16, gran) + sub);
      o[d] = E::mfma16(u32x4_t{lo[0], lo[1], hi[0], hi[1]}, pf, o[d]);
    }
  }

  // ---- merge the waves: [wave][col][128], the pieces of a row XORed with the column ----
  const float l_tot = quad_sum(l_run);
  __syncthreads();
  float *lo_f = reinterpret_cast<float *>(lds), *lml = reinterpret_cast<float *>(lds + 4 * kWaveStage);
#pragma unroll
  for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4_t *>(lo_f + (wave * kFewCols + col) * kHeadDim + (((4 * d + cg) ^ col) << 2)) = o[d];
  if (cg == 0) {
    lml[(wave * kFewCols + col) * 2] = m_run;
    lml[(wave * kFewCols + col) * 2 + 1] = l_tot;
  }
  __syncthreads();
  const int c = tid >> 4, dch = tid & 15;  // 16 lanes to a row, 8 dims each
  if (c >= t.rows) return;
  float M = -INFINITY, L = 0.0f, acc[8];
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, lml[(w * kFewCols + c) * 2]);
  const float M_use = M == -INFINITY ? 0.0f : M;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float wt = fast_exp2(lml[(w * kFewCols + c) * 2] - M_use);
    L += wt * lml[(w * kFewCols + c) * 2 + 1];
    const float *src = lo_f + (w * kFewCols + c) * kHeadDim;
    const f32x4_t s0 = *reinterpret_cast<const f32x4_t *>(src + (((2 * dch) ^ c) << 2)), s1 = *reinterpret_cast<const f32x4_t *>(src + (((2 * dch + 1) ^ c) << 2));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[j] += wt * s0[j];
      acc[4 + j] += wt * s1[j];
    }
  }
  const int tok = (int)fast_div(c, p.g_div);
  const size_t row_at = ((size_t)(t.start + tok) * p.H + kvh * p.g + c - tok * p.g) * kRowBytes;
  float size = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) size += __builtin_fabsf(acc[j]);
  const bool finite = size < INFINITY;
  if (__builtin_expect(((__builtin_amdgcn_ballot_w64(!finite) >> (lane & 48)) & 0xffff) != 0, 0))
    exact_row<T, EIGHT, 16, kFewUnit>(p, t.b, kvh, p.q + row_at, p0 + tok, keys, part.u0, part.u1, M, L, acc);
  if (part.count == 1) {
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);  // (NaN stays NaN)
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = E::pack2(acc[2 * j] * inv, acc[2 * j + 1] * inv);
    *reinterpret_cast<u32x4_t *>(p.out + row_at + dch * 16) = w;
    return;
  }
  const size_t slot = (((size_t)tile * p.Hkv + kvh) * p.few_splits + split) * kFewCols + c;
  float *wo = p.few_o + slot * kHeadDim + 8 * dch;
  *reinterpret_cast<f32x4_t *>(wo) = f32x4_t{acc[0], acc[1], acc[2], acc[3]};
  *reinterpret_cast<f32x4_t *>(wo + 4) = f32x4_t{acc[4], acc[5], acc[6], acc[7]};
  if (dch == 0) *reinterpret_cast<float2 *>(p.few_ml + slot * 2) = float2{M, L};
}

// ---- tiles ----

// 1 KiB from a descriptor into LDS, lane by lane.  Inline: the compiler would order every later LDS read behind the load; what it is for
// is waited for where the waves meet (s_waitcnt vmcnt before a barrier).
__device__ __forceinline__ void load_to_lds(u32x4_t r, int lane_off, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(lane_off), "s"(r), "s"(lds_at) : "m0", "memory");
}

template <typename T, bool EIGHT> __device__ __forceinline__ void tile_rows(const PagedAttn &p, int unit, char *lds) {
  using E = Elem<T>;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int rest = (int)fast_div(unit, p.Hkv_div), kvh = unit - rest * p.Hkv;
  const int tile = (int)fast_div(rest, p.tile_splits_div), split = rest - tile * p.tile_splits;
  PagedTile t;
  if (!find_tile<false>(p, tile, lane, t)) return;
  const int before = t.len - t.m;  // tokens cached before the new ones
  const int p0 = before + (int)fast_div(t.row0, p.g_div), p1 = before + (int)fast_div(t.row0 + t.rows - 1, p.g_div);
  const PagedKeys keys = keys_seen<kTileUnit>(p, p0, p1, t.len);
  const PagedSplit part = split_of(keys.units, split, p.tile_splits, p.tile_chunk);
  if (split >= part.count) return;

  // this wave's rows, and this lane's
  const int w_rows = min(t.rows - 32 * wave, 32), w_row0 = t.row0 + 32 * wave;  // (none: w_rows <= 0)
  const int w_p0 = w_rows > 0 ? before + (int)fast_div(w_row0, p.g_div) : 0;
  const int w_p1 = w_rows > 0 ? before + (int)fast_div(w_row0 + w_rows - 1, p.g_div) : -1;
  WaveAttn<T, 2> w;
  w.init(lds, lane, 2 * kUnitBytes);
  auto place_of = [&](int r, int &tok) {  // byte offset of row r of the wave's, in q and in out
    tok = (int)fast_div(w_row0 + r, p.g_div);
    return ((size_t)(t.start + tok) * p.H + kvh * p.g + w_row0 + r - tok * p.g) * kRowBytes;
  };
  int my_tok = 0;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) w.qf[kk] = u32x4_t{0u, 0u, 0u, 0u};
  if (w.l32 < w_rows) {
    const char *qp = p.q + place_of(w.l32, my_tok) + w.hh * 16;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) w.qf[kk] = global_load_b128(qp + kk * 32);
  }
  const int my_pos = before + my_tok;

  // Wave i fetches group i of every tile: 16 rows of K and of V.  Lane offsets of the four loads of 4 rows (16 bits), which
  // undo the swizzle of the LDS rows.
  const int r4 = lane >> 4, c16 = lane & 15;
  int k_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) k_off[i] = (4 * i + r4) * kRowBytes + ((c16 ^ (4 * i + r4)) << 4);
  const int v_off = r4 * kRowBytes + (((((c16 >> 2) ^ r4) << 2) | (c16 & 3)) << 4);
  const uint32_t lds_k = lds_address(lds) + wave * kPageGroup * kRowBytes, lds_v = lds_k + 2 * kUnitBytes;
  u32x4_t kn[2], vn[2];
  int exps = 0;

  const int iters = part.u1 - part.u0;
  GroupPlaces places = {-1, 0}, later = {-1, 0};
  auto look = [&](GroupPlaces &to, int it) {  // 16 tiles, four groups each
    const int i = it + (lane >> 2), u = part.u0 + i, key = keys.base(u, kTileUnit) + 16 * (lane & 3);
    to.page = -1;
    if (i < iters && key < keys.limit(u)) to.look(p, t.b, key);
  };
  auto issue = [&](int it) {
    const int u = part.u0 + it, key = keys.base(u, kTileUnit) + 16 * wave;
    const Group g = group_of(p, places, (it & 15) * 4 + wave, kvh, key, keys.limit(u));
    if constexpr (EIGHT) {
      const __amdgpu_buffer_rsrc_t kb = group_buffer<true>(p.k, g), vb = group_buffer<true>(p.v, g);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kn[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(kb, i * 1024 + lane * 16, 0, 0));
        vn[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vb, i * 1024 + lane * 16, 0, 0));
      }
      exps = 127;
      if ((lane & 15) < g.have && !(lane & 16)) exps = *(group_exponents(p, lane < 32 ? p.k : p.v, g) + (lane & 15));
    } else {
      const uint32_t slot = (it & 1) * kUnitBytes;
      const u32x4_t kb = group_words(p.k, g), vb = group_words(p.v, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) load_to_lds(kb, k_off[i], __builtin_amdgcn_readfirstlane(lds_k + slot + i * 1024));
#pragma unroll
      for (int i = 0; i < 4; ++i) load_to_lds(vb, v_off + i * 1024, __builtin_amdgcn_readfirstlane(lds_v + slot + i * 1024));
    }
  };
  auto widen = [&](int it) {  // 8 bits: what issue() fetched goes to LDS
    char *k_to = lds + (it & 1) * kUnitBytes, *v_to = k_to + 2 * kUnitBytes;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * i + (lane >> 3), row = 16 * wave + r, granule = 2 * (lane & 7);
      const float ks = power_of_two(__builtin_amdgcn_ds_bpermute(4 * r, exps)), vs = power_of_two(__builtin_amdgcn_ds_bpermute(4 * (r + 32), exps));
      lds_write_b128(k_to, k_swizzle_off(row, granule), widen8<T>(kn[i][0], kn[i][1], ks));
      lds_write_b128(k_to, k_swizzle_off(row, granule + 1), widen8<T>(kn[i][2], kn[i][3], ks));
      lds_write_b128(v_to, v_swizzle_off(row, granule), widen8<T>(vn[i][0], vn[i][1], vs));
      lds_write_b128(v_to, v_swizzle_off(row, granule + 1), widen8<T>(vn[i][2], vn[i][3], vs));
    }
  };
  if (iters > 0) {
    look(places, 0);
    issue(0);
    if (EIGHT) widen(0);
    look(later, 16);
  }
  for (int it = 0; it < iters; ++it) {
    const int u = part.u0 + it, base = keys.base(u, kTileUnit), limit = keys.limit(u);
    const uint64_t there = __builtin_amdgcn_ballot_w64(places.page >= 0) >> ((it & 15) * 4);
    // the tile is there, in all waves' groups, and the other slot is free
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (it + 1 < iters) {
      if (((it + 1) & 15) == 0) {
        places = later;
        look(later, it + 17);
      }
      issue(it + 1);
    }
    if (base <= w_p1) {
      f32x16_t s[2];
      const int slot = (it & 1) * kUnitBytes;
      w.qk(lds, slot, s);
      if (base + kTileUnit > min(w_p0 + 1, limit) || (there & 15) != 15 || (p.window > 0 && base <= w_p1 - p.window && base + kTileUnit > p.sinks)) {
        const int from = base + 4 * w.hh, last = min(my_pos, limit - 1) - from;
        const int first = p.window > 0 ? my_pos - p.window - from : -(1 << 30), sink = p.sinks - from;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int c = kb * 32 + 8 * (i >> 2) + (i & 3);
            if (c > last || (c <= first && c >= sink) || !(there >> (2 * kb + (i >> 3)) & 1)) s[kb][i] = -INFINITY;
          }
      }
      w.row_max(s, kScaleLog2e);
      w.l_run += w.probabilities(s, kScaleLog2e);
      w.pv(slot);
    }
    if (EIGHT && it + 1 < iters) widen(it + 1);
  }

  // ---- rows that are not finite, key by key ----
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  char *mine = lds + wave * 32 * kRowBytes;
  float size = 0.0f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) size += __builtin_fabsf(w.o[d][i]);
  uint64_t bad = __builtin_amdgcn_ballot_w64(!(size < INFINITY));
  for (uint32_t rows = (uint32_t)(bad | bad >> 32); __builtin_expect(rows != 0, 0); rows &= rows - 1) {
    const int r = __builtin_ctz(rows);
    if (r >= w_rows) break;
    float M, L, x[2];
    int tok;
    const char *q_row = p.q + place_of(r, tok);
    exact_row<T, EIGHT, 64, kTileUnit>(p, t.b, kvh, q_row, before + tok, keys, part.u0, part.u1, M, L, x);
    *reinterpret_cast<float2 *>(mine + lane * 8) = float2{x[0], x[1]};
    __builtin_amdgcn_wave_barrier();
    if (w.l32 == r) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) w.o[d][i] = *reinterpret_cast<const float *>(mine + (32 * d + 8 * (i >> 2) + 4 * w.hh + (i & 3)) * 4);
      w.m_run = M / kScaleLog2e;
      w.l_run = w.hh == 0 ? L : 0.0f;
    }
    __builtin_amdgcn_wave_barrier();
  }

  const float l_tot = pair_sum(w.l_run);
  if (part.count > 1) {
    if (w.l32 < w_rows) {
      const size_t slot = (((size_t)tile * p.Hkv + kvh) * p.tile_splits + split) * kTileRows + 32 * wave + w.l32;
      float *o_row = p.tile_o + slot * kHeadDim;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          *reinterpret_cast<f32x4_t *>(o_row + 32 * d + 8 * i4 + 4 * w.hh) = f32x4_t{w.o[d][4 * i4], w.o[d][4 * i4 + 1], w.o[d][4 * i4 + 2], w.o[d][4 * i4 + 3]};
      if (w.hh == 0) *reinterpret_cast<float2 *>(p.tile_ml + slot * 2) = float2{w.m_run * kScaleLog2e, l_tot};
    }
    return;
  }
  // through 8 KiB of LDS of this wave, so that whole rows leave
  const float inv = l_tot > 0.0f ? 1.0f / l_tot : (l_tot == 0.0f ? 0.0f : l_tot);  // (NaN stays NaN)
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const u32x2_t v = {E::pack2(w.o[d][4 * i4] * inv, w.o[d][4 * i4 + 1] * inv), E::pack2(w.o[d][4 * i4 + 2] * inv, w.o[d][4 * i4 + 3] * inv)};
      *reinterpret_cast<u32x2_t *>(mine + k_swizzle_off(w.l32, 4 * d + i4) + w.hh * 8) = v;
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + r4;
    int tok;
    if (r < w_rows) store_device_b128(p.out + place_of(r, tok) + c16 * 16, lds_read_b128(mine, k_swizzle_off(r, c16)));
  }
}

enum PagedMode { kFewRows, kTiles, kBoth };

template <typename T, bool EIGHT, PagedMode MODE> __global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedAttn p) {
  __shared__ __attribute__((aligned(16))) char lds[kPagedLds];
  const int unit = blockIdx.x;
  if (MODE == kFewRows || (MODE == kBoth && unit < p.few_blocks))
    few_rows<T, EIGHT>(p, unit, lds);
  else
    tile_rows<T, EIGHT>(p, unit - (MODE == kBoth ? p.few_blocks : 0), lds);
}

// Partials of a (tile, kv head), 16 rows to a workgroup, 16 lanes to a row.
template <typename T> __global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttn p) {
  const int tid = threadIdx.x, lane = tid & 63, dch = tid & 15;
  const bool few = (int)blockIdx.x < p.few_blocks;
  int unit = few ? blockIdx.x : blockIdx.x - p.few_blocks;
  const int rows0 = few ? 0 : (unit & 7) * 16;
  if (!few) unit >>= 3;
  const int tile = (int)fast_div(unit, p.Hkv_div), kvh = unit - tile * p.Hkv;
  PagedTile t;
  if (!(few ? find_tile<true>(p, tile, lane, t) : find_tile<false>(p, tile, lane, t))) return;
  const int before = t.len - t.m, p0 = before + (int)fast_div(t.row0, p.g_div), p1 = before + (int)fast_div(t.row0 + t.rows - 1, p.g_div);
  const int units = few ? keys_seen<kFewUnit>(p, p0, p1, t.len).units : keys_seen<kTileUnit>(p, p0, p1, t.len).units;
  const int splits = few ? p.few_splits : p.tile_splits, count = split_of(units, 0, splits, few ? p.few_chunk : p.tile_chunk).count;
  const int c = rows0 + (tid >> 4), slot_rows = few ? kFewCols : kTileRows;
  if (count == 1 || c >= t.rows) return;
  const size_t slot = ((size_t)tile * p.Hkv + kvh) * splits * slot_rows + c;
  const float *po = (few ? p.few_o : p.tile_o) + slot * kHeadDim + 8 * dch, *pml = (few ? p.few_ml : p.tile_ml) + slot * 2;
  float M = -INFINITY, L = 0.0f, acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
  for (int s = 0; s < count; ++s) M = fmaxf(M, pml[(size_t)s * slot_rows * 2]);
  const float M_use = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
  for (int s = 0; s < count; ++s) {
    const float2 ml = *reinterpret_cast<const float2 *>(pml + (size_t)s * slot_rows * 2);
    const float *row = po + (size_t)s * slot_rows * kHeadDim;
    const f32x4_t a = *reinterpret_cast<const f32x4_t *>(row), b = *reinterpret_cast<const f32x4_t *>(row + 4);
    const float wt = fast_exp2(ml.x - M_use);
    L += wt * ml.y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[j] += wt * a[j];
      acc[4 + j] += wt * b[j];
    }
  }
  const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
  const int tok = (int)fast_div(t.row0 + c, p.g_div);
  u32x4_t w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = Elem<T>::pack2(acc[2 * j] * inv, acc[2 * j + 1] * inv);
  *reinterpret_cast<u32x4_t *>(p.out + ((size_t)(t.start + tok) * p.H + kvh * p.g + t.row0 + c - tok * p.g) * kRowBytes + dch * 16) = w;
}

// How a launch is cut, from what the host knows: bounds, not lengths.
struct PagedPlan {
  bool few, tiles;
  long long few_tiles, row_tiles;
  int few_splits, few_chunk, tile_splits, tile_chunk;
  size_t few_slots() const { return few && few_splits > 1 ? (size_t)few_tiles * few_splits * kFewCols : 0; }
  size_t tile_slots() const { return tiles && tile_splits > 1 ? (size_t)row_tiles * tile_splits * kTileRows : 0; }
  size_t bytes(int Hkv) const { return (few_slots() + tile_slots()) * Hkv * (kHeadDim + 2) * sizeof(float); }
};
static PagedPlan plan_paged(int tokens, int batch, int max_q_len, int max_kv_len, int window, int sinks, int g, int Hkv) {
  PagedPlan pl = {};
  const long long cus = device_compute_units(), most_rows = (long long)max_q_len * g;
  const long long sequences = batch < tokens ? batch : tokens;  // that have new tokens at all
  pl.tiles = most_rows > kFewCols;
  // all sequences have max_q_len tokens, or the tokens do not add up
  pl.few = !pl.tiles || (g <= kFewCols && (long long)batch * max_q_len != tokens);
  pl.few_tiles = sequences;
  pl.row_tiles = (long long)tokens * g / kTileRows + sequences;
  auto cut = [&](long long wgs, int unit, long long seen, long long target, int least, int &splits, int &chunk) {
    const long long units = (seen + unit - 1) / unit;
    long long s = (target + wgs - 1) / wgs;
    if (s > (units + least - 1) / least) s = (units + least - 1) / least;
    s = s < 1 ? 1 : s > 64 ? 64 : s;
    chunk = units > s ? (int)((units + s - 1) / s) : 1;
    splits = (int)((units + chunk - 1) / chunk);
    if (splits < 1) splits = 1;
  };
  auto seen = [&](long long rows_span) {
    const long long most = (long long)window + rows_span + sinks + 2 * kPageGroup;
    return window > 0 && most < max_kv_len ? most : (long long)max_kv_len;
  };
  if (pl.few) cut(pl.few_tiles * Hkv, kFewUnit, seen(kFewCols), 4 * cus, 4, pl.few_splits, pl.few_chunk);
  if (pl.tiles) cut(pl.row_tiles * Hkv, kTileUnit, seen(kTileRows / g + 1), 2 * cus, 8, pl.tile_splits, pl.tile_chunk);
  return pl;
}

size_t paged_attn_workspace_bytes(int tokens, int batch, int max_q_len, int max_kv_len, int window, int sinks, int g, int Hkv) {
  return plan_paged(tokens, batch, max_q_len, max_kv_len, window, sinks, g, Hkv).bytes(Hkv);
}

hipError_t launch_paged_attn(void *out, const void *q, const void *k_pages, const void *v_pages, const PagedBatch &batch, void *workspace,
                             int max_q_len, int max_kv_len, int window, int sinks, int g, int Hkv, bool eight, int dt, hipStream_t stream) {
  const PagedPlan pl = plan_paged(batch.tokens, batch.batch, max_q_len, max_kv_len, window, sinks, g, Hkv);
  PagedAttn p = {};
  p.batch = batch;
  p.out = static_cast<char *>(out);
  p.q = static_cast<const char *>(q);
  p.k = static_cast<const char *>(k_pages);
  p.v = static_cast<const char *>(v_pages);
  p.H = g * Hkv;
  p.Hkv = Hkv;
  p.g = g;
  p.g_div = make_fast_div(g);
  p.Hkv_div = make_fast_div(Hkv);
  p.few_splits = pl.few ? pl.few_splits : 1;
  p.few_chunk = pl.few_chunk;
  p.tile_splits = pl.tiles ? pl.tile_splits : 1;
  p.tile_chunk = pl.tile_chunk;
  p.few_splits_div = make_fast_div(p.few_splits);
  p.tile_splits_div = make_fast_div(p.tile_splits);
  p.window = window;
  p.sinks = sinks;
  p.max_q_len = max_q_len;
  p.few_rows = pl.few ? kFewCols : 0;
  float *ws = static_cast<float *>(workspace);
  const size_t few_slots = pl.few_slots() * Hkv, tile_slots = pl.tile_slots() * Hkv;
  p.few_o = ws;
  p.tile_o = p.few_o + few_slots * kHeadDim;
  p.few_ml = p.tile_o + tile_slots * kHeadDim;
  p.tile_ml = p.few_ml + few_slots * 2;
  const long long few_blocks = pl.few ? pl.few_tiles * Hkv * p.few_splits : 0, tile_blocks = pl.tiles ? pl.row_tiles * Hkv * p.tile_splits : 0;
  if (few_blocks + tile_blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  p.few_blocks = (int)few_blocks;
  auto kernel_of = [&](auto mode) {
    constexpr PagedMode MODE = decltype(mode)::value;
    if (dt == kDtFloat16) return eight ? paged_attn_kernel<_Float16, true, MODE> : paged_attn_kernel<_Float16, false, MODE>;
    return eight ? paged_attn_kernel<__bf16, true, MODE> : paged_attn_kernel<__bf16, false, MODE>;
  };
  const auto kern = !pl.tiles ? kernel_of(std::integral_constant<PagedMode, kFewRows>())
                    : !pl.few ? kernel_of(std::integral_constant<PagedMode, kTiles>())
                              : kernel_of(std::integral_constant<PagedMode, kBoth>());
  hipError_t e = launch(kern, dim3((uint32_t)(few_blocks + tile_blocks)), 256, 0, stream, p);
  if (e != hipSuccess) return e;
  const long long few_folds = pl.few_slots() ? pl.few_tiles * Hkv : 0, tile_folds = pl.tile_slots() ? pl.row_tiles * Hkv * (kTileRows / 16) : 0;
  if (few_folds + tile_folds == 0) return hipSuccess;
  if (few_folds + tile_folds > 0x7fffffffLL) return hipErrorInvalidValue;
  p.few_blocks = (int)few_folds;
  return launch(dt == kDtFloat16 ? paged_combine_kernel<_Float16> : paged_combine_kernel<__bf16>, dim3((uint32_t)(few_folds + tile_folds)), 256, 0,
                stream, p);
}

}  // namespace llmhip
