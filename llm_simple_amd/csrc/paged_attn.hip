// Attention of new tokens over a cache in pages, gfx950: a batch of sequences of their own lengths, each with one new token or many, over
// all keys up to a token or over a sliding window of them and the first `sinks` keys.
//
//   out[t][h] = sum_c softmax_c(q[t][h] . K[c][h / g] / sqrt(128)) V[c][h / g],   c <= p, and c > p - window or c < sinks
//
// with p the position of token t (paged.hpp).  Query rows of a kv head are (token, head of its g) pairs, token-major, so that K and V of
// a kv head are read for all g heads at once.  Two kinds of workgroups, of four waves:
//
//  * few rows: a sequence with at most 16 rows.  A stream of K and V through the chip: the rows are the 16 columns of mfma 16x16x32, a wave
//    takes every fourth piece of 32 keys and keeps its own running maximum, sum and O; the four are merged at the end.  V goes through LDS
//    of the wave's own and is read transposed.
//  * tiles: 128 rows, 32 to a wave (wave_attn.hpp), over tiles of 64 keys in LDS, two of them, so that a tile is on its way while
//    the one before it is worked on.  Wide ones have 256 rows and eight waves (plan_paged).
//
// 8-bit rows become rows of the storage type before the matrix instructions: each is widened once by a workgroup, for all rows that use
// it, by a conversion that takes the row's power of two along, and everything after is the same code.
//
// What a workgroup is for is found on the device (lengths may change between replays of a graph), see find_work: a wave looks at 64 sequences
// at a time.  Where the keys that a tile's rows see are dealt to several workgroups, each leaves an fp32 partial.  Few rows' are folded by
// the workgroup that finds all of them stored, tiles' by a second launch, which has the whole chip for them.  A unit of keys is 128 (few rows)
// or 64.
//
// Few rows are bound by the memory system: 16 sequences of 32768 keys of 8 kv heads, 8 bits, 1.08 GB in 171 us, 6.3 TB/s (16 bits 2.15 GB, 326 us,
// 6.6); a short cache by its chain of memory round trips (starts and lengths, page table, K and V; 384 keys of 2 kv heads 6.4 us, of which an
// empty launch is 1.6).  Tiles are bound, as the prefill kernels are, by matrix and vector instructions that share a SIMD and the chip's power:
// a step of two workgroups to a CU takes 2.0-2.2 us, 1.0 PFLOP/s; 4 us of a workgroup's time are its start.  (us, on the
// faster and on the slower of two cards: a prompt of 4096 tokens of 28 + 4 heads 131 / 141, 0.85-0.92 PFLOP/s, in 8 bits 129 / 137; 200 past 16001 60 / 64;
// 8192 with a window of 1024 147 / 155.  Figures below are pairs of one card each.)
//
// More scalars are alive than there are scalar registers, and some are kept in lanes of vector registers: none that a loop over keys asks for, but
// for the runs in 8 bits, six of the 450 instructions of two steps.
//
// Keys that a row must not see: their scores become -inf, so their K does not matter, but a weight of 0 times a V that is not finite
// would be NaN.  Rows behind the last key, and pages that are not there, are zeros (the loads' descriptors end before them).  V of keys
// that only some rows see is what it is: a wave that finds a row of its own not finite in the end goes over its keys once more
// (rows_again), and adds up those 32 of which a row must not see one key by key, from what each row sees.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "paged.hpp"
#include "paged_plan.hpp"
#include "wave_attn.hpp"

namespace llmhip {

constexpr int kUnitBytes = kTileUnit * kRowBytes;
constexpr int kWaveStage = 32 * kRowBytes;  // staging of a few-rows wave, for K and for V
constexpr int kFewLds = 8 * kWaveStage, kTilesLds = 4 * kUnitBytes;

// One kind of work of a launch
struct PagedKind {
  float *o, *ml;     // partials [slot][kv head][row][128], and [2]: maximum (times scale and log2 e), sum
  char *flags;       // [slot][kv head], see few_rows_of
  int slots;         // room for so many; 0: nothing is split
  int tiles;         // so many at most, or the grid is too small for them
  int least;         // units that a part has at least
  int parts;         // workgroups of a kv head that run at a time
};
struct PagedAttn {
  PagedBatch batch;
  char *out;
  const char *q, *k, *v;
  PagedKind few, tiles;
  int H, Hkv, g;
  FastDiv g_div, Hkv_div;
  int window, sinks;  // window 0: none
  int max_q_len;
  int few_rows;    // sequences of up to so many rows are few-rows ones; 0: none is
  int tile_shift;  // a tile has 2^this rows
  int few_blocks;  // workgroups of few rows, the first ones in a launch of both
  int fold_shift;  // 2^this times 8 rows to a workgroup that folds
  uint64_t number;  // of the launch
};
// What the first loads of a workgroup need, in its registers when it starts (common.hpp).
// a: starts, lengths, page table, q; b: sequences, tokens, max_q_len, few_rows; c: keys_max, heads of a group
struct PagedEarly {
  addresses_t a;
  u32x4_t b;
  u32x2_t c;
  explicit PagedEarly(const PagedAttn &p) {
    a = addresses_t{address(p.batch.q_starts), address(p.batch.kv_lens), address(p.batch.page_table), address(p.q)};
    b = u32x4_t{(uint32_t)p.batch.batch, (uint32_t)p.batch.tokens, (uint32_t)p.max_q_len, (uint32_t)p.few_rows};
    c = u32x2_t{(uint32_t)p.batch.keys_max, (uint32_t)p.g};
  }
};
__device__ __forceinline__ void take_early(PagedAttn &p, addresses_t a, u32x4_t b, u32x2_t c) {
  p.batch.q_starts = at_address<const int>(a[0]);
  p.batch.kv_lens = at_address<const int>(a[1]);
  p.batch.page_table = at_address<const int>(a[2]);
  p.q = at_address<const char>(a[3]);
  p.batch.batch = b[0];
  p.batch.tokens = b[1];
  p.max_q_len = b[2];
  p.few_rows = b[3];
  p.batch.keys_max = c[0];
  p.g = c[1];
}

// The keys that rows at positions p0 .. p1 see, in units of UNIT keys: the first `sink_units` of them are keys 0 .. sink_end, the rest
// begin at key `first`, a multiple of 16, and end at `end`.
struct PagedKeys {
  int sink_units, sink_end, first, end, units;
  __device__ __forceinline__ int base(int unit, int size) const { return unit < sink_units ? unit * size : first + (unit - sink_units) * size; }
  // (as a sum: as a choice the compiler keeps the two in memory and loads one)
  __device__ __forceinline__ int limit(int unit) const { return end - (int)(unit < sink_units) * (end - sink_end); }
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

// Inclusive sum over the lanes of a wave
template <typename X> __device__ __forceinline__ X wave_prefix(X x) {
  auto from = [&](auto control, auto rows) {
    const int v = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(control)::value, decltype(rows)::value, 0xf, false);
    x += __builtin_bit_cast(X, v);
  };
  using std::integral_constant;
  from(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // row_shr:1
  from(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  from(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  from(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  from(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // row_bcast:15, into rows 1 and 3
  from(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());  // row_bcast:31, into rows 2 and 3
  return x;
}

// What a workgroup works on: `rows` rows from row `row0` of a sequence on, and of the keys that they see part `split` of `splits`.  slot: of
// the first part's partial.
struct PagedTile {
  int b, start, m, len, row0, rows, split, splits, slot;
  int u0 = 0, u1 = -1;  // a run's part: these units (else u1 < 0, see part_of)
};

// The sequences of one kind, 64 at a time, a lane each.
template <bool FEW> struct PagedSeqs {
  int start, m, len, tiles, units;  // units: of the last tile, which sees most
  PagedSeqs() = default;
  __device__ __forceinline__ PagedSeqs(const PagedAttn &p, int base, int lane) {
    const int i = min(base + lane, p.batch.batch - 1), end = p.batch.q_starts[i + 1];
    start = p.batch.q_starts[i];
    len = p.batch.kv_lens[i];
    const bool valid = base + lane < p.batch.batch && sequence_ok(p.batch, start, end, len) && end - start <= p.max_q_len;
    m = valid ? end - start : 0;
    const int rows = m * p.g;
    tiles = FEW ? (m > 0 && rows <= p.few_rows ? 1 : 0) : rows <= p.few_rows ? 0 : (rows + (1 << p.tile_shift) - 1) >> p.tile_shift;
    const int first = FEW ? 0 : (int)fast_div(max(tiles - 1, 0) << p.tile_shift, p.g_div);
    units = tiles ? keys_seen<FEW ? kFewUnit : kTileUnit>(p, len - m + first, len - 1, len).units : 0;
  }
};

// Dealing keys to workgroups.  A sequence's tiles are split into as many parts as it has chunks of units; the chunk is the least for which
// all parts of all tiles (each counted like its sequence's last) run at a time, or an equal share of all units where there are too many
// tiles for that.  That is at most a part to a tile more than run at a time, and a sequence in parts has at least half a chunk to a
// part: at most twice as many partials.  Whoever needs it works it out by itself, with the same instructions, so all agree; a
// sequence whose partials find no room is not split.
//
// Few rows: a workgroup to a CU, in parts of 3 units or more (us, one / two to a CU: 5 x 2999 keys of 8 kv heads in 8 bits 15.6 / 17.2, 48 ragged
// sequences with a window of 4096 61 / 76; parts of 2: 384 keys of 2 kv heads 8.6 -> 9.4, 5 x 2999 16.8 -> 16.4).  Tiles: two to a CU, 6 units or
// more (4: 16 prompts of 300 36.6 -> 43; 12: 64 past 4000 of 40 + 8 heads in 8 bits 26.2 -> 32.8; three to a CU beside few rows: 101 -> 116).
//
// FOLD: the tile of number w among those that are split.  Else: the part of number w of all; a sequence's last tiles first.
__device__ __forceinline__ int parts_of(int units, float chunk) {
  return max((int)__builtin_ceilf((float)units * __builtin_amdgcn_rcpf(chunk) * (1.0f - 0x1p-20f)), 1);  // (a whole number stays one)
}
template <typename X> __device__ __forceinline__ X wave_sum(X x) {
  return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_prefix(x)), 63));
}
// One sequence by itself: the same in scalar registers, a third of the instructions (us, 384 keys of 2 kv heads 7.2 -> 6.8, a prompt of 8192 with a
// window 155 -> 152; a prompt of 1000 of 40 + 8 heads, whose tiles are half of what runs at a time and are not split, 48 -> 34).
template <bool FEW, bool FOLD> __device__ __forceinline__ bool find_alone(const PagedAttn &p, int w, PagedTile &t) {
  const PagedKind &kind = FEW ? p.few : p.tiles;
  const int start = p.batch.q_starts[0], end = p.batch.q_starts[1], len = p.batch.kv_lens[0];
  if (!sequence_ok(p.batch, start, end, len) || end <= start || end - start > p.max_q_len) return false;
  const int m = end - start, rows = m * p.g;
  if (FEW != (rows <= p.few_rows)) return false;
  const int tiles = FEW ? 1 : (rows + (1 << p.tile_shift) - 1) >> p.tile_shift, first = FEW ? 0 : (int)fast_div((tiles - 1) << p.tile_shift, p.g_div);
  int splits = 1;
  if (kind.slots && tiles <= kind.parts / 2) {
    const int units = keys_seen<FEW ? kFewUnit : kTileUnit>(p, len - m + first, len - 1, len).units;
    splits = max(min(kind.parts / tiles, units / kind.least), 1);
    if (splits > 1 && tiles * splits > kind.slots) splits = 1;
  }
  if (FOLD && splits == 1) return false;
  const int tile = FOLD || splits == 1 ? w : w / splits;
  if (tile >= tiles) return false;
  t = PagedTile{0, start, m, len, FEW ? 0 : (tiles - 1 - tile) << p.tile_shift, 0, FOLD ? 0 : w - tile * splits, splits, tile * splits};
  if (!FOLD && splits == 1) t.split = 0;
  t.rows = min(rows - t.row0, FEW ? kFewCols : 1 << p.tile_shift);
  return true;
}
// Where sequences' lengths leave the greatest chunk well above an equal share, or more parts than run at a time, few-rows workgroups
// take runs of the units of all sequences one after the other, equal to a unit; a run may end one sequence and begin another, and then
// costs the start of another.  (us, parts / runs: 48 sequences of up to 16384 keys of 4 kv heads, 48 units to a run, 16 bits 167 / 145, 8 bits 107 /
// 85; 24 of up to 8192 of 8, 24 units, 76.7 / 72.2 and 52.4 / 51.4; with a window of 4096, 20 units, 61.2 / 67.0; 64 of up to 2048 of 2, 4 units,
// 19.9 / 23.2.)  A kernel of its own, for bounds that allow runs: the loop over sequences costs a call of 7 us 0.6.
struct FewRuns {
  PagedSeqs<true> s;
  int units, upto, slot;  // of a lane's sequence: units, those up to its end, its first partial's slot
  int total, runs, w, at, end;
  __device__ __forceinline__ int run_of(int unit) const { return (int)(((uint32_t)(unit + 1) * (uint32_t)runs - 1) / (uint32_t)total); }
  // False: they are not to be taken in runs.
  __device__ __forceinline__ bool begin(const PagedAttn &p, int run, int lane) {
    units = s.tiles ? max(s.units, 1) : 0;
    upto = wave_prefix(units);
    total = __builtin_amdgcn_readlane(upto, 63);
    if (total > 1 << 22) return false;  // (32-bit products)
    runs = max(min(p.few.parts, total / p.few.least), 1);
    const int partials = units ? run_of(upto - 1) - run_of(upto - units) + 1 : 0, kept = partials > 1 ? partials : 0, slots_upto = wave_prefix(kept);
    slot = slots_upto - kept;
    if (__builtin_amdgcn_readlane(slots_upto, 63) > p.few.slots) return false;
    w = run;
    at = (int)((uint32_t)w * (uint32_t)total / (uint32_t)runs);
    end = w < runs ? (int)((uint32_t)(w + 1) * (uint32_t)total / (uint32_t)runs) : at;
    return true;
  }
  // The next sequence of the run
  __device__ __forceinline__ bool next(const PagedAttn &p, PagedTile &t) {
    if (at >= end) return false;
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > at));
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
    const int last = of(upto), first = last - of(units), run0 = run_of(first);
    t = PagedTile{l, of(s.start), of(s.m), of(s.len), 0, 0, w - run0, run_of(last - 1) - run0 + 1, of(slot), at - first, min(end, last) - first};
    t.rows = min(t.m * p.g, kFewCols);
    at = last;
    return true;
  }
};
// runs: few rows, where it is taken (`in_runs` then says so, and t is not set).
template <bool FEW, bool FOLD>
__device__ __forceinline__ bool find_work(const PagedAttn &p, int w, int lane, PagedTile &t, FewRuns *runs = nullptr, bool *in_runs = nullptr) {
  if (p.batch.batch == 1) return find_alone<FEW, FOLD>(p, w, t);
  const PagedKind &kind = FEW ? p.few : p.tiles;
  PagedSeqs<FEW> s(p, 0, lane);
  float chunk = 0.0f;
  bool split = false;
  if (kind.slots) {
    float units = 0.0f;
    int tiles = 0;
    for (int base = 0;;) {
      units += wave_sum((float)s.tiles * (float)s.units);
      tiles += wave_sum(s.tiles);
      if ((base += 64) >= p.batch.batch) break;
      s = PagedSeqs<FEW>(p, base, lane);
    }
    const float least = (float)kind.least;
    chunk = fmaxf(units * __builtin_amdgcn_rcpf((float)kind.parts), least);
    // (More tiles: sequences overlap, which is not allowed.  A part that no workgroup takes would leave the others' flags up.)
    split = tiles <= kind.tiles;
    if (p.batch.batch <= 64) {
      [[maybe_unused]] bool even = false;
      for (int fit = kind.parts, tries = 0; tries < 6 && 2 * fit > kind.parts && tiles <= kind.parts; ++tries) {
        const float tried = fmaxf(units * __builtin_amdgcn_rcpf((float)fit), least);
        const int over = wave_sum(s.tiles * parts_of(s.units, tried)) - kind.parts;
        if (over <= 0) {
          chunk = tried;
          even = chunk * (float)kind.parts <= 1.2f * units;
          break;
        }
        fit -= over;
      }
      if constexpr (FEW) {
        if (runs && !even && units >= (float)(kRunUnits * kind.parts)) {
          runs->s = s;
          if (runs->begin(p, w, lane)) {
            *in_runs = true;
            return true;
          }
        }
      }
    } else {
      s = PagedSeqs<FEW>(p, 0, lane);
    }
  }
  int slot = 0;
  for (int base = 0; base < p.batch.batch; base += 64) {
    if (base > 0) s = PagedSeqs<FEW>(p, base, lane);
    int splits = split ? parts_of(s.units, chunk) : 1;
    const int partials = splits > 1 ? s.tiles * splits : 0;
    const int slots_upto = slot + wave_prefix(partials);
    if (slots_upto > kind.slots) splits = 1;
    const int mine = FOLD ? (splits > 1 ? s.tiles : 0) : s.tiles * splits;
    const int upto = wave_prefix(mine), all = __builtin_amdgcn_readlane(upto, 63);
    if (w >= all) {
      w -= all;
      slot = __builtin_amdgcn_readlane(slots_upto, 63);
      continue;
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > w));
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
    const int at = w - (of(upto) - of(mine));
    t.b = base + l;
    t.start = of(s.start);
    t.m = of(s.m);
    t.len = of(s.len);
    t.splits = of(splits);
    const int tile = FOLD || t.splits == 1 ? at : at / t.splits;
    t.split = FOLD ? 0 : at - tile * t.splits;
    t.slot = of(slots_upto) - of(partials) + tile * t.splits;
    t.row0 = FEW ? 0 : (of(s.tiles) - 1 - tile) << p.tile_shift;
    t.rows = min(t.m * p.g - t.row0, FEW ? kFewCols : 1 << p.tile_shift);
    return true;
  }
  return false;
}

// Units u0 .. u1 of a part
struct PagedPart {
  int u0, u1;
};
__device__ __forceinline__ PagedPart part_of(const PagedTile &t, int units) {
  if (t.u1 >= 0) return PagedPart{min(t.u0, units), min(t.u1, units)};
  if (t.splits == 1) return PagedPart{0, units};
  const int each = (units + t.splits - 1) / t.splits, u0 = min(t.split * each, units);
  return PagedPart{u0, min(u0 + each, units)};
}

// 64 groups of 16 keys of a kv head, one to a lane: as the table has them, nothing waits for that load before places() ...
constexpr int kHaveShift = 27;  // rest: row among the page's rows of all kv heads (at most 65535 * 1024), and behind it how many of the 16 are there
struct GroupLook {
  int page;
  uint32_t rest;
};
__device__ __forceinline__ GroupLook group_look(const PagedAttn &p, int b, int kvh, int key, int limit) {
  GroupLook l = {-1, 0};
  const int have = min(max(limit - key, 0), kPageGroup);
  if (have > 0) {
    const PagePlace at = page_place(p.batch, b, key);
    l.page = at.page;
    l.rest = (uint32_t)(kvh * (int)p.batch.page_size.d + at.row) | (uint32_t)have << kHaveShift;
  }
  return l;
}
// ... and as bytes from the pool's base on
struct GroupPlaces {
  uint32_t lo, hi, rest;
};
struct Group {  // one of them
  uint64_t at;
  uint32_t rest;
  __device__ __forceinline__ int have() const { return rest >> kHaveShift; }
  __device__ __forceinline__ uint32_t row() const { return rest & ((1u << kHaveShift) - 1); }
};
template <bool EIGHT> __device__ __forceinline__ GroupPlaces group_places(const PagedAttn &p, const GroupLook &l) {
  const bool there = (uint32_t)l.page < (uint32_t)p.batch.num_pages;
  const uint32_t row = l.rest & ((1u << kHaveShift) - 1);
  const uint64_t at = there ? (uint64_t)((int64_t)l.page * p.batch.page_stride) + (uint64_t)row * cached_row_bytes(EIGHT) : 0;
  return GroupPlaces{(uint32_t)at, (uint32_t)(at >> 32), there ? l.rest : 0u};
}
__device__ __forceinline__ Group group_at(const GroupPlaces &places, int lane) {
  return Group{(uint64_t)(uint32_t)__builtin_amdgcn_readlane(places.hi, lane) << 32 | (uint32_t)__builtin_amdgcn_readlane(places.lo, lane),
               (uint32_t)__builtin_amdgcn_readlane(places.rest, lane)};
}
template <bool EIGHT> __device__ __forceinline__ __amdgpu_buffer_rsrc_t group_buffer(const char *pool, const Group &g) {
  return byte_buffer(pool + g.at, g.have() * cached_row_bytes(EIGHT));
}
// The same descriptor of a 16-bit group as words, for assembly (in scalar registers, whatever the compiler makes of it)
__device__ __forceinline__ u32x4_t group_words(const char *pool, const Group &g) {
  const uint64_t at = reinterpret_cast<uintptr_t>(pool) + g.at;
  auto scalar = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); };
  return u32x4_t{scalar((uint32_t)at), scalar((uint32_t)(at >> 32) & 0xffffu), scalar(g.have() * kRowBytes), 0x00020000u};
}
// Address of the exponent byte of a group's first row: behind the page's values, of which 128 bytes are before it for each byte of these
__device__ __forceinline__ const uint8_t *group_exponents(const PagedAttn &p, const char *pool, const Group &g) {
  return reinterpret_cast<const uint8_t *>(pool + g.at - (uint64_t)g.row() * (kHeadDim - 1) + (uint64_t)((uint32_t)p.Hkv * p.batch.page_size.d) * kHeadDim);
}

__device__ __forceinline__ bool sees(const PagedAttn &p, int pos, int key) {
  return key <= pos && (p.window <= 0 || key > pos - p.window || key < p.sinks);
}

// The lane, and the kernels' arguments, of which the compiler has computed or loaded nothing before: code that hardly runs keeps nothing in
// registers elsewhere.
__device__ __forceinline__ int fresh_lane() {
  int none = 0;
  asm volatile("" : "+v"(none));
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (uint32_t)none));
}
struct PagedArguments {  // as the kernels have them
  addresses_t a;
  u32x4_t b;
  u32x2_t c;
  PagedAttn p;
};
static_assert(__builtin_offsetof(PagedArguments, p) == sizeof(addresses_t) + sizeof(u32x4_t) + sizeof(u32x2_t));
__device__ __forceinline__ PagedAttn fresh_arguments() {
  typedef __attribute__((address_space(4))) const PagedArguments Constant;
  uint64_t at = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  PagedAttn p;
  __builtin_memcpy(&p, (const void *)&((Constant *)at)->p, sizeof(p));
  return p;
}

// The 32 rows of a wave (w.qf, at positions pos) over keys first .. first + 31 of every `step` of the part's units, once more and by the wave alone; see
// the header.  32 keys at a time, K and then V through `mine`, 8 KiB of the wave's own.  Where a row must not see one of the keys that are there,
// the product goes key by key, a key's V for the rows that see it.  The reference of the weights is the running maximum itself: a sum that only
// its slack made too large for 32 bits is none here.
//
// Nothing of this is on the way of rows that are finite, and no row, nor any number of such V, makes a call more than some times longer (us of 28 + 4
// heads, without / with a NaN in one dim of the first key / row by row and key by key as the only way: a prompt of 1024 31 / 90 / 3700, of 4096 152 / 740 /
// 30000, 200 past 16001 67 / 290 / 12400, 3 past 2000 17 / 51 / 1900).
template <typename T, bool EIGHT, int UNIT>
__device__ __forceinline__ void rows_again(int b, int kvh, WaveAttn<T, 1> &w, int pos, const PagedKeys &keys, int u0, int u1,
                                           int first, int step, char *mine) {
  constexpr int W = cached_row_bytes(EIGHT), kLoads = EIGHT ? 4 : 8;  // bytes of a row; loads of a lane, which has half of one
  const PagedAttn p = fresh_arguments();
  int lane = fresh_lane(), r = lane >> 1, half = lane & 1;
  const size_t exponents = (size_t)p.Hkv * p.batch.page_size.d * kHeadDim;
  w.init(mine, lane, 0);
  f32x16_t s[1];
  auto stage = [&](const u32x4_t (&x)[kLoads], int byte, auto place) {
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
      if constexpr (EIGHT) {
        const float scale = power_of_two(byte);
        lds_write_b128(mine, place(r, 8 * half + 2 * c), widen8<T>(x[c][0], x[c][1], scale));
        lds_write_b128(mine, place(r, 8 * half + 2 * c + 1), widen8<T>(x[c][2], x[c][3], scale));
      } else {
        lds_write_b128(mine, place(r, 8 * half + c), x[c]);
      }
    }
  };
#pragma unroll 1
  for (int u = u0; u < u1; ++u)
#pragma unroll 1
    for (int k0 = first; k0 < UNIT; k0 += step) {
      asm volatile("" : "+v"(r), "+v"(half));  // (the places in LDS worked out anew: registers)
      const int base = keys.base(u, UNIT) + k0, limit = keys.limit(u);
      PagePlace at = {-1, 0};
      if (base + r < limit) at = page_place(p.batch, b, base + r);
      const bool there = at.there(p.batch);
      const uint64_t rows_there = __builtin_amdgcn_ballot_w64(there);
      if (rows_there == 0) continue;
      const int64_t page_at = there ? (int64_t)at.page * p.batch.page_stride : 0;
      const uint32_t row = (uint32_t)(kvh * (int)p.batch.page_size.d + at.row);
      auto fetch = [&](const char *pool, u32x4_t (&x)[kLoads], int &byte) {
        byte = 127;
#pragma unroll
        for (int c = 0; c < kLoads; ++c) x[c] = u32x4_t{};
        if (!there) return;
        const char *page = pool + page_at;
#pragma unroll
        for (int c = 0; c < kLoads; ++c) x[c] = global_load_b128(page + (size_t)row * W + half * (W / 2) + c * 16);
        if constexpr (EIGHT) byte = (uint8_t)page[exponents + row];
      };
      u32x4_t x[kLoads];
      int byte;
      fetch(p.k, x, byte);
      __builtin_amdgcn_wave_barrier();
      stage(x, byte, [](int row, int granule) { return k_swizzle_off(row, granule); });
      __builtin_amdgcn_wave_barrier();
      fetch(p.v, x, byte);
      w.qk(mine, 0, s);
      __builtin_amdgcn_wave_barrier();
      stage(x, byte, [](int row, int granule) { return v_swizzle_off(row, granule); });
      __builtin_amdgcn_wave_barrier();
      const uint64_t mine_there = rows_there >> (8 * w.hh);
      bool some_hidden = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = 8 * (i >> 2) + (i & 3);
        const bool is_there = mine_there >> (2 * c) & 1, seen = sees(p, pos, base + 4 * w.hh + c);
        some_hidden |= is_there && !seen;
        s[0][i] = is_there && seen ? s[0][i] : -INFINITY;
      }
      w.template row_max<false>(s, kScaleLog2e);
      w.l_run += w.probabilities(s, kScaleLog2e);
      if (__builtin_amdgcn_ballot_w64(some_hidden) == 0) {
        w.pv(0);
        continue;
      }
#pragma unroll 1
      for (int key = 0; key < 32; ++key) {
        const int i = 4 * (key >> 3) + (key & 3);  // element of the half key >> 2 & 1 of the lanes
        uint32_t pair = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) pair = j == i >> 1 ? w.pf[0][j >> 2][j & 3] : pair;
        pair = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (w.l32 + 8 * (key & 4)), (int)pair);
        const float weight = Elem<T>::widen((uint16_t)(i & 1 ? pair >> 16 : pair));
        const bool seen = sees(p, pos, base + key);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const u32x2_t x = *reinterpret_cast<const u32x2_t *>(mine + v_swizzle_off(key, 4 * d + i4) + w.hh * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float o = w.o[d][4 * i4 + j];
              const float more = __builtin_fmaf(weight, Elem<T>::widen((uint16_t)(x[j >> 1] >> ((j & 1) * 16))), o);
              w.o[d][4 * i4 + j] = seen ? more : o;
            }
          }
      }
    }
}

// ---- few rows ----

template <typename T, bool EIGHT> __device__ __forceinline__ void few_rows_of(const PagedAttn &p, const PagedTile &t, int kvh, char *lds) {
  using E = Elem<T>;
  constexpr int kLoads = EIGHT ? 4 : 8;  // of 1 KiB, for 32 rows
  constexpr int W = cached_row_bytes(EIGHT);
  // 16 bits: K through LDS like V, whole 1 KiB pieces to a load, one step on its way (us, loaded as the operand has it, 64 bytes of 16
  // rows / this: 48 ragged sequences with a window 72 / 61, without 185 / 167; 16 x 32768 keys 315 / 327).  8 bits: as the operand has it, and two
  // steps on their way, as many bytes (16 x 32768, through LDS 175 / 169, one step 190; 48 ragged 120 / 107).
  constexpr bool kStaged = !EIGHT;
  constexpr int kAhead = EIGHT ? 2 : 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = fresh_lane(), tid = wave * 64 + lane, col = lane & 15, cg = lane >> 4;
  const int p0 = t.len - t.m, p1 = t.len - 1;
  const PagedKeys keys = keys_seen<kFewUnit>(p, p0, p1, t.len);
  const PagedPart part = part_of(t, keys.units);

  const int iters = part.u1 - part.u0;
  auto piece = [&](int it) { return keys.base(part.u0 + it, kFewUnit) + 32 * wave; };
  auto look = [&](int it) {  // 32 steps, two groups each
    const int i = it + (lane >> 1), u = part.u0 + i;
    return group_look(p, t.b, kvh, keys.base(u, kFewUnit) + 32 * wave + 16 * (lane & 1), i < iters ? keys.limit(u) : 0);
  };
  GroupLook later = look(0);  // (before Q: loads come back in order)

  // Columns past the rows have the last row once more.  (Without a branch: the compiler would not know how many loads came after the page
  // table's, and wait for Q where it needs that one only.)
  const int c_row = min(col, t.rows - 1), c_tok = (int)fast_div(c_row, p.g_div), c_pos = p0 + c_tok;
  u32x4_t qf[4];
  {
    // Dims of a lane's fragment kk: 32 kk + 8 cg .. + 7; in 8 bits, where its 16 bytes of K are 16 dims, 64 (kk / 2) + 16 cg + 8 (kk % 2)
    const char *qp = p.q + ((size_t)(t.start + c_tok) * p.H + kvh * p.g + c_row - c_tok * p.g) * kRowBytes + cg * (kStaged ? 16 : 32);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[kk] = global_load_b128(qp + (kStaged ? 64 * kk : 128 * (kk >> 1) + 16 * (kk & 1)));
  }

  char *vl = lds + wave * kWaveStage, *kl = lds + (4 + wave) * kWaveStage;
  GroupPlaces places = {0, 0, 0};
  auto group = [&](int it, int half) { return group_at(places, (it & 31) * 2 + half); };
  // A step's 32 keys on their way: two steps are
  struct Step {
    Group g[2];
    u32x4_t k[kLoads], v[kLoads];
    uint8_t k_exps[2], v_exps[2];  // 8 bits: bytes of rows col (K) and lane % 16 (V) of either group
  };
  // (Steps past the last find no groups: loads of nothing.  No branch round the loads, and K's before V's, so that the compiler can count
  // them, and waits for a step's alone.)
  auto fetch = [&](Step &s, int it) {
    if ((it & 31) == 0 && it > 0) {
      places = group_places<EIGHT>(p, later);
      later = look(it + 32);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      s.g[half] = group_at(places, (it & 31) * 2 + half);
      const __amdgpu_buffer_rsrc_t r = group_buffer<EIGHT>(p.k, s.g[half]);
#pragma unroll
      for (int i = 0; i < kLoads / 2; ++i) s.k[half * (kLoads / 2) + i] = stream_load(r, kStaged ? i * 1024 + lane * 16 : col * W + cg * 16 + i * 64);
      if constexpr (EIGHT) s.k_exps[half] = __builtin_amdgcn_raw_buffer_load_b8(byte_buffer(group_exponents(p, p.k, s.g[half]), s.g[half].have()), col, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const __amdgpu_buffer_rsrc_t r = group_buffer<EIGHT>(p.v, s.g[half]);
#pragma unroll
      for (int i = 0; i < kLoads / 2; ++i) s.v[half * (kLoads / 2) + i] = stream_load(r, i * 1024 + lane * 16);
      if constexpr (EIGHT) s.v_exps[half] = __builtin_amdgcn_raw_buffer_load_b8(byte_buffer(group_exponents(p, p.v, s.g[half]), s.g[half].have()), col, 0, 0);
    }
  };
  f32x4_t o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.0f;
  auto stage = [&](const u32x4_t (&from)[kLoads], const uint8_t (&exps)[2], char *to, auto place) {
    if constexpr (EIGHT) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = 8 * i + (lane >> 3), granule = 2 * (lane & 7);
        const float scale = power_of_two(__builtin_amdgcn_ds_bpermute(4 * (row & 15), exps[i >> 1]));
        lds_write_b128(to, place(row, granule), widen8<T>(from[i][0], from[i][1], scale));
        lds_write_b128(to, place(row, granule + 1), widen8<T>(from[i][2], from[i][3], scale));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_write_b128(to, place(4 * i + cg, col), from[i]);
    }
  };
  auto step = [&](Step &in, int it) {
    const int base = piece(it), limit = keys.limit(part.u0 + it);
    const bool whole = in.g[0].have() == kPageGroup && in.g[1].have() == kPageGroup;
    const bool there[2] = {in.g[0].have() > 0, in.g[1].have() > 0};
    if constexpr (kStaged) {
      __builtin_amdgcn_wave_barrier();
      stage(in.k, in.k_exps, kl, [](int row, int granule) { return k_swizzle_off(row, granule); });
      __builtin_amdgcn_wave_barrier();
    }
    // ---- S^T = K Q^T ----
    f32x4_t s[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      s[blk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        if constexpr (kStaged) {
          s[blk] = E::mfma16(lds_read_b128(kl, k_swizzle_off(blk * 16 + col, 4 * kk + cg)), qf[kk], s[blk]);
        } else if constexpr (EIGHT) {
          const u32x4_t from = in.k[2 * blk + (kk >> 1)];
          s[blk] = E::mfma16(widen8<T>(from[2 * (kk & 1)], from[2 * (kk & 1) + 1], power_of_two(in.k_exps[blk])), qf[kk], s[blk]);
        } else {
          s[blk] = E::mfma16(in.k[4 * blk + kk], qf[kk], s[blk]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    stage(in.v, in.v_exps, vl, [](int row, int granule) { return v_swizzle32_off(row, granule); });
    __builtin_amdgcn_wave_barrier();
    fetch(in, it + kAhead);
    if (!there[0] && !there[1]) return;
    if (!whole || base + 31 > p0 || (p.window > 0 && base <= p1 - p.window && base + 31 >= p.sinks)) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = base + blk * 16 + 4 * cg + i;
          const bool hidden = (int)!there[blk] | (int)(key >= limit) | (int)(key > c_pos) |
                              ((int)(p.window > 0) & (int)(key <= c_pos - p.window) & (int)(key >= p.sinks));
          s[blk][i] = hidden ? -INFINITY : s[blk][i];
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
    // ---- O^T += V^T P^T ----
    const int vr = 4 * cg + (col >> 2), sub = (col & 1) * 8;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int gran = 2 * d + ((col & 3) >> 1);
      const u32x2_t lo = lds_read_tr16(vl, v_swizzle32_off(vr, gran) + sub);
      const u32x2_t hi = lds_read_tr16(vl, v_swizzle32_off(vr + 16, gran) + sub);
      o[d] = E::mfma16(u32x4_t{lo[0], lo[1], hi[0], hi[1]}, pf, o[d]);
    }
  };
  if (iters > 0) {
    places = group_places<EIGHT>(p, later);
    later = look(32);
    Step a = {}, b = {};
    fetch(a, 0);
    if (kAhead > 1) {
      __builtin_amdgcn_sched_barrier(0);
      fetch(b, 1);
    }
    int it = 0;
    for (; it + kAhead <= iters; it += kAhead) {
      step(a, it);
      if (kAhead > 1) step(b, it + 1);
    }
    if (kAhead > 1 && it < iters) step(a, it);
  }
  // Rows that are not finite, where some see keys that others do not
  if (t.m > 1 || p.window > 0) {
    float size = 0.0f;
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) size += __builtin_fabsf(o[d][i]);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(size < INFINITY)) != 0, 0)) {
      WaveAttn<T, 1> w;
      const int l = fresh_lane(), row = min(l & 31, t.rows - 1), tok = (int)fast_div(row, p.g_div);
      const char *qp = p.q + ((size_t)(t.start + tok) * p.H + kvh * p.g + row - tok * p.g) * kRowBytes + (l >> 5) * 16;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) w.qf[kk] = global_load_b128(qp + kk * 32);
      rows_again<T, EIGHT, kFewUnit>(t.b, kvh, w, p0 + tok, keys, part.u0, part.u1, 32 * wave, kFewUnit, vl);
      // from its columns to those here, through LDS as below
      float *rows = reinterpret_cast<float *>(vl);
      __builtin_amdgcn_wave_barrier();
      if (w.l32 < kFewCols) {
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            *reinterpret_cast<f32x4_t *>(rows + w.l32 * kHeadDim + (((8 * d + 2 * i4 + w.hh) ^ w.l32) << 2)) =
                f32x4_t{w.o[d][4 * i4], w.o[d][4 * i4 + 1], w.o[d][4 * i4 + 2], w.o[d][4 * i4 + 3]};
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] = *reinterpret_cast<const f32x4_t *>(rows + (l & 15) * kHeadDim + (((4 * d + (l >> 4)) ^ (l & 15)) << 2));
      m_run = __shfl(w.m_run * kScaleLog2e, l & 15, 64);
      l_run = __shfl(pair_sum(w.l_run), l & 15, 64);
      if (l >> 4 != 0) l_run = 0.0f;
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
  float M = -INFINITY, L = 0.0f, acc[8];
  const int tok = (int)fast_div(c, p.g_div);
  const size_t row_at = ((size_t)(t.start + tok) * p.H + kvh * p.g + c - tok * p.g) * kRowBytes;
  auto store_row = [&] {
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);  // (NaN stays NaN)
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = E::pack2(acc[2 * j] * inv, acc[2 * j + 1] * inv);
    *reinterpret_cast<u32x4_t *>(p.out + row_at + dch * 16) = w;
  };
  const int bytes = p.few.slots * p.Hkv * kFewCols;
  const __amdgpu_buffer_rsrc_t po = byte_buffer(p.few.o, bytes * kHeadDim * 4), pml = byte_buffer(p.few.ml, bytes * 8);
  auto slot_row = [&](int part_) { return ((t.slot + part_) * p.Hkv + kvh) * kFewCols + c; };
  if (c < t.rows) {
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
    if (t.splits == 1) {
      store_row();
    } else {
      store_device(po, slot_row(t.split) * 512 + dch * 32, f32x4_t{acc[0], acc[1], acc[2], acc[3]});
      store_device(po, slot_row(t.split) * 512 + dch * 32 + 16, f32x4_t{acc[4], acc[5], acc[6], acc[7]});
      if (dch == 0) store_device(pml, slot_row(t.split) * 8, u32x2_t{__builtin_bit_cast(uint32_t, M), __builtin_bit_cast(uint32_t, L)});
    }
  }
  if (t.splits == 1) return;
  // The partials are folded by the workgroup that finds all of them stored.  Each raises its flag once its partial is where all XCDs see it,
  // and looks at the others' after that: the last one to raise its flag finds all of them up (if two do, both write the same rows).  A
  // flag is up if it holds the launch's number, whatever the workspace held before; who folds takes them down for a replay.  Nobody waits
  // for another.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  unsigned *all_up = reinterpret_cast<unsigned *>(lds);
  const __amdgpu_buffer_rsrc_t pf = byte_buffer(p.few.flags, p.few.slots * p.Hkv * kFlagBytes);
  auto flag_at = [&](int part_) { return ((t.slot + part_) * p.Hkv + kvh) * kFlagBytes; };
  if (wave == 0) {
    const u32x2_t up = {(uint32_t)p.number, (uint32_t)(p.number >> 32)};
    if (lane == 0) store_device(pf, flag_at(t.split), up);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool down = false;
    for (int i = lane; i < t.splits; i += 64) {
      const u32x2_t f = load_device2(pf, flag_at(i));
      down |= f[0] != up[0] || f[1] != up[1];
    }
    const bool all = __builtin_amdgcn_ballot_w64(down) == 0;
    if (lane == 0) *all_up = all;
  }
  __syncthreads();
  if (*all_up == 0) return;
  for (int i = tid; i < t.splits; i += 256) store_device(pf, flag_at(i), u32x2_t{0u, 0u});
  if (c >= t.rows) return;
  M = -INFINITY;
  L = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
  constexpr int D = 8;  // on their way at a time
  for (int s0 = 0; s0 < t.splits; s0 += D) {
    u32x2_t ml[D];
    f32x4_t x[D], y[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int at = slot_row(min(s0 + j, t.splits - 1));
      ml[j] = load_device2(pml, at * 8);
      x[j] = load_device(po, at * 512 + dch * 32);
      y[j] = load_device(po, at * 512 + dch * 32 + 16);
    }
    float most = M;
#pragma unroll
    for (int j = 0; j < D; ++j) most = fmaxf(most, __builtin_bit_cast(float, (uint32_t)ml[j][0]));
    const float m_use = most == -INFINITY ? 0.0f : most, before = fast_exp2(M - m_use);
    M = most;
    L *= before;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= before;
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (s0 + j >= t.splits) continue;
      const float wt = fast_exp2(__builtin_bit_cast(float, (uint32_t)ml[j][0]) - m_use);
      L += wt * __builtin_bit_cast(float, (uint32_t)ml[j][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i] += wt * x[j][i];
        acc[4 + i] += wt * y[j][i];
      }
    }
  }
  store_row();
}

template <typename T, bool EIGHT, bool RUNS> __device__ __forceinline__ void few_rows(const PagedAttn &p, int unit, char *lds) {
  const int lane = threadIdx.x & 63, item = (int)fast_div(unit, p.Hkv_div), kvh = unit - item * p.Hkv;
  PagedTile t;
  if constexpr (RUNS) {
    FewRuns runs;
    bool in_runs = false;
    if (!find_work<true, false>(p, item, lane, t, &runs, &in_runs) || (in_runs && !runs.next(p, t))) return;
    for (;;) {
      few_rows_of<T, EIGHT>(p, t, kvh, lds);
      if (!in_runs || !runs.next(p, t)) return;
      __syncthreads();  // (the merge still reads what the next one stages in)
    }
  } else {
    if (find_work<true, false>(p, item, lane, t)) few_rows_of<T, EIGHT>(p, t, kvh, lds);
  }
}
// ---- tiles ----

// N (4 or 2) times 4 rows of a group into LDS, 1 KiB each, lane by lane: the instruction's offset moves both addresses.  Inline: the compiler would
// order every later LDS read behind the loads; they are waited for where the waves meet (s_waitcnt vmcnt before a barrier).
template <int N> __device__ __forceinline__ void load_group(u32x4_t r, const int (&o)[N], uint32_t lds_at) {
  if constexpr (N == 2)
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds\n\tbuffer_load_dwordx4 %1, %2, 0 offen offset:0x400 lds"
                 :
                 : "v"(o[0]), "v"(o[1]), "s"(r), "s"(lds_at)
                 : "m0", "memory");
  else
    asm volatile(
        "s_mov_b32 m0, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %4, 0 offen lds\n\tbuffer_load_dwordx4 %1, %4, 0 offen offset:0x400 lds\n\t"
        "buffer_load_dwordx4 %2, %4, 0 offen offset:0x800 lds\n\tbuffer_load_dwordx4 %3, %4, 0 offen offset:0xc00 lds"
        :
        : "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3]), "s"(r), "s"(lds_at)
        : "m0", "memory");
}

// The loop is that of the prefill kernels: K runs one tile ahead of V, so that the matrix instructions of S(j + 1) = K(j + 1) Q^T stand
// beside the softmax of tile j, and those of P(j) V(j) beside the exponentials.  In a step, K(j + 2) goes where K(j) was and V(j + 1) where
// V(j - 1) was, both read in the step before.
template <typename T, bool EIGHT, int WAVES> __device__ __forceinline__ void tile_rows(const PagedAttn &p, int unit, char *lds) {
  using E = Elem<T>;
  constexpr int kVRegion = 2 * kUnitBytes;
  constexpr int kPieces = 16 / WAVES, kPieces8 = 8 / WAVES;  // loads of a wave for K or V of a tile, in 16 and in 8 bits
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int item = (int)fast_div(unit, p.Hkv_div), kvh = unit - item * p.Hkv;
  PagedTile t;
  if (!find_work<false, false>(p, item, lane, t)) return;
  const int before = t.len - t.m;  // tokens cached before the new ones
  const int p0 = before + (int)fast_div(t.row0, p.g_div), p1 = before + (int)fast_div(t.row0 + t.rows - 1, p.g_div);
  const PagedKeys keys = keys_seen<kTileUnit>(p, p0, p1, t.len);
  const PagedPart part = part_of(t, keys.units);

  const int iters = part.u1 - part.u0;
  auto look = [&](int it) {  // 16 tiles, four groups each
    const int i = it + (lane >> 2), u = part.u0 + i;
    return group_look(p, t.b, kvh, keys.base(u, kTileUnit) + 16 * (lane & 3), i < iters ? keys.limit(u) : 0);
  };
  GroupLook later = look(0);  // (before Q: loads come back in order)

  // this wave's rows, and this lane's
  const int w_rows = min(t.rows - 32 * wave, 32), w_row0 = t.row0 + 32 * wave;  // (none: w_rows <= 0)
  const int w_p0 = w_rows > 0 ? before + (int)fast_div(w_row0, p.g_div) : 0;
  const int w_p1 = w_rows > 0 ? before + (int)fast_div(w_row0 + w_rows - 1, p.g_div) : -1;
  WaveAttn<T, 2> w;
  w.init(lds, lane, kVRegion);
  auto place_of = [&](int r, int &tok) {  // byte offset of row r of the wave's, in q and in out
    tok = (int)fast_div(w_row0 + r, p.g_div);
    return ((size_t)(t.start + tok) * p.H + kvh * p.g + w_row0 + r - tok * p.g) * kRowBytes;
  };
  int my_tok;
  {
    // (rows past the last are that one once more; without a branch, as in few_rows)
    const char *qp = p.q + place_of(min(w.l32, t.rows - 1 - 32 * wave), my_tok) + w.hh * 16;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) w.qf[kk] = global_load_b128(qp + kk * 32);
  }
  const int my_pos = before + my_tok;

  // A wave fetches a group of every tile, 16 rows of K and of V, or with 8 waves half of one.  Lane offsets within 4 rows (16 bits), which
  // undo the swizzle of the LDS rows.
  const int group = wave * 4 / WAVES, part_row = wave * 64 / WAVES - 16 * group;
  const int r4 = lane >> 4, c16 = lane & 15;
  int k_off[kPieces], v_off[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    k_off[i] = (part_row + r4) * kRowBytes + ((c16 ^ (part_row + 4 * i + r4)) << 4);
    v_off[i] = (part_row + r4) * kRowBytes + (((((c16 >> 2) ^ r4) << 2) | (c16 & 3)) << 4);
  }
  const uint32_t lds_k = __builtin_amdgcn_readfirstlane(lds_address(lds) + (16 * group + part_row) * kRowBytes), lds_v = lds_k + kVRegion;
  u32x4_t kn[kPieces8], vn[kPieces8];  // 8 bits: what is on its way to slots of K and V
  int exps = 0;

  GroupPlaces places = {0, 0, 0};
  // Where this wave's group of tile `it` is, and which groups of the tile are there at all
  struct Next {
    Group g;
    uint32_t there;
  };
  auto next_of = [&](int it) {
    if ((it & 15) == 0) {
      places = group_places<EIGHT>(p, later);
      later = look(it + 16);
    }
    Next n;
    n.g = group_at(places, (it & 15) * 4 + group);
    n.there = (uint32_t)(__builtin_amdgcn_ballot_w64(places.rest != 0) >> ((it & 15) * 4)) & 15u;
    return n;
  };
  auto issue_k = [&](const Group &g, int slot) {
    if constexpr (EIGHT) {
      const __amdgpu_buffer_rsrc_t r = group_buffer<true>(p.k, g);
#pragma unroll
      for (int i = 0; i < kPieces8; ++i)
        kn[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, part_row * kHeadDim + i * 1024 + lane * 16, 0, 0));
    } else {
      load_group<kPieces>(group_words(p.k, g), k_off, lds_k + slot * kUnitBytes);
    }
  };
  auto issue_v = [&](const Group &g, int slot) {
    if constexpr (EIGHT) {
      const __amdgpu_buffer_rsrc_t r = group_buffer<true>(p.v, g);
#pragma unroll
      for (int i = 0; i < kPieces8; ++i)
        vn[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, part_row * kHeadDim + i * 1024 + lane * 16, 0, 0));
    } else {
      load_group<kPieces>(group_words(p.v, g), v_off, lds_v + slot * kUnitBytes);
    }
  };
  auto issue_exponents = [&](const Group &gk, const Group &gv) {  // of K's rows in lanes 0 .. 15, of V's in lanes 32 .. 47
    if constexpr (EIGHT) {
      const bool upper = lane & 32;
      exps = 127;
      if ((lane & 31) < (upper ? gv.have() : gk.have())) exps = *((upper ? group_exponents(p, p.v, gv) : group_exponents(p, p.k, gk)) + (lane & 31));
    }
  };
  auto widen = [&](const u32x4_t (&from)[kPieces8], int lane0, char *to, auto place) {
#pragma unroll
    for (int i = 0; i < kPieces8; ++i) {
      const int r = part_row + 8 * i + (lane >> 3), row = 16 * group + r, granule = 2 * (lane & 7);
      const float scale = power_of_two(__builtin_amdgcn_ds_bpermute(4 * (r + lane0), exps));
      lds_write_b128(to, place(row, granule), widen8<T>(from[i][0], from[i][1], scale));
      lds_write_b128(to, place(row, granule + 1), widen8<T>(from[i][2], from[i][3], scale));
    }
  };
  auto widen_k = [&](int slot) {
    if constexpr (EIGHT) widen(kn, 0, lds + slot * kUnitBytes, [](int row, int granule) { return k_swizzle_off(row, granule); });
  };
  auto widen_v = [&](int slot) {
    if constexpr (EIGHT) widen(vn, 32, lds + kVRegion + slot * kUnitBytes, [](int row, int granule) { return v_swizzle_off(row, granule); });
  };

  // tiles in which this wave's rows see a key
  const int w_keys = w_p1 + 1;
  const int w_units = w_keys > keys.first ? keys.sink_units + (w_keys - keys.first + kTileUnit - 1) / kTileUnit : (max(w_keys, 0) + kTileUnit - 1) / kTileUnit;
  const int w_iters = max(0, min(iters, w_units - part.u0));
  // tiles from clear0 to clear1 are seen whole by all of this wave's rows, as far as they are there
  const int clear0 = (p.window > 0 ? keys.sink_units + max(((w_p1 - p.window - keys.first) >> 6) + 1, 0) : 0) - part.u0;
  const int clear1 = keys.sink_units + max((min(w_p0 + 1, keys.end) - keys.first) >> 6, 0) - part.u0;
  static_assert(kTileUnit == 64);
  f32x16_t sa[2], sb[2];
  Next cur = {}, nxt = {}, after = {};  // of tiles j, j + 1 and j + 2
  float scale = kScaleLog2e;
  asm volatile("" : "+s"(scale));
  if (iters > 0) {
    cur = next_of(0);
    nxt = next_of(1);
    after = next_of(2);
    issue_k(cur.g, 0);
    issue_v(cur.g, 0);
    issue_exponents(cur.g, cur.g);
    widen_k(0);
    widen_v(0);
    issue_k(nxt.g, 1);
    issue_exponents(nxt.g, cur.g);
    widen_k(1);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (w_iters > 0) w.qk(lds, 0, sa);
    // K(2) goes where tile 0 was just read: no wave may issue it before all have
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  auto step = [&](int it, auto slot_, f32x16_t (&s)[2], f32x16_t (&s_next)[2]) {
    constexpr int slot = decltype(slot_)::value;
    issue_k(after.g, slot);
    issue_v(nxt.g, slot ^ 1);
    issue_exponents(after.g, nxt.g);
    if (it < w_iters) {
      if (it < clear0 || it >= clear1 || cur.there != 15) {
        const int u = part.u0 + it, base = keys.base(u, kTileUnit), limit = keys.limit(u);
        const int from = base + 4 * w.hh;
        // a lane's keys are 8 * (i / 4) + i % 4 of 32 from its first one on
        auto hide = [&](auto hidden) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = hidden(kb * 32 + 8 * (i >> 2) + (i & 3), 2 * kb + (i >> 3)) ? -INFINITY : s[kb][i];
        };
        const int last = min(my_pos, limit - 1) - from;
        hide([&](int c, int) { return c > last; });
        if (p.window > 0) {
          const int first = my_pos - p.window - from, sink = p.sinks - from;
          hide([&](int c, int) { return (int)(c <= first) & (int)(c >= sink); });
        }
        if (cur.there != 15) hide([&](int, int group) { return !(cur.there >> group & 1); });
      }
      // (the last tile's S(j + 1) is not used: a branch would part these matrix instructions from what they stand beside)
      constexpr int next = (slot ^ 1) * kUnitBytes;
      w.template qk<0, 3>(lds, next, s_next);
      w.row_max(s, scale);
      w.template qk<3, 8>(lds, next, s_next);
      if constexpr (EIGHT) {
        w.l_run += w.probabilities_and_pv(s, scale, slot * kUnitBytes);
      } else {
        w.l_run += w.probabilities(s, scale);
        w.pv(slot * kUnitBytes);
      }
    }
    widen_k(slot);
    widen_v(slot ^ 1);
    cur = nxt;
    nxt = after;
    after = next_of(it + 3);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  // (The compiler knows nothing of the waits above, and would wait for Q, and with it for the tiles on their way, in the loop.  Here, where
  // there are no tiles too: it would do so on their account.)
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) asm volatile("" : "+v"(w.qf[kk]));
  for (int it = 0; it < iters; it += 2) {
    step(it, std::integral_constant<int, 0>(), sa, sb);
    if (it + 1 < iters) step(it + 1, std::integral_constant<int, 1>(), sb, sa);
  }

  // ---- rows that are not finite, once more ----
  char *mine = lds + wave * 32 * kRowBytes;
  float size = 0.0f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) size += __builtin_fabsf(w.o[d][i]);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(size < INFINITY)) != 0 && w_rows > 0, 0)) {
    WaveAttn<T, 1> again;
    const int l = fresh_lane();
    int tok;
    const char *qp = p.q + place_of(min(l & 31, w_rows - 1), tok) + (l >> 5) * 16;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) again.qf[kk] = global_load_b128(qp + kk * 32);
    rows_again<T, EIGHT, kTileUnit>(t.b, kvh, again, before + tok, keys, part.u0, part.u1, 0, 32, mine);
#pragma unroll
    for (int d = 0; d < 4; ++d) w.o[d] = again.o[d];
    w.m_run = again.m_run;
    w.l_run = again.l_run;
    __builtin_amdgcn_wave_barrier();
  }

  const float l_tot = pair_sum(w.l_run);
  if (t.splits > 1) {
    const size_t slot0 = (((size_t)(t.slot + t.split) * p.Hkv + kvh) << p.tile_shift) + 32 * wave;
    if (w.l32 < w_rows && w.hh == 0) *reinterpret_cast<float2 *>(p.tiles.ml + (slot0 + w.l32) * 2) = float2{w.m_run * kScaleLog2e, l_tot};
    if constexpr (EIGHT) {
      // straight from the accumulators: the registers of this kernel are full (a prompt of 4096 of 28 heads, us: 150, 158 with the way below)
      if (w.l32 < w_rows) {
        float *o_row = p.tiles.o + (slot0 + w.l32) * kHeadDim;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            *reinterpret_cast<f32x4_t *>(o_row + 32 * d + 8 * i4 + 4 * w.hh) = f32x4_t{w.o[d][4 * i4], w.o[d][4 * i4 + 1], w.o[d][4 * i4 + 2], w.o[d][4 * i4 + 3]};
      }
      return;
    }
    // through 8 KiB of LDS of this wave, half of the dims at a time, so that whole 256-byte pieces leave, past the L2 (us, from the
    // accumulators / this: 200 tokens past 16001 of 28 + 4 heads 68.1 / 65.3, 20 past 30000 37.8 / 35.8)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const f32x16_t &o = w.o[2 * half + d];
          const f32x4_t v = {o[4 * i4], o[4 * i4 + 1], o[4 * i4 + 2], o[4 * i4 + 3]};
          lds_write_b128(mine, k_swizzle_off(w.l32, 8 * d + 2 * i4 + w.hh), __builtin_bit_cast(u32x4_t, v));
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + r4;
        if (r < w_rows) store_device_b128(p.tiles.o + (slot0 + r) * kHeadDim + 64 * half + c16 * 4, lds_read_b128(mine, k_swizzle_off(r, c16)));
      }
      __builtin_amdgcn_wave_barrier();
    }
    return;
  }
  // so that whole rows leave
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

template <typename T, bool EIGHT, PagedMode MODE> __global__ __launch_bounds__(threads_of(MODE), 2) void paged_attn_kernel(addresses_t a, u32x4_t b, u32x2_t c, PagedAttn p) {
  take_early(p, a, b, c);
  __shared__ __attribute__((aligned(16))) char lds[MODE == kFewRows || MODE == kFewRuns ? kFewLds : kTilesLds];
  const int unit = blockIdx.x;
  if (MODE == kFewRows || MODE == kFewRuns || (MODE == kBoth && unit < p.few_blocks))
    few_rows<T, EIGHT, MODE == kFewRuns>(p, unit, lds);
  else
    tile_rows<T, EIGHT, threads_of(MODE) / 64>(p, unit - (MODE == kBoth ? p.few_blocks : 0), lds);
}

template <typename T> __device__ __forceinline__ void fold_row(const PagedAttn &p, const PagedTile &t, int kvh, int c, int d4) {
  const size_t row = (((size_t)t.slot * p.Hkv + kvh) << p.tile_shift) + c, step = (size_t)p.Hkv << p.tile_shift;
  const float *po = p.tiles.o + row * kHeadDim + d4, *pml = p.tiles.ml + row * 2;
  float M = -INFINITY, L = 0.0f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int D = 8;
  for (int s0 = 0; s0 < t.splits; s0 += D) {
    float2 ml[D];
    f32x4_t o[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const size_t at = min(s0 + j, t.splits - 1) * step;
      ml[j] = *reinterpret_cast<const float2 *>(pml + at * 2);
      o[j] = *reinterpret_cast<const f32x4_t *>(po + at * kHeadDim);
    }
    float most = M;
#pragma unroll
    for (int j = 0; j < D; ++j) most = fmaxf(most, ml[j].x);
    const float m_use = most == -INFINITY ? 0.0f : most, before = fast_exp2(M - m_use);
    M = most;
    L *= before;
    acc *= before;
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const float wt = s0 + j < t.splits ? fast_exp2(ml[j].x - m_use) : 0.0f;
      if (s0 + j < t.splits) {
        L += wt * ml[j].y;
        acc += wt * o[j];
      }
    }
  }
  const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);  // (NaN stays NaN)
  const int tok = (int)fast_div(t.row0 + c, p.g_div);
  const u32x2_t w = {Elem<T>::pack2(acc[0] * inv, acc[1] * inv), Elem<T>::pack2(acc[2] * inv, acc[3] * inv)};
  *reinterpret_cast<u32x2_t *>(p.out + ((size_t)(t.start + tok) * p.H + kvh * p.g + t.row0 + c - tok * p.g) * kRowBytes + d4 * 2) = w;
}
// Partials of a tile of a kv head, 8 rows to a workgroup, or 16 or 32 one after the other, 32 lanes of 4 dims to a row; 8 partials are on
// their way at a time.  The more tiles the host counts with, the fewer are split, and a workgroup that finds nothing to fold costs its
// start (us, 8 rows / 16 / 32, tiles of a kv head by the parts that run at a time: a prompt of 4096, 1.8, 143.0 / 141.4 / 140.4; six of up to 1019
// of 32 kv heads, 2.7, 68.1 / 65.4 / 64.2; six of up to 700 past up to 2000, 1.2, 100.2 / 97.2 / 99.0; 4 x 400 past 3000, 0.7, 97.0 / 94.4 / 93.9;
// 200 past 16001, 0.1, 65.2 / 65.7 / 67.9; 100 past 4000, 0.05, 22.6 / 23.6 / 27.4).
template <typename T> __global__ __launch_bounds__(256) void paged_combine_kernel(addresses_t a, u32x4_t b, u32x2_t c_, PagedAttn p) {
  take_early(p, a, b, c_);
  const int tid = threadIdx.x, lane = tid & 63, d4 = (tid & 31) * 4;
  const int eights = (int)(blockIdx.x << p.fold_shift), unit = eights >> (p.tile_shift - 3), item = (int)fast_div(unit, p.Hkv_div), kvh = unit - item * p.Hkv;
  PagedTile t;
  if (!find_work<false, true>(p, item, lane, t)) return;
  const int c0 = (eights * 8) & ((1 << p.tile_shift) - 1), c1 = min(c0 + (8 << p.fold_shift), t.rows);
  for (int c = c0 + (tid >> 5); c < c1; c += 8) fold_row<T>(p, t, kvh, c, d4);
}

size_t paged_attn_workspace_bytes(int tokens, int batch, int max_q_len, int max_kv_len, int window, int sinks, int g, int Hkv) {
  const auto bytes = [&](bool eight) { return plan_paged(tokens, batch, max_q_len, max_kv_len, window, sinks, g, Hkv, eight).bytes(Hkv); };
  return bytes(false) > bytes(true) ? bytes(false) : bytes(true);
}

hipError_t launch_paged_attn(void *out, const void *q, const void *k_pages, const void *v_pages, const PagedBatch &batch, void *workspace,
                             int max_q_len, int max_kv_len, int window, int sinks, int g, int Hkv, bool eight, int dt, hipStream_t stream) {
  const PagedPlan pl = plan_paged(batch.tokens, batch.batch, max_q_len, max_kv_len, window, sinks, g, Hkv, eight);
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
  p.window = window;
  p.sinks = sinks;
  p.max_q_len = max_q_len;
  p.few_rows = pl.few.tiles ? kFewCols : 0;
  float *ws = static_cast<float *>(workspace);
  auto kind_of = [&](const PagedPlan::Kind &k) {
    float *const ml = ws + (size_t)k.slots * Hkv * k.rows * kHeadDim;
    const PagedKind kind = {ws, ml, reinterpret_cast<char *>(ml + (size_t)k.slots * Hkv * k.rows * 2), (int)k.slots, (int)k.tiles, k.least, k.parts};
    if (k.slots) ws += k.bytes(Hkv) / sizeof(float);
    return kind;
  };
  p.few = kind_of(pl.few);
  p.tiles = kind_of(pl.by_tiles);
  const long long few_blocks = pl.few.items * Hkv, tile_blocks = pl.by_tiles.items * Hkv;
  p.fold_shift = pl.by_tiles.tiles > 2 * pl.by_tiles.parts ? 2 : 2 * pl.by_tiles.tiles > pl.by_tiles.parts ? 1 : 0;
  p.tile_shift = pl.wide ? 8 : 7;
  static_assert(kTileRows == 128);
  const long long folds = pl.by_tiles.folds() * Hkv * (1 << (p.tile_shift - 3 - p.fold_shift));
  const long long threads = threads_of(pl.mode());
  // (a launch takes fewer than 2^32 threads along a dimension)
  if ((few_blocks + tile_blocks) * threads > 0xffffffffLL || folds * 256 > 0xffffffffLL) return hipErrorNotSupported;
  p.number = pl.few.slots ? launch_number() : 0;
  p.few_blocks = (int)few_blocks;
  auto kernel_of = [&](auto mode) {
    constexpr PagedMode MODE = decltype(mode)::value;
    if (dt == kDtFloat16) return eight ? paged_attn_kernel<_Float16, true, MODE> : paged_attn_kernel<_Float16, false, MODE>;
    return eight ? paged_attn_kernel<__bf16, true, MODE> : paged_attn_kernel<__bf16, false, MODE>;
  };
  auto kern = kernel_of(std::integral_constant<PagedMode, kBoth>());
  switch (pl.mode()) {
    case kFewRows: kern = kernel_of(std::integral_constant<PagedMode, kFewRows>()); break;
    case kFewRuns: kern = kernel_of(std::integral_constant<PagedMode, kFewRuns>()); break;
    case kTiles: kern = kernel_of(std::integral_constant<PagedMode, kTiles>()); break;
    case kWideTiles: kern = kernel_of(std::integral_constant<PagedMode, kWideTiles>()); break;
    case kBoth: break;
  }
  const PagedEarly early(p);
  const hipError_t e = launch(kern, dim3((uint32_t)(few_blocks + tile_blocks)), (unsigned)threads, 0, stream, early.a, early.b, early.c, p);
  if (e != hipSuccess || folds == 0) return e;
  return launch(dt == kDtFloat16 ? paged_combine_kernel<_Float16> : paged_combine_kernel<__bf16>, dim3((uint32_t)folds), 256, 0, stream, early.a,
                early.b, early.c, p);
}

}  // namespace llmhip
