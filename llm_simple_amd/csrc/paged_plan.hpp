// How a launch of the attention over pages is shaped (paged_attn.hip), from bounds on its sizes.  Host code.
#pragma once
#include "common.hpp"
#include "kernels.hpp"
#include "paged.hpp"

namespace LLMHIP_NS {

constexpr int kFewCols = 16;     // rows of a few-rows workgroup
constexpr int kFlagBytes = 16;   // place of a flag (few_rows_of)
constexpr int kFewUnit = 128;    // keys of a unit, 32 to a wave
constexpr int kTileRows = 128;   // rows of a tile (wide: twice as many)
constexpr int kTileUnit = 64;    // keys of a unit
constexpr int kRunUnits = 24;    // of each part, where few rows may be taken in runs (FewRuns)

// The kernels
enum PagedMode { kFewRows, kFewRuns, kTiles, kWideTiles, kBoth };
constexpr int threads_of(PagedMode mode) { return mode == kWideTiles ? 512 : 256; }

// How a launch is shaped, from what the host knows: bounds, not lengths.
struct PagedPlan {
  struct Kind {
    long long tiles, items, slots, rows;  // at most; rows of a partial
    int least, parts;
    bool flags;
    size_t bytes(int Hkv) const { return (size_t)slots * Hkv * (rows * (kHeadDim + 2) * sizeof(float) + (flags ? kFlagBytes : 0)); }
    long long folds() const { return slots / 2 < tiles ? slots / 2 : tiles; }  // tiles that are split, at most
  } few, by_tiles;
  bool runs;  // may be taken
  bool wide;  // tiles of 256 rows, for launches without few rows
  size_t bytes(int Hkv) const { return few.bytes(Hkv) + by_tiles.bytes(Hkv); }
  PagedMode mode() const { return by_tiles.items == 0 ? (runs ? kFewRuns : kFewRows) : few.items != 0 ? kBoth : wide ? kWideTiles : kTiles; }
};
// Wide tiles, 8 waves of 32 rows and one workgroup to a CU, read K and V half as often, and widen 8 bits half as often, but are half as many,
// to be dealt to half as many places.  They are taken where rows do not fill them much worse than narrow ones, and either long caches
// behind few tokens, which are cut into parts of about one length, are work for all places, or 8-bit prompts make rounds enough (us, narrow / wide:
// 500 past 30000 of 28 + 4 heads 240 / 226, in 8 bits 273 / 239; 200 past 16001 67.2 / 65.5, 73.7 / 69.5; 4 x 130 past 9000 91.0 / 87.6; 100 past
// 4000 22.6 / 26.3, 27.5 / 30.9; prompts, whose tiles differ in length: of 2048 52.1 / 58.9, 63.4 / 66.4, of 4096 141 / 132, 156 / 137, of 6000 273 / 276,
// 299 / 291, of 4000 of 40 + 8 180 / 185, 198 / 194).
inline PagedPlan plan_paged(int tokens, int batch, int max_q_len, int max_kv_len, int window, int sinks, int g, int Hkv, bool eight) {
  PagedPlan pl = {};
  const long long cus = device_compute_units(), sequences = batch < tokens ? batch : tokens;  // that have new tokens at all
  const bool tiles = (long long)max_q_len * g > kFewCols;
  // (all sequences have max_q_len tokens, or the tokens do not add up: no few-rows ones)
  if (!tiles || (g <= kFewCols && (long long)batch * max_q_len != tokens)) pl.few.tiles = sequences;
  auto deal = [&](PagedPlan::Kind &kind, int rows, int unit, long long span, long long workgroups, int least) {
    kind.rows = rows;
    kind.flags = rows == kFewCols;
    kind.least = least;
    kind.parts = Hkv <= workgroups ? (int)(workgroups / Hkv) : 1;
    const long long windowed = (long long)window + span + sinks + 2 * kPageGroup, seen = window > 0 && windowed < max_kv_len ? windowed : max_kv_len;
    const long long units = (seen + unit - 1) / unit, all = (long long)kind.parts + 1 + kind.parts / 64;
    kind.slots = kind.tiles > 0 && units > least && Hkv <= workgroups ? 2 * all : 0;
    const long long most = kind.tiles * (units / least + 1);
    if (kind.slots > most) kind.slots = most;
    kind.items = kind.tiles + (kind.slots ? all : 0);
    return units;
  };
  const long long units = deal(pl.few, kFewCols, kFewUnit, kFewCols, cus, 3);
  pl.runs = batch > 1 && batch <= 64 && pl.few.slots > 0 && pl.few.tiles * units >= (long long)kRunUnits * pl.few.parts;
  auto deal_tiles = [&](bool wide) {
    const int rows = wide ? 2 * kTileRows : kTileRows;
    pl.wide = wide;
    if (tiles) pl.by_tiles.tiles = (long long)tokens * g / rows + sequences;
    return deal(pl.by_tiles, rows, kTileUnit, rows / g + 1, wide ? cus : 2 * cus, 6);
  };
  if (tiles && !pl.few.tiles) {
    auto filled = [&](int rows) { return ((long long)max_q_len * g + rows - 1) / rows * rows; };
    const long long seen = deal_tiles(true), count = pl.by_tiles.tiles, parts = pl.by_tiles.parts;
    const bool chunks = max_kv_len / 4 >= max_q_len && count * (seen / 6) >= parts, rounds = eight && window <= 0 && 2 * count >= 3 * parts;
    if (8 * filled(2 * kTileRows) <= 9 * filled(kTileRows) && (chunks || rounds)) return pl;
  }
  deal_tiles(false);
  return pl;
}

}  // namespace LLMHIP_NS
