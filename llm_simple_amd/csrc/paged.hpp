// A KV cache in pages: where a sequence's rows are, and the 8-bit form of a row.
//
// K and V each have a pool of pages, page_stride bytes apart.  A page holds [kv head][page_size] rows of 128, so that the 16 keys of
// a matrix instruction are one piece of 4 KiB (2 KiB in 8 bits), and in 8 bits behind them [kv head][page_size] exponent bytes.
// page_size is a multiple of 16: 16 keys that begin at a multiple of 16 are in one page.
//
// 8 bits: x = e4m3 * 2^(byte - 127), the byte of each row the least one with max|x| <= 448 * 2^(byte - 127), at least 64.  A power of two,
// because then nothing but the rounding to e4m3 is lost: division by the scale, and the product on the way back, are exact, and a
// conversion instruction takes the scale along.  (Below 2^-63 a row is as good as zero: the floor keeps all of it away from subnormals.)
//
// Lengths, starts and the page table are device memory that a captured graph may see change: the kernels trust none of it.  A page
// number outside of the pool, or beyond the table, is a page that is not there: its keys are not seen, rows for it are not written.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"

namespace LLMHIP_NS {

constexpr int kPageGroup = 16;  // keys that are in one page whatever its size

// [rows of the dense tensors] q_starts[b] .. q_starts[b + 1] are the last rows of the kv_lens[b] cached ones of sequence b.
struct PagedBatch {
  const int *page_table, *q_starts, *kv_lens;
  int batch, tokens, pages_per_seq, num_pages;
  int keys_max;  // pages_per_seq * page_size, at most 2^31 - 2^16
  FastDiv page_size;
  int64_t page_stride;
};

__host__ __device__ constexpr int cached_row_bytes(bool eight) { return eight ? kHeadDim : kRowBytes; }

// Where a key's row is.  page: as it stands in the table, nothing waits for the load before there() asks; -1 past the table.
struct PagePlace {
  int page, row;
  __device__ __forceinline__ bool there(const PagedBatch &p) const { return (uint32_t)page < (uint32_t)p.num_pages; }
};
__device__ __forceinline__ PagePlace page_place(const PagedBatch &p, int b, int key) {
  const int i = (int)fast_div(key, p.page_size);
  PagePlace at = {-1, key - i * (int)p.page_size.d};
  if (key >= 0 && i < p.pages_per_seq) at.page = p.page_table[(size_t)b * p.pages_per_seq + i];
  return at;
}

// Whether a sequence's rows and length are such as to be worked on
__device__ __forceinline__ bool sequence_ok(const PagedBatch &p, int first, int end, int len) {
  return first >= 0 && first <= end && end <= p.tokens && len >= 0 && len <= p.keys_max;
}

// The sequence that a token belongs to, and the token's position in it; b = -1: none's.  A token is a sequence's that is worked on and has it
// among its rows.
struct TokenSequence {
  int b, pos;
};
// Whether it is the one of number b's
__device__ __forceinline__ bool token_of(const PagedBatch &p, int b, int token, TokenSequence &t) {
  const int first = p.q_starts[b], end = p.q_starts[b + 1], len = p.kv_lens[b];
  t = TokenSequence{b, len - end + token};
  return sequence_ok(p, first, end, len) && first <= token && token < end;
}
// How many sequences end before or at a token, the same one to all lanes of the wave: the number of the one it belongs to, if no start goes backwards.
// ordered: none does of those that were looked at, which are all of them where all end before or at the token.
__device__ __forceinline__ int ends_upto(const PagedBatch &p, int token, int lane, bool &ordered) {
  int b = 0;
  ordered = true;
  for (int base = 0; base < p.batch; base += 64) {
    const int i = base + lane, at = min(i, p.batch - 1), first = p.q_starts[at], end = p.q_starts[at + 1];
    const bool past = i < p.batch && end <= token;
    ordered = ordered && __builtin_amdgcn_ballot_w64(first > end) == 0;
    const int count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(past));
    b += count;
    if (count < 64) break;
  }
  return __builtin_amdgcn_readfirstlane(b);
}
// The same one to all lanes: looked for in all sequences, as a start that goes backwards asks for.  (Always this way:
// append of 8 x 512 tokens of 28 + 2 x 4 heads 18.1 -> 19.0 us, of 300 x 1 5.45 -> 6.6.)
__device__ __forceinline__ TokenSequence search_sequence(const PagedBatch &p, int token, int lane) {
  for (int base = 0; base < p.batch; base += 64) {
    TokenSequence t;
    const uint64_t mine = __builtin_amdgcn_ballot_w64(token_of(p, min(base + lane, p.batch - 1), token, t));
    if (mine == 0) continue;
    const int l = __builtin_ctzll(mine);  // (lanes past the last sequence have it once more)
    return TokenSequence{base + l, __builtin_amdgcn_readlane(t.pos, l)};
  }
  return TokenSequence{-1, -1};
}
__device__ __forceinline__ TokenSequence sequence_of(const PagedBatch &p, int token, int lane) {
  TokenSequence t;
  if (p.batch == 1) return token_of(p, 0, token, t) ? t : TokenSequence{-1, -1};
  bool ordered;
  const int b = ends_upto(p, token, lane, ordered);
  if (__builtin_expect(b < p.batch && token_of(p, b, token, t), 1)) return t;
  if (b >= p.batch && ordered) return TokenSequence{-1, -1};  // (behind the last one's)
  return search_sequence(p, token, lane);
}

// Where the cached rows of TOKENS tokens from token0 on are, one to each of the first lanes.
struct TokenPlace {
  int pos;   // -1: no sequence's token, or of one that is passed over; below that: before the sequence's first row
  int page;  // -1: nowhere
  int row;
};
template <int TOKENS> __device__ __forceinline__ TokenPlace token_places(const PagedBatch &p, int token0, int lane) {
  const int token = token0 + min(lane, TOKENS - 1);
  bool ordered;
  int b = ends_upto(p, token0, lane, ordered);
  const bool behind = token >= p.tokens || (b >= p.batch && ordered);  // all sequences
  if (token != token0)
    while (b < p.batch && p.q_starts[b + 1] <= token) ++b;
  TokenSequence s = {-1, -1};
  const bool found = b < p.batch && token_of(p, b, token, s);
  if (!found) s = TokenSequence{-1, -1};
  for (uint64_t left = __builtin_amdgcn_ballot_w64(!found && !behind); left != 0; left &= left - 1) {
    const int i = __builtin_ctzll(left);
    if (i >= TOKENS) break;
    const TokenSequence x = search_sequence(p, token0 + i, lane);
    if (token == token0 + i) s = x;
  }
  TokenPlace t = {-1, -1, 0};
  if (s.b < 0) return t;
  t.pos = s.pos;
  if (t.pos < 0) {
    --t.pos;
    return t;
  }
  const PagePlace at = page_place(p, s.b, t.pos);
  t.row = at.row;
  if (at.there(p)) t.page = at.page;
  return t;
}

// ---- the 8-bit form ----

constexpr int kLeastExponent = 64;
// Magnitudes above the largest that has four significant bits in the storage type count as that one, so that what the 8 bits stand for is
// in the type.  (1.875 * 2^15, 1.875 * 2^127)
template <typename T> __device__ __forceinline__ constexpr float most_cached() { return std::is_same<T, _Float16>::value ? 61440.0f : 3.190147190316315e38f; }
// The exponent byte of a row whose largest finite magnitude is `most`: 448 = 1.75 * 2^8, so a mantissa above 1.75 takes one more.
__device__ __forceinline__ int exponent_byte(float most) {
  const int e = (int)((__builtin_bit_cast(uint32_t, most) + 0x1FFFFFu) >> 23) - 8;
  return max(e, kLeastExponent);
}
__device__ __forceinline__ float power_of_two(int byte) { return __builtin_bit_cast(float, (uint32_t)byte << 23); }

// Two e4m3 of the low or high half of a word, times a power of two, as two values of the storage type
template <typename T, bool HIGH> __device__ __forceinline__ uint32_t widen_pair(uint32_t word, float scale) {
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, HIGH));
}
// 8 e4m3 -> 8 values of the storage type
template <typename T> __device__ __forceinline__ u32x4_t widen8(uint32_t lo, uint32_t hi, float scale) {
  return u32x4_t{widen_pair<T, false>(lo, scale), widen_pair<T, true>(lo, scale), widen_pair<T, false>(hi, scale), widen_pair<T, true>(hi, scale)};
}

}  // namespace LLMHIP_NS
