// Rows into a cache of pages, rotated and in 8 bits if the cache is, and back out of it.  gfx950.
//
//   append:  out_q[t] = rope(in_q[t], position p of token t);  K[p] = store(rope(in_k[t], p));  V[p] = store(in_v[t])
//   read:    out_k[t] = widen(K[p]), out_v[t] = widen(V[p]);  zeros where there is no such row
//
// with p = kv_lens[b] - q_starts[b + 1] + t for the tokens t of sequence b, store() and widen() the identity in a 16-bit cache and the
// 8-bit form of paged.hpp otherwise.  The rotation is that of rope_kv_append.hip (every product and sum rounded on its own, this file is
// compiled with -ffp-contract=off; then once to the storage type), and 8 bits are taken of its result: what the cache holds does
// not depend on whether a row went in at once or by way of a 16-bit cache.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "paged.hpp"
#include "rotate.hpp"

namespace llmhip {

// Rows read back: this many tokens to a workgroup from so many on, which are two workgroups to a CU (below, one: 301 tokens 2.3 us).
constexpr int kReadTokens = 4, kManyTokens = 2048;

// A launch takes fewer than 2^32 threads along a dimension: workgroup w is the one at (w % 2^20, w / 2^20) of the first and third.
constexpr int kGridShift = 20;
static dim3 grid_of(int workgroups, unsigned y = 1) {
  const unsigned all = (unsigned)workgroups, most = 1u << kGridShift;
  return all <= most ? dim3(all, y) : dim3(most, y, (all + most - 1) >> kGridShift);
}
__device__ __forceinline__ int workgroup() { return (int)(blockIdx.z << kGridShift | blockIdx.x); }

struct PagedAppend {
  PagedBatch batch;
  char *out_q, *k_pages, *v_pages;
  const char *in_q, *in_k, *in_v;
  const float *freq_cis;
  int table_rows, q_heads, kv_heads;
};

// e4m3 of 8 values of the storage type, scaled; not finite: NaN.
template <typename T> __device__ __forceinline__ u32x2_t narrow8(const float (&x)[8], float scale) {
  u32x2_t out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * scale, x[4 * i + 1] * scale, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * scale, x[4 * i + 3] * scale, w, true);
    out[i] = (uint32_t)w;
  }
  return out;
}
// 8 values as floats, limited; the largest finite magnitude goes into `most`
template <typename T> __device__ __forceinline__ void limited8(u32x4_t v, float (&x)[8], float &most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = Elem<T>::widen((uint16_t)(v[i >> 1] >> ((i & 1) * 16)));
    const bool finite = __builtin_fabsf(f) < INFINITY;
    x[i] = finite ? __builtin_amdgcn_fmed3f(f, -most_cached<T>(), most_cached<T>()) : __builtin_nanf("");
    most = fmaxf(most, finite ? __builtin_fabsf(x[i]) : 0.0f);
  }
}

// A workgroup has a token, 8 lanes to a row as in rope_kv_append.hip, 32 rows at a time.  Where the token is is the same to all: scalar
// work.  Many tokens are bound by the memory system: 4096 of 28 + 2 x 4 heads, 78 MB in and out, in 17.7 us, 4.4 TB/s (a plain copy of as
// much 16.3; the contiguous cache's kernel, which deals rows to lanes across tokens, 14.4: here 36 rows are two turns of 32, the second with
// four); in 8 bits, 73 MB, as long.  Several tokens to a workgroup, and rows dealt to lanes across tokens, were slower (20-23).  Few by their chain of
// loads, starts to page table to stores: 24 in 8 bits 2.8 us, of which an empty launch is 1.6.
template <typename T, bool NEOX, bool EIGHT> __global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend p) {
  const int token = workgroup(), tid = threadIdx.x, lane = tid & 63, j = tid & 7;
  const TokenSequence s = sequence_of(p.batch, token, lane);
  const int pos = s.pos;
  if (s.b < 0 || pos < 0 || pos >= p.table_rows) return;
  const PagePlace at = page_place(p.batch, s.b, pos);
  const int rows = p.q_heads + 2 * p.kv_heads, page_rows = (int)p.batch.page_size.d;
  const float *tab = p.freq_cis + (size_t)pos * kHeadDim + (NEOX ? 16 : 8) * j;
  f32x4_t cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = *reinterpret_cast<const f32x4_t *>(tab + (NEOX ? 4 * i : 64 * (i >> 1) + 4 * (i & 1)));
  for (int r = blockIdx.y * 32 + (tid >> 3); r < rows; r += 32 * gridDim.y) {
    const bool is_q = r < p.q_heads, is_v = r >= p.q_heads + p.kv_heads;
    const int h = is_q ? r : r - p.q_heads - (is_v ? p.kv_heads : 0);
    const char *in = (is_q ? p.in_q + ((size_t)token * p.q_heads + h) * kRowBytes : (is_v ? p.in_v : p.in_k) + ((size_t)token * p.kv_heads + h) * kRowBytes) + j * 16;
    u32x4_t va = global_load_b128(in), vb = global_load_b128(in + 128);
    if (!is_v) rotate8<T, NEOX>(va, vb, cs);
    if (is_q) {
      char *out = p.out_q + ((size_t)token * p.q_heads + h) * kRowBytes + j * 16;
      store_device_b128(out, va);
      store_device_b128(out + 128, vb);
      continue;
    }
    if (!at.there(p.batch)) continue;
    char *page = (is_v ? p.v_pages : p.k_pages) + (int64_t)at.page * p.batch.page_stride;
    const int row = h * page_rows + at.row;
    if constexpr (!EIGHT) {
      char *out = page + (size_t)row * kRowBytes + j * 16;
      store_device_b128(out, va);
      store_device_b128(out + 128, vb);
    } else {
      float x[8], y[8], most = 0.0f;
      limited8<T>(va, x, most);
      limited8<T>(vb, y, most);
      most = max_of_lanes<8>(most);
      const int byte = exponent_byte(most);
      const float scale = power_of_two(254 - byte);
      char *out = page + (size_t)row * kHeadDim + j * 8;
      *reinterpret_cast<u32x2_t *>(out) = narrow8<T>(x, scale);
      *reinterpret_cast<u32x2_t *>(out + 64) = narrow8<T>(y, scale);
      if (j == 0) page[(size_t)p.kv_heads * page_rows * kHeadDim + row] = (char)byte;
    }
  }
}

hipError_t launch_paged_append(void *out_q, void *k_pages, void *v_pages, const PagedBatch &batch, const void *freq_cis, const void *in_q,
                               const void *in_k, const void *in_v, int table_rows, int q_heads, int kv_heads, int is_neox, bool eight,
                               int dt, hipStream_t stream) {
  // A token's rows over several workgroups where there are fewer tokens than CUs (us, one / several: 24 tokens of 40 + 2 x 8 heads in 8
  // bits 3.4 / 2.8; 300 of 28 + 2 x 4 5.7 / 5.1; 8 x 512 of them 19.1 / 20.8, in 8 bits 19.4 / 21.5).
  const unsigned spread = batch.tokens < device_compute_units() ? (unsigned)(q_heads + 2 * kv_heads + 31) / 32 : 1u;
  const PagedAppend p = {batch,
                         static_cast<char *>(out_q),
                         static_cast<char *>(k_pages),
                         static_cast<char *>(v_pages),
                         static_cast<const char *>(in_q),
                         static_cast<const char *>(in_k),
                         static_cast<const char *>(in_v),
                         static_cast<const float *>(freq_cis),
                         table_rows,
                         q_heads,
                         kv_heads};
  auto kernel_of = [&](auto t) {
    using T = decltype(t);
    if (eight) return is_neox ? paged_append_kernel<T, true, true> : paged_append_kernel<T, false, true>;
    return is_neox ? paged_append_kernel<T, true, false> : paged_append_kernel<T, false, false>;
  };
  return launch(dt == kDtFloat16 ? kernel_of(_Float16()) : kernel_of(__bf16()), grid_of(batch.tokens, spread), 256, 0, stream, p);
}

struct PagedRead {
  PagedBatch batch;
  char *out_k, *out_v;
  const char *k_pages, *v_pages;
  int kv_heads;
};

// A workgroup has TOKENS tokens; 16 lanes to a row, 16 rows of a token at a time.  All loads of a turn go out before the first is used.  Bound by
// the memory system: 32768 rows of 8 kv heads in 8 bits, 202 MB in and out, in 39.6 us, 5.1 TB/s.  (TOKENS, us: 1 56, 2 46, 4 39.7, 8 41; with
// ordinary stores 44.)
template <typename T, bool EIGHT, int TOKENS> __global__ __launch_bounds__(256) void paged_read_kernel(PagedRead p) {
  const int token0 = workgroup() * TOKENS, tid = threadIdx.x, lane = tid & 63, j = tid & 15;
  const TokenPlace places = token_places<TOKENS>(p.batch, token0, lane);
  const int page_rows = (int)p.batch.page_size.d;
  for (int r = tid >> 4; r < 2 * p.kv_heads; r += 16) {
    const bool is_v = r >= p.kv_heads;
    const int h = r - (is_v ? p.kv_heads : 0);
    const char *pool = is_v ? p.v_pages : p.k_pages;
    using Raw = std::conditional_t<EIGHT, u32x2_t, u32x4_t>;
    Raw v[TOKENS];
    int byte[TOKENS];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
      const int at_page = __builtin_amdgcn_readlane(places.page, i), row = h * page_rows + __builtin_amdgcn_readlane(places.row, i);
      v[i] = Raw{};
      byte[i] = 127;
      if (at_page < 0) continue;
      const char *page = pool + (int64_t)at_page * p.batch.page_stride;
      v[i] = __builtin_nontemporal_load(reinterpret_cast<const Raw *>(page + (size_t)row * cached_row_bytes(EIGHT) + j * sizeof(Raw)));
      if (EIGHT) byte[i] = (uint8_t)page[(size_t)p.kv_heads * page_rows * kHeadDim + row];
    }
    char *out = (is_v ? p.out_v : p.out_k) + ((size_t)token0 * p.kv_heads + h) * kRowBytes + j * 16;
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
      if (__builtin_amdgcn_readlane(places.pos, i) == -1) continue;
      u32x4_t x;
      if constexpr (EIGHT)
        x = widen8<T>(v[i][0], v[i][1], power_of_two(byte[i]));
      else
        x = v[i];
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t *>(out + (size_t)i * p.kv_heads * kRowBytes));
    }
  }
}

hipError_t launch_paged_read(void *out_k, void *out_v, const void *k_pages, const void *v_pages, const PagedBatch &batch, int kv_heads, bool eight,
                             int dt, hipStream_t stream) {
  const PagedRead p = {batch,
                       static_cast<char *>(out_k),
                       static_cast<char *>(out_v),
                       static_cast<const char *>(k_pages),
                       static_cast<const char *>(v_pages),
                       kv_heads};
  auto kernel_of = [&](auto t, auto tokens) {
    constexpr int N = decltype(tokens)::value;
    return eight ? paged_read_kernel<decltype(t), true, N> : paged_read_kernel<decltype(t), false, N>;
  };
  const bool many = batch.tokens >= kManyTokens;
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, kReadTokens> some;
  const auto kern = dt == kDtFloat16 ? (many ? kernel_of(_Float16(), some) : kernel_of(_Float16(), one))
                                     : (many ? kernel_of(__bf16(), some) : kernel_of(__bf16(), one));
  return launch(kern, grid_of((batch.tokens + (many ? kReadTokens - 1 : 0)) / (many ? kReadTokens : 1)), 256, 0, stream, p);
}

}  // namespace llmhip
