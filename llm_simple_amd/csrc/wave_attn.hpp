// The attention state of one wave with 32 query rows and its work on tiles of keys in LDS: of the prefill kernels
// (flash_prefill.hip, whose header comment describes it) and of the kernel over pages (paged_attn.hip).
#pragma once
#include <type_traits>

#include "common.hpp"

namespace LLMHIP_NS {

constexpr float kLazyLog2 = 8.0f;                // rescale threshold, log2 units

// max / sum over the lane pair (l, l^32) without going through the LDS
// crossbar.  v_permlane32_swap(a, b) exchanges a[32..63] with b[0..31]; with
// a == b == x the two results are (x_lo, x_lo) and (x_hi, x_hi).  The results
// are copied to scalars before the bit cast: a bit cast applied directly to a
// vector element reads element 0.
__device__ __forceinline__ void pair_swap(float x, float &lo, float &hi) {
  typedef __attribute__((ext_vector_type(2))) unsigned u2;
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const u2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned r0 = r[0], r1 = r[1];
  lo = __builtin_bit_cast(float, r0);
  hi = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float pair_max(float x) {
  float lo, hi;
  pair_swap(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float pair_sum(float x) {
  float lo, hi;
  pair_swap(x, lo, hi);
  return lo + hi;
}

// LDS visibility + workgroup barrier that does not drain outstanding global loads.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// State of one wave: 32 query rows (one per lane pair), fp32 O^T accumulators.  KB = 32-key blocks
// of every 64-key tile that the wave works on: 2 normally; 1 when two waves share the rows and
// each takes one half of every tile (short sequences: halves the serial MFMA chain of a wave).
template <typename T, int KB = 2> struct WaveAttn {
  using E = Elem<T>;
  f32x16_t o[4];       // O^T: d block x (16 d rows of this lane)
  u32x4_t pf[KB][2];   // P^T packed as B operand: key block x k-step
  u32x4_t qf[8];       // Q^T fragments (B operand), loaded once
  float m_run, l_run;  // running max (raw score units) and sum of this lane's keys
  float move_above, neg_ms;  // m_run plus the slack of its move; what it adds to the exponent
  int lane, l32, hh, g16, li;
  int k_addr[8];  // LDS byte offset of this lane's K fragment kk in tile slot 0, key block 0
  uint32_t v_addr[4];  // LDS address of the V^T fragment of d block d (k-step 0, low half)

  // kb0: first 32-key block of a tile this wave works on (0, or 1 for the second wave of a pair)
  __device__ __forceinline__ void init(const char *lds, int lane_, int v_region, int kb0 = 0) {
    lane = lane_;
    l32 = lane & 31;
    hh = lane >> 5;
    g16 = lane >> 4;
    li = lane & 15;
    m_run = -INFINITY;
    move_above = -INFINITY;
    neg_ms = 0.0f;
    l_run = 0.0f;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    // Every other fragment address of the loop is one of these plus a compile-time constant
    // that fits the 16-bit offset field of the LDS instructions; the empty asm keeps the
    // compiler from recomputing them (it otherwise spends ~50 VALU instructions per tile).
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      k_addr[kk] = k_swizzle_off(l32, 2 * kk + hh) + kb0 * 32 * kRowBytes;
      asm volatile("" : "+v"(k_addr[kk]));
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int gran = d * 4 + (g16 & 1) * 2 + ((li & 3) >> 1);
      v_addr[d] = lds_address(lds) + v_region + v_swizzle_off(4 * hh + (li >> 2), gran) + (li & 1) * 8 + kb0 * 32 * kRowBytes;
      asm volatile("" : "+v"(v_addr[d]));
    }
  }

  // Q^T fragments of 32 rows in LDS, laid out like a K tile; off: their place less this wave's first tile row
  __device__ __forceinline__ void load_q_lds(const char *lds, int off) {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) qf[kk] = lds_read_b128(lds, k_addr[kk] + off);
  }
  struct NoHook {
    template <typename I> __device__ __forceinline__ void operator()(I) const {}
  };
  // S^T = K Q^T for the wave's keys of the K tile at byte offset `koff` of the LDS segment.
  // The fragments of step kk+1 are requested before the MFMAs of step kk.  hook(i) runs
  // after MFMA i (0..8*KB-1): the callers spread their global loads over the MFMA stream with it.
  template <int KK0 = 0, int KK1 = 8, typename Hook = NoHook>
  __device__ __forceinline__ void qk(const char *lds, int koff, f32x16_t (&s)[KB], Hook hook = Hook()) {
    static_for<KK0, KK1>([&](auto kk_) {
      constexpr int kk = decltype(kk_)::value;
      static_for<0, KB>([&](auto kb_) {
        constexpr int kb = decltype(kb_)::value;
        const u32x4_t kf = lds_read_b128(lds, k_addr[kk] + koff + kb * 32 * kRowBytes);
        if constexpr (kk == 0) {
          f32x16_t z;
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = 0.0f;
          s[kb] = E::mfma32(kf, qf[kk], z);
        } else {
          s[kb] = E::mfma32(kf, qf[kk], s[kb]);
        }
        hook(std::integral_constant<int, kk * KB + kb>());
      });
    });
  }

  // O^T += V^T P^T over the V tile at byte offset `voff` past the start of the V region, pieces I0 .. I1 - 1 of 16 keys.
  // Lane (d = 32*dblk + l32, hh): element e of k-step (kb, ks2) is the key
  // 32*kb + 16*ks2 + 8*(e/4) + 4*hh + e%4 -- the key P's element e carries.
  template <int I0 = 0, int I1 = 2 * KB, typename Hook = NoHook>
  __device__ __forceinline__ void pv(int voff, Hook hook = Hook()) {
    static_for<4 * I0, 4 * I1>([&](auto i_) {
      constexpr int i = decltype(i_)::value, kb = i / 8, ks2 = i / 4 % 2, d = i % 4;
      const int c = voff + (kb * 32 + ks2 * 16) * kRowBytes;
      const u32x2_t lo = lds_read_tr16(v_addr[d], c);
      const u32x2_t hi = lds_read_tr16(v_addr[d], c + 8 * kRowBytes);
      const u32x4_t vf = {lo[0], lo[1], hi[0], hi[1]};
      o[d] = E::mfma32(vf, pf[kb][ks2], o[d]);
      hook(i_);
    });
  }

  // Causal / length mask of one tile of scores (only called for tiles that can be cut); key0 =
  // first key of the wave's part of the tile.
  __device__ __forceinline__ void mask(f32x16_t (&s)[KB], int key0, int qrow, int offset, int n) {
    const int last = min(qrow + offset, n - 1) - key0 - 4 * hh;  // the lane's last key, from its first one
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kb * 32 + 8 * (i >> 2) + (i & 3) > last) s[kb][i] = -INFINITY;
  }

  // P = exp2(s*c + neg_ms) rounded to T and packed as the B operand; returns this lane's sum
  // of the rounded values.
  __device__ __forceinline__ float probabilities(const f32x16_t (&s)[KB], float c) {
    float ps0 = 0.0f, ps1 = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int ks2 = 0; ks2 < 2; ++ks2) {
        u32x4_t w;
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) {
          const float e0 = fast_exp2(__builtin_fmaf(s[kb][8 * ks2 + 2 * e2], c, neg_ms));
          const float e1 = fast_exp2(__builtin_fmaf(s[kb][8 * ks2 + 2 * e2 + 1], c, neg_ms));
          w[e2] = E::pack2(e0, e1);
          // l sums the ROUNDED probabilities, the values P.V really used: for rows that see few
          // keys the rounding errors of numerator and denominator then cancel.  (In a design that
          // separates MFMA and softmax phases these dot instructions are costly -- they queue
          // behind the MFMAs of every wave on the SIMD: a softmax pass beside an MFMA-issuing wave
          // takes 1690 cycles with them, 1070 with plain adds -- in this interleaved loop the
          // two versions time the same.)
          if (e2 & 1)
            ps1 = dot2_ones<T>(w[e2], ps1);
          else
            ps0 = dot2_ones<T>(w[e2], ps0);
        }
        pf[kb][ks2] = w;
      }
    return ps0 + ps1;
  }

  // probabilities() and pv() in one, the exponentials between the matrix instructions, in the order they are to be issued: for kernels whose
  // registers are so full that the compiler leaves the order as it is.  The first five quarters of a piece of 16 keys go before, then one to a
  // matrix instruction (8-bit tiles over pages, us, all before / 4 / 5 / 6 quarters: a prompt of 2048 tokens of 28 + 4 heads 68.5 / 66.0 / 63.7 / 69.1,
  // 8192 with a window of 1024 176 / 169 / 165 / 177; and in qk's place, from its third fragment on, 67-70 and 171-178).
  __device__ __forceinline__ float probabilities_and_pv(const f32x16_t (&s)[KB], float c, int voff) {
    constexpr int kAhead = 5;
    float ps0 = 0.0f, ps1 = 0.0f;
    auto quarter = [&](auto j_) {  // of the four pairs of each piece
      constexpr int j = decltype(j_)::value, kb = j / 8, ks2 = j / 4 % 2, e2 = j % 4;
      const float e0 = fast_exp2(__builtin_fmaf(s[kb][8 * ks2 + 2 * e2], c, neg_ms));
      const float e1 = fast_exp2(__builtin_fmaf(s[kb][8 * ks2 + 2 * e2 + 1], c, neg_ms));
      const uint32_t w = E::pack2(e0, e1);
      pf[kb][ks2][e2] = w;
      if (e2 & 1)
        ps1 = dot2_ones<T>(w, ps1);
      else
        ps0 = dot2_ones<T>(w, ps0);
    };
    static_for<0, kAhead>(quarter);
    static_for<0, 2 * KB>([&](auto i_) {
      constexpr int i = decltype(i_)::value;
      pv<i, i + 1>(voff, [&](auto j_) {
        constexpr int j = decltype(j_)::value + kAhead;
        if constexpr (j < 8 * KB) quarter(std::integral_constant<int, j>());
      });
    });
    return ps0 + ps1;
  }

  // First half of the online softmax of one tile of (already masked) scores: row maxima and,
  // rarely, the move of the reference.  m_run is the reference maximum used in the exponent,
  // in raw score units.  It moves only when a row maximum exceeds it by more than kLazyLog2
  // in log2 units (probabilities then stay below 2^kLazyLog2, harmless in fp32 sums and in
  // the 16-bit P operand); a -inf reference always moves.  O and l are rescaled only then,
  // which after the first tiles is rare: what depends on the reference alone (the line `move_above`, the additive term
  // of the exponent) is computed then too, and a lane pair compares notes only then.  LAZY false: it moves with every new maximum.
  template <bool LAZY = true> __device__ __forceinline__ void row_max(const f32x16_t (&s)[KB], float scale_log2e) {
    float m0 = -INFINITY, m1 = -INFINITY;  // two chains: half the dependent latency
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (KB == 2) {
        m0 = fmaxf(m0, s[0][i]);
        m1 = fmaxf(m1, s[KB - 1][i]);
      } else if (i & 1) {
        m1 = fmaxf(m1, s[0][i]);
      } else {
        m0 = fmaxf(m0, s[0][i]);
      }
    }
    float mloc = fmaxf(m0, m1);
    if (__builtin_amdgcn_ballot_w64(mloc > move_above) != 0) {
      mloc = pair_max(mloc);
      const bool move = mloc > move_above;
      const float m_new = move ? mloc : m_run;
      const float m_use = (m_new == -INFINITY) ? 0.0f : m_new;
      const float alpha = move ? fast_exp2((m_run - m_use) * scale_log2e) : 1.0f;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
      m_run = m_new;
      move_above = LAZY ? m_new + kLazyLog2 / scale_log2e : m_new;
      neg_ms = -m_use * scale_log2e;
    }
  }

  // KP waves that shared the rows (KB == 1) trade pieces of O^T: wave `part` keeps and will store the
  // ND = 4 / KP d blocks part*ND .., and hands every other wave the blocks that one keeps, with its maximum and
  // sum.  All as 16-byte pieces, lane by lane: conflict-free.  The maxima are uniform over a lane pair in
  // all of them.  lds_rows: trade_bytes(KP) bytes of the row block.
  static constexpr int kPieceBytes = 4 * 1024;  // one d block of a wave
  static constexpr int give_bytes(int kp) { return (4 - 4 / kp) * kPieceBytes + 512; }
  static constexpr int trade_bytes(int kp) { return kp * give_bytes(kp); }
  template <int KP> __device__ __forceinline__ void give(char *lds_rows, int part) const {
    constexpr int ND = 4 / KP;
    char *mine = lds_rows + part * give_bytes(KP);
    f32x4_t *dst = reinterpret_cast<f32x4_t *>(mine) + lane;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if (d / ND == part) continue;  // (wave-uniform)
      f32x4_t *piece = dst + (d / ND < part ? d : d - ND) * 256;
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
        piece[i4 * 64] = f32x4_t{o[d][4 * i4], o[d][4 * i4 + 1], o[d][4 * i4 + 2], o[d][4 * i4 + 3]};
    }
    *reinterpret_cast<float2 *>(mine + give_bytes(KP) - 512 + lane * 8) = float2{m_run, l_run};
  }
  // Folds what the others gave into d blocks PART*ND ..
  template <int KP, int PART> __device__ __forceinline__ void take(const char *lds_rows, float scale_log2e) {
    constexpr int ND = 4 / KP;
    float2 ml[KP];
    float m_new = m_run;
#pragma unroll
    for (int q = 0; q < KP; ++q) {
      ml[q] = float2{m_run, l_run};
      if (q != PART)
        ml[q] = *reinterpret_cast<const float2 *>(lds_rows + (q + 1) * give_bytes(KP) - 512 + lane * 8);
    }
#pragma unroll
    for (int q = 0; q < KP; ++q) m_new = fmaxf(m_new, ml[q].x);
    const float m_use = (m_new == -INFINITY) ? 0.0f : m_new;
    const float f_own = fast_exp2((m_run - m_use) * scale_log2e);
    float l = 0.0f;  // in the same order in every wave
#pragma unroll
    for (int d = PART * ND; d < PART * ND + ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] *= f_own;
#pragma unroll
    for (int q = 0; q < KP; ++q) {
      const float f = fast_exp2((ml[q].x - m_use) * scale_log2e);
      l = __builtin_fmaf(ml[q].y, f, l);
      if (q == PART) continue;
      const f32x4_t *src = reinterpret_cast<const f32x4_t *>(lds_rows + q * give_bytes(KP)) + lane;
#pragma unroll
      for (int d = PART * ND; d < PART * ND + ND; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const f32x4_t v = src[((d / ND < q ? d : d - ND) * 4 + i4) * 64];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][4 * i4 + i] = __builtin_fmaf(v[i], f, o[d][4 * i4 + i]);
        }
    }
    m_run = m_new;
    l_run = l;
  }

  // out[row][head][32*D0 .. +32*ND) = O^T / l, rounded once.  The lane layout of O^T (a lane holds 4
  // contiguous dims of one row at 4*ND places) would make every store instruction touch 32
  // rows with 16 bytes each; the tile goes through 2*ND KiB of LDS of this wave instead
  // (16-byte granule XOR row: conflict-free both ways with four d blocks; rows of one or two are shorter
  // than the banks, and up to 8 lanes meet in one, 1-2 % of a launch's cycles) and leaves as whole pieces of
  // 64*ND bytes, 4*ND lanes per row, past the L2: lines that are left there are written back at the end of the launch (rope
  // and attention, us, ordinary stores / these: 256 tokens of 28 heads 9.39 / 9.20, 600 14.64 / 14.16, 1019 20.5 / 19.7, of
  // 32 26.3 / 25.7, 2048 of 28 44.5 / 43.8; up to 128 tokens and from 4096 on the same).  So too with ND = 1, pieces of 64 bytes from
  // two waves to a line: a sector is enough (attention alone, us: 256 of 32 5.44 / 5.29, 512 of 28 7.98 / 7.78, 2000 of 12 22.7 / 22.4), and
  // where the output begins off a sector (16 bytes off: 512 of 28 8.80 / 8.60, 1019 18.0 / 17.4, of 32 19.8 / 19.6, 2048 of 28 41.7 / 41.7, 4096
  // 125.4 / 125.2).  lds_wave: this wave's region; out_blk: &out[first row of the
  // wave][head]; rows_valid: how many of the wave's 32 rows exist.
  template <int D0 = 0, int ND = 4>
  __device__ __forceinline__ void store(char *lds_wave, char *out_blk, size_t row_bytes, int rows_valid) {
    constexpr int G = 4 * ND, RB_ = G * 16, RPI = 64 / G;  // granules and bytes of a row, rows per instruction
    const float l_tot = pair_sum(l_run);
    const float inv = (l_tot > 0.0f) ? 1.0f / l_tot : 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        u32x2_t w;
        w[0] = E::pack2(o[D0 + d][4 * i4] * inv, o[D0 + d][4 * i4 + 1] * inv);
        w[1] = E::pack2(o[D0 + d][4 * i4 + 2] * inv, o[D0 + d][4 * i4 + 3] * inv);
        const int gran = 4 * d + i4;  // 16-byte granule of dims 32d + 8*i4 .. +7; hh picks its half
        *reinterpret_cast<u32x2_t *>(lds_wave + l32 * RB_ + ((gran ^ (l32 & (G - 1))) << 4) + hh * 8) = w;
      }
    __builtin_amdgcn_wave_barrier();  // wave-private region: LDS ops of one wave complete in order
    const int r0 = lane / G, g0 = lane % G;
    u32x4_t v[2 * ND];
#pragma unroll
    for (int t = 0; t < 2 * ND; ++t) {
      const int r = RPI * t + r0;
      v[t] = lds_read_b128(lds_wave, r * RB_ + ((g0 ^ (r & (G - 1))) << 4));
    }
    char *dst = out_blk + (size_t)r0 * row_bytes + D0 * 64 + g0 * 16;
#pragma unroll
    for (int t = 0; t < 2 * ND; ++t) {
      if (RPI * t + r0 < rows_valid) store_device_b128(dst, v[t]);
      dst += RPI * row_bytes;
    }
  }
};

}  // namespace LLMHIP_NS
