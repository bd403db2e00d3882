// The per-wave half of the one-wave-per-SIMD dQ (attn_bwd_dq_ks.hip: four
// waves of the same 64 queries, each with key blocks of its own; sparse_bwd.hip:
// each wave is a workgroup): 64 queries' operands and accumulators, and the
// slot schedule and DMA of one 32-key block.
//
// Per key block j of a wave, 48 slots of one MFMA, with the block's VALU work
// dealt to fixed slots (sched_barrier), as in the other one-wave kernels:
//   slots  0-15: dP^T - D = V dO^T of block j+1 | dZ^T of block j:
//   slots 16-31: S^T = K Q^T of block j+1       |   fma, exp, mul, pack
//   slots 32-47: dQ^T += K^T dZ^T of block j    | (slots 0-38)
// K blocks live in a ring of three 8 KB places (rows of j+1, transposed reads
// of j, and j+2 on its way), V blocks in a ring of two: 40 KB per wave, the
// CU's whole LDS for four. Each place is refilled as soon as its last operand
// is read, by one DMA instruction per odd slot: V of block j+3 in slots 17-31
// (8), the first 16 keys of K of block j+3 in slots 41-47 (4) and the last 16
// of block j+2 in slots 1-7 (4). They then have 50-70 slots (about 1 us) to
// arrive, and the waits ahead of the first V read (all but the 20 youngest)
// and the first K read (16) cover exactly the loads up to those blocks.
#pragma once

#include <type_traits>

#include "tile_io.h"

namespace aa {
namespace bwd {
namespace dqks {

constexpr int kD = 128;
constexpr int kKeys = 32;                                  // keys per block
constexpr uint32_t kBlock = kKeys * kD * sizeof(bf16);     // 8 KB
constexpr uint32_t kVRing = 3 * kBlock;                    // V ring past the K ring
constexpr uint32_t kWaveBytes = 5 * kBlock;                // 40 KB

template <int n>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}
__device__ __forceinline__ void mfma_acc(f32x16& acc, bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
// 16 products of 4 x 4 x 4: with ones for A, every element of a lane's result is
// the sum of the lane's own four values of B. (Two on one accumulator stand two
// instructions apart or more.)
__device__ __forceinline__ void mfma_sum(f32x4& acc, u32x2 ones, bf16x4 b) {
  asm volatile("v_mfma_f32_4x4x4_16b_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(ones), "v"(b));
}
__device__ __forceinline__ void keep_alive(bf16x8 v) { asm volatile("" ::"v"(v)); }

// Unit u of a block: scores 2 jp, 2 jp + 1 of the dZ operand (c, qb), c =
// u >> 3, qb = (u >> 2) & 1, jp = u & 3; three stages from slot unit_slot(u).
constexpr int unit_slot(int u) { return (12 * u) / 5; }
// Operands are read two pairs of slots ahead of their MFMAs.
constexpr int kPf = 2, kRowQ = kPf + 1, kTrQ = kPf + 2;
constexpr int vrow_slot(int j) { return j < kPf ? 0 : 2 * (j - kPf); }
constexpr int krow_slot(int j) { return 16 + 2 * (j - kPf); }
constexpr int ktr_slot(int j) { return 32 + 2 * (j - kPf); }

// A block as 8 KB of dual line tile (tile_io.h) with 4 row blocks per d half:
// 1 KB block 4 dh + row / 8.
struct BlockDma {
  uint32_t ko[4], vo[4];    // per-lane byte offsets of the 8-row blocks
  const bf16 *kt, *vt;      // first rows of the K block (its last 16 keys) and V block being
                            // fetched, and of the K block whose first 16 keys are
  const bf16* ka;
  uint32_t kdst, vdst, kadst;  // LDS byte addresses of their places

  // Rows at or past Sk are never fetched: fewer than 32 keys re-read the last
  // one, more have no block that reaches past them (row_of in the dense kernel),
  // or one that re-reads its own last row (end_k, end_v in the sparse one).
  __device__ __forceinline__ void setup(int64_t ks1, int64_t vs1, int Sk, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = min(8 * i + (lane >> 3), Sk - 1), col = 8 * dual_chunk(lane, i & 1);
      ko[i] = (uint32_t)(r * ks1 + col) * 2u;
      vo[i] = (uint32_t)(r * vs1 + col) * 2u;
    }
  }
  // From now on the rows past `last` re-read it: min(r, last) rows are the smaller
  // of the two offsets, as no stride is negative. Of K the 8-row blocks I .. I + 1
  // (0: issue_ka's, 2: issue_kb's). (Opaque: the loop around has no registers for
  // what does not change in it.)
  template <int I>
  __device__ __forceinline__ void end_k(int64_t ks1, int last, int lane) {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int i = I; i < I + 2; ++i) ko[i] = min(ko[i], (uint32_t)(last * ks1 + 8 * dual_chunk(lane, i & 1)) * 2u);
  }
  __device__ __forceinline__ void end_v(int64_t vs1, int last, int lane) {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int i = 0; i < 4; ++i) vo[i] = min(vo[i], (uint32_t)(last * vs1 + 8 * dual_chunk(lane, i & 1)) * 2u);
  }
  template <int i>
  __device__ __forceinline__ void issue_k() const {
    dma16_sva_off<128 * (i >> 2), 1024 * i>(kt, ko[i & 3], kdst);
  }
  // Instruction i (0-3) of the first 16 keys of the block at ka; of the last
  // 16 of the block at kt.
  template <int i>
  __device__ __forceinline__ void issue_ka() const {
    constexpr int m = (i & 1) + 4 * (i >> 1);
    dma16_sva_off<128 * (m >> 2), 1024 * m>(ka, ko[m & 3], kadst);
  }
  template <int i>
  __device__ __forceinline__ void issue_kb() const {
    this->template issue_k<2 + (i & 1) + 4 * (i >> 1)>();
  }
  template <int i>
  __device__ __forceinline__ void issue_v() const {
    dma16_sva_off<128 * (i >> 2), 1024 * i>(vt, vo[i & 3], vdst);
  }
  __device__ __forceinline__ void all_k() const {
    static_for<0, 8>([&](auto I) { this->template issue_k<decltype(I)::value>(); });
  }
  __device__ __forceinline__ void all_v() const {
    static_for<0, 8>([&](auto I) { this->template issue_v<decltype(I)::value>(); });
  }
};

struct DqWave {
  bf16x8 qop[2][8], dop[2][8];  // Q^T (AGPRs) / dO^T (qb, kk): [query 32 qb + li][16 kk + 8 hh + ..]
  f32x16 dq[4][2];              // dQ^T (dt, qb): d = 32 dt + rows, query 32 qb + li; AGPRs
  f32x16 s[2][2], dp[2][2];     // S^T, dP^T - D (buffer, qb): keys of the block, query 32 qb + li
  bf16x8 zb[2][2];              // dZ^T (c, qb): keys 16 c + .. in accumulator order
  float lse2[2];                // lse * log2(e) of query 32 qb + li
  f32x16 nd[2];                 // its -D in every element: where dP^T - D starts
  float c;
  int li, hh;
  uint32_t krd[4], vrd[4];      // LDS byte addresses of the next block's K / V row operands
  uint32_t ktr[4];              // ... of this block's K transposed operands
  // With SUMS: sums of this lane's rounded dZ of query 32 qb + li, in AGPRs (every
  // element). Nothing of another lane is in them: what a product over more lanes
  // multiplies by 0 is NaN where a query's dZ are. And the squares of an eighth of
  // the blocks' dZ; lane l: those of the blocks of group l.
  f32x4 zsum[2];
  float zsq, weight;

  template <int j>
  __device__ __forceinline__ bf16x8 k_row() const {
    return lds_ld16(krd[j & 3] + 4096u * (j >> 2));
  }
  template <int j>
  __device__ __forceinline__ bf16x8 v_row() const {
    return lds_ld16(vrd[j & 3] + 4096u * (j >> 2));
  }
  // K^T operand j = 4 c + dt.
  template <int j>
  __device__ __forceinline__ bf16x8 k_tr() const {
    constexpr int c4 = j >> 2, dt = j & 3;
    constexpr uint32_t off = 4096u * (dt >> 1) + 2048u * c4;
    const s16x4 lo = lds_ld8_tr(ktr[2 * (dt & 1)] + off);
    const s16x4 hi = lds_ld8_tr(ktr[2 * (dt & 1) + 1] + off + 1024u);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // Move the read bases on by `dk`, `dv` bytes (the next places of the rings).
  __device__ __forceinline__ void advance_rows(uint32_t dk, uint32_t dv) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      krd[i] += dk;
      vrd[i] += dv;
      asm volatile("" : "+v"(krd[i]), "+v"(vrd[i]));
    }
  }
  __device__ __forceinline__ void advance_tr(uint32_t dk) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ktr[i] += dk;
      asm volatile("" : "+v"(ktr[i]));
    }
  }

  // MFMA g (0-31) of dP^T - D and S^T into buffer B.
  template <int B, int g>
  __device__ __forceinline__ void x_mfma(bf16x8 a) {
    constexpr int kk = (g & 15) >> 1, qb = g & 1;
    if constexpr (g < 16) dp[B][qb] = mfma32(a, dop[qb][kk], kk == 0 ? nd[qb] : dp[B][qb]);
    else s[B][qb] = mfma32(a, qop[qb][kk], kk == 0 ? f32x16{} : s[B][qb]);
  }

  // Scores of keys outside [lo, Sk) (block at key row kb) to -inf: dZ = 0.
  template <int B>
  __device__ __forceinline__ void mask(int kb, int lo, int Sk) {
#pragma unroll
    for (int qb = 0; qb < 2; ++qb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kb + 8 * (r >> 2) + 4 * hh + (r & 3);
        if (key < lo || key >= Sk) s[B][qb][r] = -INFINITY;
      }
  }

  // S^T and dP^T - D of the wave's first block (no other work).
  template <int B>
  __device__ __forceinline__ void first() {
    bf16x8 rq[kRowQ];
    static_for<0, 32>([&](auto G) {
      constexpr int g = decltype(G)::value;
      static_for<0, 8>([&](auto J) {
        constexpr int j = decltype(J)::value;
        if constexpr (vrow_slot(j) == g) rq[j % kRowQ] = this->template v_row<j>();
        if constexpr (krow_slot(j) == g) rq[(8 + j) % kRowQ] = this->template k_row<j>();
      });
      this->template x_mfma<B, g>(rq[(g >> 1) % kRowQ]);
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // Block j: dZ^T and dQ^T of block j (its S^T, dP^T - D in buffer SB) and,
  // with NEXT, those of block j+1 into the other buffer. SUMS: sums of dZ too,
  // the block one of `group`.
  template <int SB, bool NEXT, bool SUMS = false>
  __device__ __forceinline__ void block(bool mask_next, int kb_next, int lo_next, int Sk,
                                        const BlockDma& dma, int group = 0) {
    constexpr int NB = 1 - SB;
    bf16x8 rq[kRowQ], tq[kTrQ];
    float fa[2][2], fe[2][2];
    u32x2 ones;
    static_for<0, 48>([&](auto G) {
      constexpr int g = decltype(G)::value;
      if constexpr (NEXT && g == krow_slot(0)) wait_vm<16>();  // K of block j+1
      static_for<0, 8>([&](auto J) {
        constexpr int j = decltype(J)::value;
        if constexpr (NEXT && vrow_slot(j) == g) rq[j % kRowQ] = this->template v_row<j>();
        if constexpr (NEXT && krow_slot(j) == g) rq[(8 + j) % kRowQ] = this->template k_row<j>();
        if constexpr (ktr_slot(j) == g) tq[j % kTrQ] = this->template k_tr<j>();
      });
      if constexpr (g < 32) {
        if constexpr (NEXT) {
          this->template x_mfma<NB, g>(rq[(g >> 1) % kRowQ]);
          // Anchored in its slot: left alone, the compiler moves these MFMAs
          // down to where mask and the next block read them, all in a row
          // behind the VALU work that they are meant to cover (backward at
          // 512 x 4096 keys 84 -> 76 us, 2048 tokens 117-119 -> 112-116).
          f32x16& acc = g < 16 ? dp[NB][g & 1] : s[NB][g & 1];
          asm volatile("" : "+v"(acc));
        }
      } else {
        constexpr int op = g - 32, j = op >> 1;
        mfma_acc(dq[j & 3][op & 1], tq[j % kTrQ], zb[j >> 2][op & 1]);
      }
      static_for<0, 16>([&](auto U) {
        constexpr int u = decltype(U)::value;
        constexpr int cz = u >> 3, qb = (u >> 2) & 1, jp = u & 3, r = 8 * cz + 2 * jp;
        if constexpr (unit_slot(u) == g) {
          fa[u & 1][0] = fmaf(s[SB][qb][r], c, -lse2[qb]);
          fa[u & 1][1] = fmaf(s[SB][qb][r + 1], c, -lse2[qb]);
          asm volatile("" : "+v"(fa[u & 1][0]), "+v"(fa[u & 1][1]));
        }
        if constexpr (unit_slot(u) + 1 == g) {
          fe[u & 1][0] = fast_exp2(fa[u & 1][0]);
          fe[u & 1][1] = fast_exp2(fa[u & 1][1]);
          asm volatile("" : "+v"(fe[u & 1][0]), "+v"(fe[u & 1][1]));
        }
        if constexpr (unit_slot(u) + 2 == g) {
          const float z0 = fe[u & 1][0] * dp[SB][qb][r], z1 = fe[u & 1][1] * dp[SB][qb][r + 1];
          zb[cz][qb][2 * jp] = (bf16)z0;
          zb[cz][qb][2 * jp + 1] = (bf16)z1;
          if constexpr (SUMS && qb == 0 && (jp & 1)) zsq = fmaf(z1, z1, zsq);
          asm volatile("" : "+v"(zb[cz][qb]));
        }
      });
      // (From slot 39 on there are registers: the scores are used up.)
      if constexpr (SUMS && g == 39) {
        ones = u32x2{0x3f803f80u, 0x3f803f80u};
        asm volatile("" : "+v"(ones));
      }
      // (Even slots: the odd ones have a DMA.)
      if constexpr (SUMS && g >= 40 && (g & 1) == 0) {
        constexpr int s = (g - 40) >> 1;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const bf16x8& z = zb[s >> 1][qb];
          mfma_sum(zsum[qb], ones, (s & 1) ? __builtin_shufflevector(z, z, 4, 5, 6, 7) : __builtin_shufflevector(z, z, 0, 1, 2, 3));
        }
      }
      // The wave's sum of squares, of two blocks (or of the first one), one step a slot, to the group's
      // lane. A lane's that is not finite does not count.
      if constexpr (SUMS && SB == 0 && g == 39) zsq = zsq < INFINITY ? zsq : 0.f;
      if constexpr (SUMS && SB == 0 && g >= 40 && g < 46) {
        constexpr int step[6] = {0x111, 0x112, 0x114, 0x118, 0x142, 0x143};  // row_shr 1, 2, 4, 8; row_bcast 15, 31
        zsq += __builtin_bit_cast(
            float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, zsq), step[(g - 40) % 6], 0xf, 0xf, false));
        asm volatile("" : "+v"(zsq));
      }
      if constexpr (SUMS && SB == 0 && g == 46) {
        const float all = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, zsq), 63));
        weight += li + 32 * hh == group ? all : 0.f;
        zsq = 0.f;
        asm volatile("" : "+v"(weight), "+v"(zsq));
      }
      if constexpr (NEXT && g == 40) {
        if (mask_next) mask<NB>(kb_next, lo_next, Sk);
      }
      if constexpr (NEXT && (g & 1)) {
        if constexpr (g < 8) dma.template issue_kb<(g >> 1)>();
        if constexpr (g >= 16 && g < 32) dma.template issue_v<((g - 16) >> 1)>();
        if constexpr (g >= 40) dma.template issue_ka<((g - 40) >> 1)>();
      }
      // The operands of the previous slot's inline-asm MFMA stay allocated to
      // the end of this slot: the compiler does not see it still reading them.
      if constexpr (g > 32) {
        constexpr int op = g - 33;
        keep_alive(tq[(op >> 1) % kTrQ]);
        keep_alive(zb[op >> 3][op & 1]);
        if constexpr (SUMS && g > 40 && (g & 1)) {
          keep_alive(zb[(g - 41) >> 2][0]);
          keep_alive(zb[(g - 41) >> 2][1]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    keep_alive(tq[7 % kTrQ]);
    keep_alive(zb[1][1]);
    if constexpr (SUMS) asm volatile("" ::"v"(ones));
  }
};

}  // namespace dqks
}  // namespace bwd
}  // namespace aa
