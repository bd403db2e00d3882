// K/V tiles of one wave's own (attn_fwd_ks.hip: each wave of a workgroup takes
// key tiles of its own; sparse_fwd.hip: each wave is a workgroup): a 64-key K
// tile and V tile in 32 KB of LDS, streamed into the place of the tile before
// without a barrier, a quarter (4 KB, 4 DMA instructions) as soon as its last
// operand has been read:
//   slots  8-15, 16-23, 24-31, 32-39: K quarters 0-3 of tile t+2 (quarter
//     2 kb + dh = keys 32 kb .., head-dim half dh, read in slots 8 q .. 8 q + 7)
//   slots 40-47, 48-55, 56-63 and 0-7 of tile t+1: V key chunks 0-3 of tile
//     t+1 (chunk c, read in slots 32 + 8 c .. 32 + 8 c + 7)
// one instruction in every odd slot, 32 per tile. Every quarter then has
// about 56 slots (2000 cycles) to arrive, and a wait for "all but the 22
// youngest" (24 at slot 0) ahead of each quarter's first read covers exactly
// the loads up to it.
#pragma once

#include "attn_fwd_wave.h"

namespace aa {
namespace ks {

template <int n>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}

// One wave's K/V DMA (the hooks of FwdWave::tile).
struct WaveDma {
  // S^T held in its slots: left alone, the compiler moved these MFMAs of a
  // tile down to the mask's branch, all 32 in a row behind the VALU work that
  // they are meant to cover (when added, 1024 tokens 15.1 -> 14.3 us, 512 11.0
  // -> 10.5; with the plain last tile below 14.1 and 10.1).
  static constexpr bool kAnchorS = true;
  const bf16 *kp, *vp;      // the (batch, head)'s K and V
  int64_t ks1, vs1;         // token strides
  uint32_t ko[8], vo[8];    // per-lane byte offsets of the tile's 8-row blocks
  uint32_t lds;             // LDS byte address of the wave's K tile
  const bf16 *kt, *vt, *v3; // first rows of the K tile and V tile (chunks 0-2; 3) being fetched

  // Rows at or past klen are never fetched (V may hold anything there, and 0
  // times a NaN is one): the wave's last tile re-reads its last row past it
  // (rows_k, rows_v from their first fetch on; what follows is that tile again).
  __device__ __forceinline__ void setup(const bf16* k, const bf16* v, int64_t ks1_, int64_t vs1_, int lane,
                                        uint32_t lds_) {
    kp = k;
    vp = v;
    ks1 = ks1_;
    vs1 = vs1_;
    rows_k(lane, kBN - 1);
    rows_v<0, 8>(lane, kBN - 1);
    lds = lds_;
  }
  // Row offsets of a tile whose rows past `last` re-read it (V: blocks I .. E - 1).
  __device__ __forceinline__ void rows_k(int lane, int last) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      ko[i] = (uint32_t)(min(8 * i + (lane >> 3), last) * ks1 + 8 * line_k_chunk(lane, i & 1)) * 2u;
  }
  template <int I, int E>
  __device__ __forceinline__ void rows_v(int lane, int last) {
#pragma unroll
    for (int i = I; i < E; ++i)
      vo[i] = (uint32_t)(min(8 * i + (lane >> 3), last) * vs1 + 8 * line_v_chunk(lane)) * 2u;
  }

  // Instruction i (0-3) of K quarter q / V chunk c: 8 rows x 64 d into the
  // line tile's block 8 dh + row / 8.
  template <int q, int i>
  __device__ __forceinline__ void issue_k() const {
    constexpr int kb = q >> 1, dh = q & 1, blk = 4 * kb + i;
    dma16_sva_off<128 * dh, (8 * dh + blk) * 1024>(kt, ko[blk], lds);
  }
  template <int c, int i>
  __device__ __forceinline__ void issue_v() const {
    constexpr int dh = i >> 1, blk = 2 * c + (i & 1);
    dma16_sva_off<128 * dh, kVOff + (8 * dh + blk) * 1024>(c == 3 ? v3 : vt, vo[blk], lds);
  }

  template <int B, class W>
  __device__ __forceinline__ void mask(W& w, int kb, int klen) const { w.template mask<B>(kb, klen); }
  template <int g>
  __device__ __forceinline__ void first_slot() const {
    constexpr int q = (g >> 3) - 1, i = (g & 7) >> 1;
    if constexpr (q >= 0 && (g & 1)) issue_k<q, i>();
  }
  template <int g, bool NEXT>
  __device__ __forceinline__ void before_slot() const {
    if constexpr (NEXT) {
      if constexpr (g == 0) wait_vm<24>();
      if constexpr (g == 4 || g == 12 || g == 20 || g == 28 || g == 36 || g == 44 || g == 52)
        wait_vm<22>();
    } else {
      // The last tile: only V chunk 3 of this tile went out in its slots.
      if constexpr (g == 28) wait_vm<12>();
      if constexpr (g == 36) wait_vm<8>();
      if constexpr (g == 44) wait_vm<4>();
      if constexpr (g == 52) wait_vm<0>();
    }
  }
  template <int g, bool NEXT>
  __device__ __forceinline__ void after_slot() const {
    if constexpr (g & 1) {
      constexpr int grp = g >> 3, i = (g & 7) >> 1;
      if constexpr (grp == 0) issue_v<3, i>();
      else if constexpr (!NEXT) return;
      else if constexpr (grp <= 4) issue_k<grp - 1, i>();
      else issue_v<grp - 5, i>();
    }
  }
};

}  // namespace ks
}  // namespace aa
