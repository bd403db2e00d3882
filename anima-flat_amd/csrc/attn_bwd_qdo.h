// What the dK/dV kernels with one wave per SIMD share (attn_bwd_dkdv.hip: 128
// keys of one head and every query tile; sparse_bwd.hip: one block of 64 keys
// and the query blocks that list it): the LDS stage of one query tile, its DMA
// and the accumulating MFMA.
#pragma once

#include "attn_bwd.h"

namespace aa {
namespace bwd {
namespace w1 {

constexpr uint32_t kTileBytes = kTileElems * 2;  // one 64 x 128 bf16 tile
constexpr uint32_t kStageBytes = 2 * kTileBytes; // Q tile, then dO tile
constexpr uint32_t kDoOff = kTileBytes;
constexpr uint32_t kStatBytes = kStat * 4;
constexpr uint32_t kNegDOff = kT * 4;            // -D in a stats record (bytes)

// DMA of one wave's quarter of the Q and dO dual line tiles of a query tile
// (tile_io.h): blocks 4 g .. 4 g + 3 (g = wave) = d-half g >> 1, rows
// 32 (g & 1) + 8 i + (lane >> 3). A job takes one scalar base per tensor (the
// tile's first row) and per-lane 32-bit byte offsets holding each lane's row
// and column. Rows at or past Sq re-read row Sq - 1 (their stats give P = 0
// and dZ = 0). Wave 0 also moves the tile's stats record (1 KB).
struct QdoDma {
  uint32_t qo[4], oo[4];  // per-lane offsets of blocks 0-3 (rows inside Sq unless `clamped`)
  bool clamped;
  const bf16* qb;
  const bf16* ob;
  const float* sb;  // the stats record
  uint32_t dst;     // LDS byte address of this wave's first Q block
  uint32_t sdst;    // LDS byte address of the stats record

  __device__ __forceinline__ static int row_of(int g, int i, int lane) {
    return 32 * (g & 1) + 8 * i + (lane >> 3);
  }
  __device__ __forceinline__ static int col(int g, int i, int lane) {
    return 64 * (g >> 1) + 8 * dual_chunk(lane, i & 1);
  }
  __device__ __forceinline__ void fixed(const Params& p, int g, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row_of(g, i, lane);
      qo[i] = (uint32_t)(r * p.s_q[1] + col(g, i, lane)) * 2u;
      oo[i] = (uint32_t)(r * p.s_do[1] + col(g, i, lane)) * 2u;
    }
    clamped = false;
  }
  // The job of the tile whose first query row is q0 (< Sq), into the ring
  // stage at byte address `stage`, stats record srec into LDS at sdst_.
  __device__ __forceinline__ void prepare(const Params& p, int q0, uint32_t stage, uint32_t sdst_,
                                          const float* srec, int g, const bf16* qbase,
                                          const bf16* obase, int lane) {
    dst = stage + (uint32_t)(4 * g) * 1024u;
    sdst = sdst_;
    sb = srec;
    if (q0 + kT <= p.Sq) {
      qb = qbase + (int64_t)q0 * p.s_q[1];
      ob = obase + (int64_t)q0 * p.s_do[1];
      if (clamped) fixed(p, g, lane);
    } else {
      const int last = p.Sq - 1;
      qb = qbase + (int64_t)q0 * p.s_q[1];
      ob = obase + (int64_t)q0 * p.s_do[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = min(q0 + row_of(g, i, lane), last) - q0;
        qo[i] = (uint32_t)(r * p.s_q[1] + col(g, i, lane)) * 2u;
        oo[i] = (uint32_t)(r * p.s_do[1] + col(g, i, lane)) * 2u;
      }
      clamped = true;
    }
  }
  // DMA instruction i of the job: 0-3 the Q blocks, 4-7 the dO blocks.
  template <int i>
  __device__ __forceinline__ void issue() const {
    constexpr uint32_t off = (i < 4 ? 0u : kDoOff) + (uint32_t)(i & 3) * 1024u;
    if constexpr (i < 4) dma16_sva(qb, qo[i & 3], dst + off);
    else dma16_sva(ob, oo[i & 3], dst + off);
  }
  __device__ __forceinline__ void issue_stats(int lane) const {
    dma16_sva(sb, 16u * (uint32_t)lane, sdst);
  }
};

// dV^T / dK^T += A B on AGPR accumulators (inline asm: the builtin would
// follow the function-wide VGPR accumulator form). The accumulators are only
// read by VALU code behind fence_acc(); the A / B operands are read when the
// MFMA issues.
__device__ __forceinline__ void mfma_acc(f32x16& acc, bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void keep_alive(bf16x8 v) { asm volatile("" ::"v"(v)); }

__device__ __forceinline__ f32x4 lds_ld16f(uint32_t addr) {
  return __builtin_bit_cast(f32x4, lds_ld16(addr));
}

}  // namespace w1
}  // namespace bwd
}  // namespace aa
