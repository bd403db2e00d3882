// Shared by the kernels of the attention over selected blocks (sparse_select.hip,
// sparse_fwd.hip, sparse_bwd.hip): block sizes, the launch parameters and the
// walk over a query block's list of key blocks.
//
// A query block is 64 queries of one (batch, head), a key block 64 keys of one
// (batch, key head). A list holds the key blocks that a query block attends,
// int32 [B, H, ceil(Sq / 64), count]: entries below 0 or past the last block
// with a key are no blocks, a block that is named twice is attended once.
#pragma once

#include <algorithm>

#include "tile_io.h"

namespace aa {
namespace sparse {

constexpr int kB = kTileRows;  // queries, and keys, of a block
constexpr int kD = 128;
// One 64-bit word of blocks for each lane of a wave.
constexpr int64_t kMaxBlocks = 64 * 64;
constexpr int64_t kMaxCount = kMaxBlocks;

struct SparseParams {
  const bf16 *q, *k, *v;
  bf16* o;
  float* lse;               // [B, H, Sq] or null
  const int32_t* seqused;   // [B] or null
  const int32_t* blocks;
  int64_t qs[3], ks[3], vs[3], os[3];
  int H, group, Sq, Sk, nq, count, items;  // group: heads of q that share a head of k
  float c;                  // softmax_scale * log2(e)
  // Split lists: workgroup (item, split) writes O (not normalised) and its row
  // statistics (max, sum of the rounded probabilities, sum of the others) of
  // the split-th part of the list, which the combine kernel merges.
  int nsplit;
  float* part_o;            // [items][nsplit][64][128]
  f32x4* part_stat;         // [items][nsplit][64]
};

__device__ __forceinline__ int key_length(const int32_t* seqused, int b, int Sk) {
  return seqused ? max(0, min((int)seqused[b], Sk)) : Sk;
}

// Workgroup -> item: a contiguous range of the items on each XCD (tile_io.h's
// xcd_remap for any number of items; the grid is a multiple of 8 long). -1: none.
__device__ __forceinline__ int item_of(int block, int grid, int items) {
  const int i = (block & 7) * (grid >> 3) + (block >> 3);
  return i < items ? i : -1;
}
inline unsigned grid_of(int64_t items) { return (unsigned)((items + 7) / 8 * 8); }

// The distinct blocks of one list in ascending order. Lane l holds the blocks
// 64 l .. 64 l + 63 as bits; the walk itself is scalar work.
struct BlockWalk {
  uint64_t mine;   // this lane's blocks
  uint64_t lanes;  // lanes with blocks still to come
  uint64_t word;   // what is left of the current lane's
  int base, n;     // its first block; blocks in all

  // From a list of `count` entries, blocks below `have`; bits: 512 bytes of LDS
  // of this wave's own.
  __device__ __forceinline__ void read(const int32_t* list, int count, int have, uint32_t* bits, int lane) {
    bits[lane] = 0;
    bits[64 + lane] = 0;
    __syncthreads();
    for (int i = lane; i < count; i += 64) {
      const int x = list[i];
      if (x >= 0 && x < have) atomicOr(bits + (x >> 5), 1u << (x & 31));
    }
    __syncthreads();
    mine = (uint64_t)bits[2 * lane] | ((uint64_t)bits[2 * lane + 1] << 32);
    __syncthreads();
  }
  __device__ __forceinline__ void start() {
    int sum = __popcll(mine);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    n = __builtin_amdgcn_readfirstlane(sum);
    lanes = __builtin_amdgcn_ballot_w64(mine != 0);
    word = 0;
    base = 0;
  }
  // Keeps the blocks of rank n s / parts .. n (s + 1) / parts - 1.
  __device__ __forceinline__ void part(int s, int parts, int lane) {
    const int c = __popcll(mine);
    int before = c;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int up = __shfl_up(before, off);
      if (lane >= off) before += up;
    }
    const int all = __shfl(before, 63);
    before -= c;
    const int r0 = (int)((int64_t)all * s / parts), r1 = (int)((int64_t)all * (s + 1) / parts);
    int drop = min(max(r0 - before, 0), c);
    int keep = min(max(r1 - max(before, r0), 0), c - drop);
    for (; drop > 0; --drop) mine &= mine - 1;
    uint64_t kept = 0;
    for (; keep > 0; --keep) {
      kept |= mine & -mine;
      mine &= mine - 1;
    }
    mine = kept;
  }
  // The next block; only while there is one.
  __device__ __forceinline__ int next() {
    if (word == 0) {
      const int l = __builtin_ctzll(lanes);
      lanes &= lanes - 1;
      const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)mine, l);
      const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(mine >> 32), l);
      word = (uint64_t)lo | ((uint64_t)hi << 32);
      base = 64 * l;
    }
    const int x = base + __builtin_ctzll(word);
    word &= word - 1;
    return x;
  }
};

// Parts of a list: as many as give every SIMD a wave, of equal numbers of blocks;
// none where that takes fewer than 4 blocks (about 2 us each) off the longest
// part: the second launch costs as much.
inline int plan_split(int64_t items, int64_t count) {
  const int64_t slots = 4 * (int64_t)device_cu_count();
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(items ? slots / items : 1, count));
  const int64_t longest = (count + parts - 1) / parts;
  return count - longest < 4 ? 1 : (int)((count + longest - 1) / longest);
}

// What the backward launches: a wave per block of queries (dQ), a workgroup of 256
// threads per 64 of them and per 4 blocks of keys (turned lists, mean keys), and
// one per block of keys (dK, dV). A forward that keeps statistics is held to it.
constexpr int64_t kTurnThreads = 256, kKvThreads = 256;
inline int64_t turn_lists(int64_t B, int64_t H, int64_t nq) { return B * H * ((nq + 63) / 64); }
inline int64_t turn_means(int64_t kitems) { return (kitems + kTurnThreads / 64 - 1) / (kTurnThreads / 64); }
inline bool backward_fits(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk) {
  const int64_t nq = (Sq + kB - 1) / kB, nk = (Sk + kB - 1) / kB;
  if ((nq && B * H > 0x1fffff0 / nq) || (nk && B * Hk > 0x1fffff0 / nk)) return false;
  return grid_fits(turn_lists(B, H, nq) + turn_means(B * Hk * nk), kTurnThreads) &&
         grid_fits(grid_of(B * Hk * nk), kKvThreads);
}

}  // namespace sparse
}  // namespace aa
