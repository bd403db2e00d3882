// Backward of the attention over selected blocks, head_dim 128 (gfx950), the
// softmax recomputed from the forward's log-sum-exp. Deterministic: every sum
// in a fixed order, no atomics on floats.
//
//   P = exp(S - lse), dP = dO V^T, D = rowsum(dO o O), dZ = P o (dP - D),
//   dQ = scale dZ K, dK = scale dZ^T Q, dV = P^T dO   over the listed blocks.
//
//   sparse_dq_kernel    one wave is one workgroup and one block of 64 queries
//                       over its list, with DqWave's slot schedule
//                       (attn_bwd_dq_wave.h); it also writes the statistics
//                       record (lse, D) of its queries
//   sparse_turn_kernel  the lists turned round: for each block of keys a bit per
//                       block of queries that names it; and its mean key
//   sparse_dkdv_kernel  one workgroup of 4 waves per block of 64 keys of one key
//                       head, over the query blocks of all heads that share it
//   sparse_sum_kernel   where few blocks would leave SIMDs or CUs idle, their
//                       lists are split and the parts' fp32 sums added up here
#include <type_traits>

#include "attn_bwd_dq_wave.h"
#include "attn_bwd_qdo.h"
#include "sparse.h"

namespace aa {
namespace sparse {

struct BwdParams {
  bwd::Params a;           // tensors, strides, statistics [B][H][nq][kStat]; ntq = nq, ntk = nk
  const int32_t* seqused;
  const int32_t* blocks;
  uint64_t* turned;        // [B][H][nk][nqw]: bit i of word w: query block 64 w + i lists the key block
  int group, count, nqw, items, kitems;
  // Parts of a query block's list (dQ) and of a key block's (dK, dV); with more
  // than one, sparse_sum_kernel adds up the parts' 32 x 32 accumulators in fp32.
  int qparts, kparts;
  f32x4* sums;             // [item][part][tile][4][64]
  float* means;            // [B][Hk][nk][128]: mean key of each block
  float* recs;             // [item][part][kRec]: what a dQ part's correction needs
};
// A part's record: the sum of dZ of each query, then the weighted sum of the
// mean keys and that of the weights.
constexpr int kRecMean = kB, kRecWeight = kB + kD, kRec = 256;
constexpr int kQTiles = 8, kKTiles = 16;  // accumulators of a dQ item; of a dK / dV item

// Accumulator tile of 32 rows x 32 head dims, as the MFMA holds it.
__device__ __forceinline__ void store_tile(f32x4* to, const f32x16& acc, int lane) {
#pragma unroll
  for (int rq = 0; rq < 4; ++rq)
    __builtin_nontemporal_store(f32x4{acc[4 * rq], acc[4 * rq + 1], acc[4 * rq + 2], acc[4 * rq + 3]}, to + rq * 64 + lane);
}

// Mean key of weighted mean keys: 0 where nothing or nothing finite is known.
__device__ __forceinline__ float mean_of(float sum, float weight) {
  const float m = sum / weight;
  return fabsf(m) < INFINITY ? m : 0.f;
}

// ---------------------------------------------------------------------- dQ --
//
// A query's dZ sum to 0 over its keys, but those that the MFMAs take do not
// quite: each is rounded to bf16, and D is that of the rounded O. What stands out
// of those errors in dQ is their sum times what the keys have in common: for
// normed keys whose neighbours are alike dQ was 3.3e-3 to 4.6e-3 of its norm off,
// where one rounding is 1.7e-3. So the kernel sums the rounded dZ (eight MFMAs of 4
// x 4 x 4, whose sums are a lane's own, in a half's last slots; v_dot2 of pairs
// took twice their time) and takes sum x mean key off at the end: 2.4e-3, two roundings. The mean is that of the
// listed blocks, weighted by a sample of their own squares of dZ, as it is there that the
// errors come from (unweighted 2.6e-3, the first block's 3.2e-3); any would be
// right, as the exact sum is 0. (Of lists of more than 64 blocks, blocks 64 apart
// have one weight, of both: 2.44e-3 at 256 blocks, where 64 have 2.37e-3.) It costs 3 to 4% of the backward, most of it in the
// loop (forward and backward at 4096 tokens x 16 blocks 193 -> 197 us, 9216 x 24
// 632 -> 650).
//
// What bounds the loop is one wave's issue: 420 instructions in a half's 48 slots
// (MFMA busy in half of the cycles), 1.43 us a half in a full CU. Beside it stands
// what a round of lists does together, start and end (4096 tokens x 16 heads x 16 blocks:
// 19 of 63 us), and a last round that is not full (9216 x 24: 2.25 rounds, 235 us).

__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void sparse_dq_kernel(BwdParams sp) {
  using namespace bwd::dqks;
  using sparse::kD;
  const bwd::Params& p = sp.a;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaveBytes];

  int item = item_of(blockIdx.x, gridDim.x, sp.items * sp.qparts);
  if (item < 0) return;
  const int whole = item;
  const int part = item % sp.qparts;
  item /= sp.qparts;
  const int qblk = item % p.ntq;
  const int bh = item / p.ntq;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / sp.group;
  const int lane = threadIdx.x;
  const int li = lane & 31, hh = lane >> 5;
  const int qrow0 = qblk * kB;
  const int klen = key_length(sp.seqused, b, p.Sk);

  // Three waits stand before the first MFMA, and all waves of a round wait
  // together: for the list with Q, dO, O and the log-sum-exp; for the first two
  // halves of K and V; and for nothing else. dO and O come straight into the
  // registers' layout (32 rows an instruction, 1 us for a CU's four waves), Q
  // through LDS (areas of 32 rows, tile_io.h) into places that the list's
  // bits, in the first K place, leave free.
  auto area = [&](uint32_t off) { return reinterpret_cast<bf16*>(lds + off); };
  const bf16* qp = p.q + b * p.s_q[0] + h * p.s_q[2];
  bf16* aq[2] = {area(kBlock), area(2 * kBlock)};
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) stage_rows_in(qp, p.s_q[1], qrow0 + 32 * qb, p.Sq, lane, aq[qb]);
  DqWave w;
  u32x4 orow[2][8];
  float lse[2];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = min(qrow0 + 32 * qb + li, p.Sq - 1);
    const bf16* dop = p.dout + b * p.s_do[0] + h * p.s_do[2] + (int64_t)q * p.s_do[1] + 8 * hh;
    const bf16* op = p.o + b * p.s_o[0] + h * p.s_o[2] + (int64_t)q * p.s_o[1] + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      w.dop[qb][kk] = __builtin_bit_cast(bf16x8, ld16(dop + 16 * kk));
      orow[qb][kk] = ld16(op + 16 * kk);
    }
    lse[qb] = p.lse[(int64_t)bh * p.Sq + q];
  }
  BlockWalk walk;
  walk.read(sp.blocks + (int64_t)item * sp.count, sp.count, (klen + kB - 1) / kB, reinterpret_cast<uint32_t*>(lds), lane);
  if (sp.qparts > 1) walk.part(part, sp.qparts, lane);
  walk.start();
  // Halves of 32 keys; the last one may hold none, and the one before it then
  // comes first: a block's two halves stay a pair that ends in buffer 0.
  const int nblk = walk.n;
  int n = 2 * nblk;
  if (nblk > 0 && klen % kB != 0 && klen % kB <= kKeys) {
    // The list's highest block is the one that klen ends in?
    const uint64_t has = __builtin_amdgcn_ballot_w64(walk.mine >> ((klen / kB) & 63) & 1);
    if (has >> ((klen / kB) >> 6) & 1) --n;
  }

  // First keys of the halves i + 1, i + 2, i + 3; past the list its last half
  // again, into places that nothing reads. In the half that klen ends in, which
  // comes last or, alone of its block, first, the rows from klen on re-read the one
  // before it, masked. (Moved back to end at klen, as in the dense kernel, the half
  // would read keys of the block before, which the list need not name: a NaN there
  // spoilt dQ.)
  int blk = 0, half = 0, left = n, lo = 0;
  auto next_half = [&]() {
    if (left > 0) {
      if (half == 0) blk = walk.next();
      lo = blk * kB + half * kKeys;
      half ^= 1;
      --left;
    }
    return lo;
  };
  const bf16* kp = p.k + b * p.s_k[0] + hk * p.s_k[2];
  const bf16* vp = p.v + b * p.s_v[0] + hk * p.s_v[2];
  const uint32_t mine = lds_addr(lds);
  BlockDma dma;
  dma.setup(p.s_k[1], p.s_v[1], kKeys, lane);
  auto k_job = [&](int i, int first) {  // its last 16 keys; the others' rows are ka_job's
    dma.kt = kp + (int64_t)first * p.s_k[1];
    dma.kdst = mine + (uint32_t)(i % 3) * kBlock;
    if (first + kKeys > klen) dma.end_k<2>(p.s_k[1], klen - 1 - first, lane);
  };
  auto ka_job = [&](int i, int first) {
    dma.ka = kp + (int64_t)first * p.s_k[1];
    dma.kadst = mine + (uint32_t)(i % 3) * kBlock;
    if (first + kKeys > klen) dma.end_k<0>(p.s_k[1], klen - 1 - first, lane);
  };
  auto v_job = [&](int i, int first) {
    dma.vt = vp + (int64_t)first * p.s_v[1];
    dma.vdst = mine + kVRing + (uint32_t)(i & 1) * kBlock;
    if (first + kKeys > klen) dma.end_v(p.s_v[1], klen - 1 - first, lane);
  };
  const bool single = n & 1;
  if (single) {
    lo = klen / kB * kB;
    --left;
  }
  const int l0 = single ? lo : next_half();
  int l1 = next_half(), l2 = next_half(), l3 = 0;
  wait_dma();
  w.li = li;
  w.hh = hh;
  w.c = p.c;
  w.zsum[0] = w.zsum[1] = f32x4{};
  asm volatile("" : "+a"(w.zsum[0]), "+a"(w.zsum[1]));
  w.zsq = w.weight = 0.f;
#pragma unroll
  for (int qb = 0; qb < 2; ++qb)
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      w.qop[qb][kk] = staged_operand(aq[qb], lane, kk);
      asm volatile("" : "+a"(w.qop[qb][kk]));
    }
  // Statistics of each query: lse2 = lse log2(e) and -D, D = rowsum(dO o O) (this
  // lane's 64 values, then the partner lane's half). Queries past Sq, and those
  // that attended nothing: lse2 = +inf, so that P = 0.
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = qrow0 + 32 * qb + li;
    float nd = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      float x[8], y[8];
      unpack8(orow[qb][kk], x);
      unpack8(__builtin_bit_cast(u32x4, w.dop[qb][kk]), y);
#pragma unroll
      for (int i = 0; i < 8; ++i) nd = fmaf(y[i], x[i], nd);
    }
    nd = pair_sum(nd);
    nd = q < p.Sq ? -nd : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) w.nd[qb][r] = nd;
    w.lse2[qb] = q >= p.Sq || lse[qb] == -INFINITY ? INFINITY : lse[qb] * kLog2e;
  }
  __syncthreads();  // the staged rows are read: their places are free
  if (n > 0) {
    ka_job(0, l0);
    k_job(0, l0);
    dma.all_k();
    v_job(0, l0);
    dma.all_v();
    if (single) dma.setup(p.s_k[1], p.s_v[1], kKeys, lane);
    ka_job(1, l1);
    k_job(1, l1);
    dma.all_k();
    v_job(1, l1);
    dma.all_v();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w.krd[j] = mine + 2u * (uint32_t)dual_row_rd(lane, j);
    w.vrd[j] = w.krd[j] + kVRing;
    w.ktr[j] = mine + 2u * (uint32_t)dual_tr_rd(lane, j >> 1, j & 1);
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      w.dq[dt][qb] = f32x16{};
      asm volatile("" : "+a"(w.dq[dt][qb]));
    }
  wait_vm<16>();  // K and V of the first half
  if (n > 0) {
    const int b0 = (n - 1) & 1;  // the last half's S^T is in buffer 0
    const bool m0 = l0 + kKeys > klen;
    if (b0) {
      w.first<1>();
      if (m0) w.mask<1>(l0, l0, klen);
    } else {
      w.first<0>();
      if (m0) w.mask<0>(l0, l0, klen);
    }
    v_job(2, l2);
    dma.all_v();
    ka_job(2, l2);
    static_for<0, 4>([&](auto I) { dma.template issue_ka<decltype(I)::value>(); });
    // Once as the halves' own counts do not hold yet: all but those 12, that
    // is K and V of half 1.
    wait_vm<12>();
    l3 = next_half();

    auto run = [&](auto sb, auto next, int i) {
      constexpr int SB = decltype(sb)::value;
      constexpr bool NEXT = decltype(next)::value;
      if constexpr (NEXT) {
        wait_vm<20>();  // V of half i + 1
        w.advance_rows((i + 1) % 3 == 0 ? 0u - 2u * kBlock : kBlock, (i + 1) & 1 ? kBlock : 0u - kBlock);
        k_job(i + 2, l2);
        ka_job(i + 3, l3);
        v_job(i + 3, l3);
      }
      w.block<SB, NEXT, true>(l1 + kKeys > klen, l1, l1, klen, dma, (i >> 1) & 63);
      w.advance_tr((i + 1) % 3 == 0 ? 0u - 2u * kBlock : kBlock);
      if constexpr (NEXT) {
        l1 = l2;
        l2 = l3;
        l3 = next_half();
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    int i = 0;
    if (b0) {
      run(I1{}, std::true_type{}, 0);
      i = 1;
    }
    for (; i + 1 < n; i += 2) {
      run(I0{}, std::true_type{}, i);
      run(I1{}, std::true_type{}, i + 1);
    }
    run(I0{}, std::false_type{}, i);
  }
  wait_dma();
  // The record that the dK/dV kernel reads (at the end: stores ahead of the
  // loop would be waited for with its first loads).
  if (hh == 0 && part == 0) {
    float* st = p.stats + (int64_t)item * bwd::kStat;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      st[32 * qb + li] = w.lse2[qb];
      st[kB + 32 * qb + li] = w.nd[qb][0];
    }
  }
  // Keeps dQ in AGPRs up to here and orders the reads after its MFMAs.
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
               : "+a"(w.dq[0][0]), "+a"(w.dq[1][0]), "+a"(w.dq[2][0]), "+a"(w.dq[3][0]),
                 "+a"(w.dq[0][1]), "+a"(w.dq[1][1]), "+a"(w.dq[2][1]), "+a"(w.dq[3][1]),
                 "+a"(w.zsum[0]), "+a"(w.zsum[1]));
  // The sums of dZ, of both lanes of a query (0 where they are not finite: so is
  // the query's dQ then), and the weighted sum of the mean keys, two head dims a
  // lane.
  float zsum[2], m[2] = {0.f, 0.f}, weight = 0.f;
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    zsum[qb] = pair_sum(w.zsum[qb][0]);
    if (!(fabsf(zsum[qb]) < INFINITY)) zsum[qb] = 0.f;
  }
  // (No square at all, of gradients below 1e-22 for example: the plain mean.)
  if (sp.qparts == 1 && __builtin_amdgcn_ballot_w64(w.weight > 0.f) == 0) w.weight = 1.f;
  walk.lanes = __builtin_amdgcn_ballot_w64(walk.mine != 0);
  walk.word = 0;
  const float* means = sp.means + ((int64_t)b * (p.H / sp.group) + hk) * p.ntk * kD + 2 * lane;
  for (int i0 = 0; i0 < nblk; i0 += 8) {
    float2 x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = i0 + e < nblk ? *reinterpret_cast<const float2*>(means + (int64_t)walk.next() * kD) : float2{0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // The group of the list's block i0 + e: a single half's block, its last, was first.
      const int group = !single ? i0 + e : i0 + e + 1 < nblk ? i0 + e + 1 : 0;
      const float g = i0 + e < nblk ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w.weight), group & 63)) : 0.f;
      m[0] = fmaf(g, x[e].x, m[0]);
      m[1] = fmaf(g, x[e].y, m[1]);
      weight += g;
    }
  }
  if (sp.qparts > 1) {
    f32x4* to = sp.sums + (int64_t)whole * kQTiles * 256;
    float* rec = sp.recs + (int64_t)whole * kRec;
    if (hh == 0) {
      rec[li] = zsum[0];
      rec[32 + li] = zsum[1];
    }
    *reinterpret_cast<float2*>(rec + kRecMean + 2 * lane) = float2{m[0], m[1]};
    if (lane == 0) rec[kRecWeight] = weight;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) store_tile(to + (4 * qb + dt) * 256, w.dq[dt][qb], lane);
    return;
  }
  __syncthreads();
  float* mean = reinterpret_cast<float*>(lds + 2 * kBlock);
  mean[2 * lane] = mean_of(m[0], weight);
  mean[2 * lane + 1] = mean_of(m[1], weight);
  __syncthreads();
  bf16* ob = p.dq + b * p.s_dq[0] + h * p.s_dq[2];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    f32x16 acc[4] = {w.dq[0][qb], w.dq[1][qb], w.dq[2][qb], w.dq[3][qb]};
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const f32x4 km = *reinterpret_cast<const f32x4*>(mean + 32 * dt + 8 * rq + 4 * hh);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[dt][4 * rq + e] = fmaf(-zsum[qb], km[e], acc[dt][4 * rq + e]);
      }
    bf16* stage = area((uint32_t)qb * kBlock);
    stage_acc_rows(acc, p.scale, lane, stage);
    stage_rows_out(ob, p.s_dq[1], qrow0 + 32 * qb, p.Sq, lane, stage);
  }
}

// ------------------------------------------------------- lists turned round --

// The mean key of each block, one wave a block: 16 lanes a row, 4 rows an
// instruction. Blocks without a key are left out: nothing reads them.
__device__ __forceinline__ void mean_keys(const BwdParams& sp, int64_t blk, int lane) {
  const bwd::Params& p = sp.a;
  if (blk >= sp.kitems) return;
  const int x = (int)(blk % p.ntk), bhk = (int)(blk / p.ntk);
  const int heads = p.H / sp.group, b = bhk / heads, hk = bhk - b * heads;
  const int n = min(key_length(sp.seqused, b, p.Sk) - x * kB, kB);
  if (n <= 0) return;
  const int c = lane & 15, r0 = lane >> 4;
  const bf16* base = p.k + b * p.s_k[0] + hk * p.s_k[2] + (int64_t)x * kB * p.s_k[1] + 8 * c;
  u32x4 raw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 4 * i + r0;
    raw[i] = r < n ? ld16(base + r * p.s_k[1]) : u32x4{0, 0, 0, 0};
  }
  float sum[8] = {};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float v[8];
    unpack8(raw[i], v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += v[e];
  }
  const float inv = 1.0f / (float)n;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    sum[e] += __shfl_xor(sum[e], 16);
    sum[e] += __shfl_xor(sum[e], 32);
    sum[e] *= inv;
  }
  if (r0 == 0) {
    f32x4* to = reinterpret_cast<f32x4*>(sp.means + blk * kD + 8 * c);
    to[0] = f32x4{sum[0], sum[1], sum[2], sum[3]};
    to[1] = f32x4{sum[4], sum[5], sum[6], sum[7]};
  }
}

// (With the mean keys 5.1 us at 4096 tokens of 16 heads, 8.3 at 9216, where K is
// 38 MB; the lists alone are a chain of latencies of 4.8 us.)
//
// One workgroup per 64 query blocks of one (batch, head): a bit each in LDS for
// every block of keys, then out. (An OR of bits: the order of the atomics does
// not matter.) The workgroups from `lists` on: mean keys.
__global__ __launch_bounds__(kTurnThreads) void sparse_turn_kernel(BwdParams sp, int lists) {
  extern __shared__ uint32_t word[];  // [nk][2]
  const bwd::Params& p = sp.a;
  if ((int)blockIdx.x >= lists) {
    const int64_t wg = (int)blockIdx.x - lists;
    mean_keys(sp, wg * (kTurnThreads / 64) + (threadIdx.x >> 6), threadIdx.x & 63);
    return;
  }
  const int w = blockIdx.x % sp.nqw, bh = blockIdx.x / sp.nqw;
  const int b = bh / p.H;
  const int have = (key_length(sp.seqused, b, p.Sk) + kB - 1) / kB;
  for (int i = threadIdx.x; i < 2 * p.ntk; i += kTurnThreads) word[i] = 0;
  __syncthreads();
  const int rows = min(64, p.ntq - 64 * w);
  const int32_t* list = sp.blocks + ((int64_t)bh * p.ntq + 64 * w) * sp.count;
  for (int i = threadIdx.x; i < rows * sp.count; i += kTurnThreads) {
    const int x = list[i], r = i / sp.count;
    if (x >= 0 && x < have) atomicOr(word + 2 * x + (r >> 5), 1u << (r & 31));
  }
  __syncthreads();
  for (int x = threadIdx.x; x < p.ntk; x += kTurnThreads)
    sp.turned[((int64_t)bh * p.ntk + x) * sp.nqw + w] = (uint64_t)word[2 * x] | ((uint64_t)word[2 * x + 1] << 32);
}

// -------------------------------------------------------------------- dK, dV --
//
// 4 waves: wave w owns keys 32 (w & 1) .. + 31 of the block and, of each 64-query
// tile, queries 32 (w >> 1) .. + 31:
//   S      = Q K^T       A = Q rows (LDS),        B = K^T (AGPRs, read once)
//   dP - D = dO V^T      A = dO rows (LDS),       B = V^T (AGPRs), started at -D
//   dV^T  += dO^T P      A = dO^T (transposed LDS reads), B = P
//   dK^T  += Q^T dZ      A = Q^T (transposed LDS reads),  B = dZ
// as attn_bwd_dkdv.hip, whose waves own 32 of 128 keys and all queries of a
// tile: with 64 keys that would leave two SIMDs without work. Every operand
// still feeds one MFMA, so a wave reads no more LDS per MFMA than there; the
// tiles come twice as fast, and the two halves of the queries' sums meet in LDS
// at the end. A tile is 32 slots of one MFMA each:
//   slots  0- 7: S of tile t+1        | P and dZ of tile t, a unit of two
//   slots  8-15: dP - D of tile t+1   |   scores every 2-3 slots from slot 2
//   slots 16-31: dV^T and dK^T of tile t, alternating
// The DMA of tile t+3 goes out one instruction in 4 slots; one barrier a tile.
//
// What bounds it: the waves' issue (matrix pipe busy in 40% of the cycles, 21%
// waits), 0.95 us a tile, and per key block 7 us with nothing beside them for the
// start (its bits, K and V, the first tiles) and the end: 4096 tokens x 16 heads over
// 1, 16, 64 blocks 37, 88-91 and 276 us; 9216 over 24 blocks 272 us, 850 TFLOP/s
// over its four products.
namespace kv {

using bwd::kStat;
using bwd::w1::kDoOff;
using bwd::w1::keep_alive;
using bwd::w1::kNegDOff;
using bwd::w1::kStageBytes;
using bwd::w1::kStatBytes;
using bwd::w1::lds_ld16f;
using bwd::w1::mfma_acc;
using bwd::w1::QdoDma;

constexpr int kWaves = 4;
static_assert(kWaves * 64 == kKvThreads, "backward_fits");
constexpr int kStages = 4;
constexpr int kLead = kStages - 1;  // tile t + kLead is fetched during tile t
// Operand reads ahead of their MFMA, and queues of them (attn_bwd_dkdv.hip).
constexpr int kRPf = 4, kRQ = kRPf + 1;
constexpr int kTPf = 4, kTQ = kTPf + 2;
constexpr int rread_slot(int j) { return j < kRPf ? 0 : j - kRPf; }
constexpr int tread_slot(int j) { return 16 + j - kTPf; }
// Unit u: scores 2 jp, 2 jp + 1 of the P / dZ operand of query chunk c (u =
// 4 c + jp): FMA in slot unit_slot(u), exp, P pack and dZ products, dZ pack in
// the three after it; chunk c's first dV MFMA is in slot 16 + 8 c.
constexpr int unit_slot(int u) { return 2 + (18 * u) / 7; }
static_assert(unit_slot(3) + 2 < 16 && unit_slot(3) + 3 < 17 && unit_slot(7) + 3 < 24, "P and dZ ahead of their use");
constexpr int dma_slot(int i) { return 4 * i + 3; }
constexpr int kStatSlot = 18;

struct Wave {
  bf16x8 kop[8], vop[8];  // K^T / V^T (kk): lane holds K / V[key li][16 kk + 8 hh + 0..7]; AGPRs
  f32x16 av[4], ak[4];    // dV^T, dK^T (dt): d = 32 dt + rows, key li; AGPRs
  f32x16 xs[2], xp[2];    // S, dP - D (buffer): queries of the wave's half, key li
  bf16x8 bp[2], bz[2];    // P, dZ (c): queries of chunk c in accumulator order, key li
  float c;
  uint32_t rrd[4], trd[4];  // LDS byte addresses of row / transposed operand reads, next / this tile
  uint32_t sthis, snext;    // ... of this lane's statistics

  __device__ __forceinline__ void setup(int lane, int hq, float c_, uint32_t ring, uint32_t stat) {
    c = c_;
    const uint32_t half = 4096u * (uint32_t)hq;  // 32 rows of a dual line tile's d half
#pragma unroll
    for (int j = 0; j < 4; ++j) rrd[j] = ring + half + 2u * (uint32_t)dual_row_rd(lane, j);
#pragma unroll
    for (int q = 0; q < 4; ++q) trd[q] = ring + half + 2u * (uint32_t)dual_tr_rd(lane, q >> 1, q & 1);
    sthis = snext = stat + 128u * (uint32_t)hq + 16u * (uint32_t)(lane >> 5);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      av[dt] = f32x16{};
      ak[dt] = f32x16{};
      asm volatile("" : "+a"(av[dt]), "+a"(ak[dt]));
    }
  }
  __device__ __forceinline__ void read_kv(const bf16* kst, const bf16* vst, int lane) {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      kop[kk] = staged_operand(kst, lane, kk);
      vop[kk] = staged_operand(vst, lane, kk);
      asm volatile("" : "+a"(kop[kk]), "+a"(vop[kk]));
    }
  }
  // Row operand j of the next tile: Q (j < 8), dO.
  template <int j>
  __device__ __forceinline__ bf16x8 row_op() const {
    constexpr int kk = j & 7;
    return lds_ld16(rrd[kk & 3] + (j < 8 ? 0u : kDoOff) + 8192u * (kk >> 2));
  }
  // Transposed operand j of this tile: dO^T (even j, for dV) or Q^T, (dt, c).
  template <int j>
  __device__ __forceinline__ bf16x8 tr_op() const {
    constexpr int cc = j >> 3, dt = (j >> 1) & 3;
    constexpr uint32_t off = ((j & 1) ? 0u : kDoOff) + 8192u * (dt >> 1) + 2048u * cc;
    const s16x4 lo = lds_ld8_tr(trd[2 * (dt & 1)] + off);
    const s16x4 hi = lds_ld8_tr(trd[2 * (dt & 1) + 1] + off + 1024u);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  template <int B, int rq>
  __device__ __forceinline__ void load_negd() {
    const f32x4 v = lds_ld16f(snext + kNegDOff + 32u * rq);
#pragma unroll
    for (int i = 0; i < 4; ++i) xp[B][4 * rq + i] = v[i];
  }
  template <int B, int j>
  __device__ __forceinline__ void next_mfma(bf16x8 a) {
    constexpr int kk = j & 7;
    if constexpr (j < 8) xs[B] = mfma32(a, kop[kk], kk == 0 ? f32x16{} : xs[B]);
    else xp[B] = mfma32(a, vop[kk], xp[B]);
  }
  __device__ __forceinline__ void advance_rows(uint32_t delta) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      rrd[j] += delta;
      asm volatile("" : "+v"(rrd[j]));
    }
  }
  __device__ __forceinline__ void advance_tr(uint32_t delta) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      trd[j] += delta;
      asm volatile("" : "+v"(trd[j]));
    }
  }

  // S and dP - D of the first tile into buffer B (no other work).
  template <int B>
  __device__ __forceinline__ void first() {
    bf16x8 rq[kRQ];
    static_for<0, 16>([&](auto G) {
      constexpr int g = decltype(G)::value;
      if constexpr (g < 4) this->template load_negd<B, g>();
      static_for<0, 16>([&](auto J) {
        constexpr int j = decltype(J)::value;
        if constexpr (rread_slot(j) == g) rq[j % kRQ] = this->template row_op<j>();
      });
      this->template next_mfma<B, g>(rq[g % kRQ]);
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // Tile t: P, dZ, dV^T, dK^T (its S and dP - D in buffer SB); with NEXT, S and
  // dP - D of tile t+1 (a ring stage, dstage bytes, on) into the other buffer.
  template <int SB, bool NEXT>
  __device__ __forceinline__ void tile(uint32_t dstage, uint32_t dstat, const QdoDma& dma, bool stats_dma, int lane) {
    constexpr int NB = 1 - SB;
    if constexpr (NEXT) {
      advance_rows(dstage);
      snext = sthis + dstat;
    }
    bf16x8 rq[kRQ], tq[kTQ];
    f32x4 l2[2];
    float fa[2][2], fe[2][2], fz[2][2];
    static_for<0, 32>([&](auto G) {
      constexpr int g = decltype(G)::value;
      if constexpr (NEXT && g < 4) this->template load_negd<NB, g>();
      static_for<0, 16>([&](auto J) {
        constexpr int j = decltype(J)::value;
        if constexpr (NEXT && rread_slot(j) == g) rq[j % kRQ] = this->template row_op<j>();
        if constexpr (tread_slot(j) == g) tq[j % kTQ] = this->template tr_op<j>();
      });
      // lse2 of each pair of units, two slots before its first.
      static_for<0, 8>([&](auto U) {
        constexpr int u = decltype(U)::value;
        if constexpr ((u & 1) == 0 && unit_slot(u) - 2 == g) l2[(u >> 1) & 1] = lds_ld16f(sthis + 32u * (u >> 1));
      });
      if constexpr (g < 16) {
        if constexpr (NEXT) this->template next_mfma<NB, g>(rq[g % kRQ]);
      } else {
        constexpr int j = g - 16, cc = j >> 3, dt = (j >> 1) & 3;
        if constexpr ((j & 1) == 0) mfma_acc(av[dt], tq[j % kTQ], bp[cc]);
        else mfma_acc(ak[dt], tq[j % kTQ], bz[cc]);
      }
      static_for<0, 8>([&](auto U) {
        constexpr int u = decltype(U)::value, cc = u >> 2, jp = u & 3, r = 8 * cc + 2 * jp, e = 2 * (jp & 1);
        float(&a)[2] = fa[u & 1];
        float(&x)[2] = fe[u & 1];
        float(&z)[2] = fz[u & 1];
        if constexpr (unit_slot(u) == g) {
          const f32x4& l = l2[(u >> 1) & 1];
          a[0] = fmaf(xs[SB][r], c, -l[e]);
          a[1] = fmaf(xs[SB][r + 1], c, -l[e + 1]);
          asm volatile("" : "+v"(a[0]), "+v"(a[1]));
        }
        if constexpr (unit_slot(u) + 1 == g) {
          x[0] = fast_exp2(a[0]);
          x[1] = fast_exp2(a[1]);
          asm volatile("" : "+v"(x[0]), "+v"(x[1]));
        }
        if constexpr (unit_slot(u) + 2 == g) {
          bp[cc][2 * jp] = (bf16)x[0];
          bp[cc][2 * jp + 1] = (bf16)x[1];
          z[0] = x[0] * xp[SB][r];
          z[1] = x[1] * xp[SB][r + 1];
          asm volatile("" : "+v"(bp[cc]), "+v"(z[0]), "+v"(z[1]));
        }
        if constexpr (unit_slot(u) + 3 == g) {
          bz[cc][2 * jp] = (bf16)z[0];
          bz[cc][2 * jp + 1] = (bf16)z[1];
          asm volatile("" : "+v"(bz[cc]));
        }
      });
      static_for<0, 8>([&](auto I) {
        constexpr int i = decltype(I)::value;
        if constexpr (dma_slot(i) == g) dma.template issue<i>();
      });
      if constexpr (g == kStatSlot) {
        if (stats_dma) dma.issue_stats(lane);
      }
      // The operands of the previous slot's inline-asm MFMA stay allocated to
      // the end of this slot: the compiler does not see it still reading them.
      if constexpr (g > 16) {
        constexpr int j = g - 17, cc = j >> 3;
        keep_alive(tq[j % kTQ]);
        if constexpr ((j & 1) == 0) keep_alive(bp[cc]);
        else keep_alive(bz[cc]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    keep_alive(tq[15 % kTQ]);
    keep_alive(bz[1]);
    advance_tr(dstage);
    if constexpr (NEXT) sthis = snext;
  }

  __device__ __forceinline__ void fence_acc() {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
                 : "+a"(av[0]), "+a"(av[1]), "+a"(av[2]), "+a"(av[3]), "+a"(ak[0]), "+a"(ak[1]),
                   "+a"(ak[2]), "+a"(ak[3]));
  }
};

// The query tiles that list one block of keys, head by head of those that
// share it, ascending: words of 64 tiles, 64 words (one a lane) at a time.
struct TileWalk {
  const uint64_t* words;  // word w of head g at g * head + w
  int64_t head;
  int nqw, total, page;   // words a head, in all; the page held
  uint64_t mine, lanes, word;
  int at;                 // the current word's index

  __device__ __forceinline__ uint64_t load(int pg, int lane) const {
    const int i = 64 * pg + lane;
    return i < total ? words[(int64_t)(i / nqw) * head + i % nqw] : 0;
  }
  // The first page opened, and the number of tiles.
  __device__ __forceinline__ int start(int lane) {
    open(0, lane);
    word = 0;
    int sum = __popcll(mine);
    for (int pg = 1; 64 * pg < total; ++pg) sum += __popcll(load(pg, lane));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    return __builtin_amdgcn_readfirstlane(sum);
  }
  __device__ __forceinline__ void open(int pg, int lane) {
    page = pg;
    mine = load(pg, lane);
    lanes = __builtin_amdgcn_ballot_w64(mine != 0);
  }
  // The next word with tiles; only while there is one.
  __device__ __forceinline__ void next_word(int lane) {
    while (lanes == 0) open(page + 1, lane);
    const int l = __builtin_ctzll(lanes);
    lanes &= lanes - 1;
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)mine, l);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(mine >> 32), l);
    word = (uint64_t)lo | ((uint64_t)hi << 32);
    at = 64 * page + l;
  }
  // Past the next k tiles; there are more than k.
  __device__ __forceinline__ void skip(int k, int lane) {
    while (k > 0) {
      if (word == 0) next_word(lane);
      const int c = __builtin_popcountll(word);
      if (c <= k) {
        word = 0;
        k -= c;
      } else {
        for (; k > 0; --k) word &= word - 1;
      }
    }
  }
  // Only while there is one: (head of the group, query tile).
  __device__ __forceinline__ void next(int lane, int& g, int& tile) {
    if (word == 0) next_word(lane);
    g = at / nqw;
    tile = 64 * (at - g * nqw) + __builtin_ctzll(word);
    word &= word - 1;
  }
};

__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void sparse_dkdv_kernel(BwdParams sp) {
  const bwd::Params& p = sp.a;
  __shared__ __attribute__((aligned(1024))) bf16 ring[kStages * 2 * kTileElems];
  __shared__ __attribute__((aligned(1024))) float stat[kStages * kStat];

  int item = item_of(blockIdx.x, gridDim.x, sp.kitems * sp.kparts);
  if (item < 0) return;
  const int whole = item;
  const int part = item % sp.kparts;
  item /= sp.kparts;
  const int kblk = item % p.ntk;
  const int bhk = item / p.ntk;
  const int heads_k = p.H / sp.group;
  const int b = bhk / heads_k, hk = bhk - b * heads_k;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int hq = wave >> 1;
  const int key0 = kblk * kB + 32 * (wave & 1);
  const int klen = key_length(sp.seqused, b, p.Sk);
  const int h0 = hk * sp.group;

  TileWalk walk;
  walk.words = sp.turned + (((int64_t)b * p.H + h0) * p.ntk + kblk) * sp.nqw;
  walk.head = (int64_t)p.ntk * sp.nqw;
  walk.nqw = sp.nqw;
  walk.total = sp.group * sp.nqw;

  const int all = walk.start(lane);
  const int from = (int)((int64_t)all * part / sp.kparts);
  const int n = (int)((int64_t)all * (part + 1) / sp.kparts) - from;
  if (n > 0) {
    walk.skip(from, lane);
  } else if (sp.kparts == 1) {
    // No list names the block: zeros (each wave 32 rows of dV or dK).
    bf16* to = hq ? p.dk + b * p.s_dk[0] + hk * p.s_dk[2] : p.dv + b * p.s_dv[0] + hk * p.s_dv[2];
    const int64_t rs = hq ? p.s_dk[1] : p.s_dv[1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = key0 + 4 * i + (lane >> 4);
      if (row < p.Sk) st16_nt(to + row * rs + 8 * (lane & 15), u32x4{0, 0, 0, 0});
    }
    return;
  }

  const uint32_t ring0 = lds_addr(ring);
  const uint32_t stat0 = lds_addr(stat);
  auto stage_addr = [&](int t) -> uint32_t { return ring0 + (uint32_t)(t % kStages) * kStageBytes; };
  auto stat_addr = [&](int t) -> uint32_t { return stat0 + (uint32_t)(t % kStages) * kStatBytes; };

  Wave w;
  w.setup(lane, hq, p.c, ring0, stat0);
  QdoDma dma;
  dma.fixed(p, wave, lane);
  const bool stats_dma = wave == 0;
  int g = 0, tile = 0, left = n;
  // The job of the next tile of the list; past it its last one again, into a
  // stage that nothing reads: every tile issues the same number of DMAs.
  auto prepare_job = [&](int t) {
    if (left > 0) {
      walk.next(lane, g, tile);
      --left;
    }
    const int h = h0 + g;
    dma.prepare(p, tile * kB, stage_addr(t), stat_addr(t),
                p.stats + (((int64_t)b * p.H + h) * p.ntq + tile) * kStat, wave,
                p.q + b * p.s_q[0] + h * p.s_q[2], p.dout + b * p.s_do[0] + h * p.s_do[2], lane);
  };
  auto issue_job = [&](int t) {
    prepare_job(t);
    static_for<0, 8>([&](auto I) { dma.template issue<decltype(I)::value>(); });
    if (stats_dma) dma.issue_stats(lane);
  };
  if (n > 0) {
    // The wave's K and V rows staged in ring stages 2 and 3 (16 KB per wave),
    // free until tile 2's DMA. Keys past klen re-read its last key (their
    // gradients are not stored).
    bf16* kst = ring + 2 * (2 * kTileElems) + wave * 8192;
    stage_rows_in(p.k + b * p.s_k[0] + hk * p.s_k[2], p.s_k[1], key0, klen, lane, kst);
    stage_rows_in(p.v + b * p.s_v[0] + hk * p.s_v[2], p.s_v[1], key0, klen, lane, kst + 4096);
    issue_job(0);
    issue_job(1);
    if (stats_dma) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    __syncthreads();  // tile 0 and every wave's K / V rows
    w.read_kv(kst, kst + 4096, lane);
    __syncthreads();  // every wave has read its K / V rows
    issue_job(2);
    const int b0 = (n - 1) & 1;  // the last tile's S is in buffer 0
    if (b0) w.first<1>();
    else w.first<0>();

    // At the top of tile t, tile t+1 (issued two tiles earlier) is complete in
    // this wave and the barrier publishes every wave's part; tile t+3 then
    // takes the stage of tile t-1, last read before that barrier.
    auto run = [&](auto sb, auto next, int t) {
      constexpr int SB = decltype(sb)::value;
      constexpr bool NEXT = decltype(next)::value;
      if (stats_dma) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      __syncthreads();
      prepare_job(t + kLead);
      w.tile<SB, NEXT>(stage_addr(t + 1) - stage_addr(t), stat_addr(t + 1) - stat_addr(t), dma, stats_dma, lane);
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    int t = 0;
    if (b0) {
      run(I1{}, std::true_type{}, 0);
      t = 1;
    }
    for (; t + 1 < n; t += 2) {
      run(I0{}, std::true_type{}, t);
      run(I1{}, std::true_type{}, t + 1);
    }
    run(I0{}, std::false_type{}, t);  // t == n - 1
  }
  wait_dma();
  __syncthreads();  // every wave is done with the ring; no DMA in flight
  w.fence_acc();

  // The waves of the two query halves swap sums: half 0 stores dV, half 1 dK.
  // Record `wave`: 16 KB, one float4 per lane in 16 blocks.
  f32x4* xch = reinterpret_cast<f32x4*>(ring) + wave * 16 * 64 + lane;
  const f32x4* other = reinterpret_cast<const f32x4*>(ring) + (wave ^ 2) * 16 * 64 + lane;
  f32x16 own[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    const f32x16& give = hq ? w.av[dt] : w.ak[dt];
    own[dt] = hq ? w.ak[dt] : w.av[dt];
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
      xch[(4 * dt + rq) * 64] = f32x4{give[4 * rq], give[4 * rq + 1], give[4 * rq + 2], give[4 * rq + 3]};
  }
  __syncthreads();
  const bool there = key0 + (lane & 31) < klen;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const f32x4 v = other[(4 * dt + rq) * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) own[dt][4 * rq + e] = there ? own[dt][4 * rq + e] + v[e] : 0.f;
    }
  if (sp.kparts > 1) {
    f32x4* dst = sp.sums + ((int64_t)whole * kKTiles + 4 * wave) * 256;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) store_tile(dst + dt * 256, own[dt], lane);
    return;
  }
  bf16* ostage = ring + 2 * (2 * kTileElems) + wave * 4096;
  stage_acc_rows(own, hq ? p.scale : 1.0f, lane, ostage);
  bf16* to = hq ? p.dk + b * p.s_dk[0] + hk * p.s_dk[2] : p.dv + b * p.s_dv[0] + hk * p.s_dv[2];
  stage_rows_out(to, hq ? p.s_dk[1] : p.s_dv[1], key0, p.Sk, lane, ostage);
}

}  // namespace kv

// ------------------------------------------------------------ sums of parts --

// One wave per accumulator tile of an item: its parts' sum, in order, to the
// gradient's rows. Q: dQ's items (tile 4 qb + dt); else dK's and dV's (tile 4
// wave + dt of sparse_dkdv_kernel).
template <bool Q>
__global__ __launch_bounds__(256) void sparse_sum_kernel(BwdParams sp) {
  constexpr int kTiles = Q ? kQTiles : kKTiles;
  const bwd::Params& p = sp.a;
  const int parts = Q ? sp.qparts : sp.kparts, items = Q ? sp.items : sp.kitems;
  const int id = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int item = id / kTiles, tile = id % kTiles;
  if (item >= items) return;
  const f32x4* from = sp.sums + ((int64_t)item * parts * kTiles + tile) * 256 + lane;
  f32x4 acc[4] = {};
#pragma unroll 4
  for (int s = 0; s < parts; ++s)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) acc[rq] += from[(int64_t)s * kTiles * 256 + rq * 64];

  const int blocks = Q ? p.ntq : p.ntk, heads = Q ? p.H : p.H / sp.group;
  const int blk = item % blocks, bh = item / blocks;
  const int64_t b = bh / heads, h = bh - b * heads;
  const int group = tile >> 2;  // Q: the row half; else the wave: key half, then dV / dK
  const int row = blk * kB + 32 * (group & 1) + (lane & 31);
  const bool dk = !Q && group >= 2;
  const int64_t* st = Q ? p.s_dq : dk ? p.s_dk : p.s_dv;
  bf16* to = (Q ? p.dq : dk ? p.dk : p.dv) + b * st[0] + row * st[1] + h * st[2] + 32 * (tile & 3) + 4 * (lane >> 5);
  const float scale = Q || dk ? p.scale : 1.0f;
  if (row >= (Q ? p.Sq : p.Sk)) return;
  if constexpr (Q) {
    // The correction of sparse_dq_kernel, over all parts.
    f32x4 m[4] = {};
    float zsum = 0.f, weight = 0.f;
    for (int s = 0; s < parts; ++s) {
      const float* rec = sp.recs + ((int64_t)item * parts + s) * kRec;
      zsum += rec[row - blk * kB];
      weight += rec[kRecWeight];
#pragma unroll
      for (int rq = 0; rq < 4; ++rq)
        m[rq] += *reinterpret_cast<const f32x4*>(rec + kRecMean + 32 * (tile & 3) + 8 * rq + 4 * (lane >> 5));
    }
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[rq][e] = fmaf(-zsum, mean_of(m[rq][e], weight), acc[rq][e]);
  }
#pragma unroll
  for (int rq = 0; rq < 4; ++rq)
    *reinterpret_cast<u32x2*>(to + 8 * rq) = u32x2{pack_bf16(acc[rq][0] * scale, acc[rq][1] * scale),
                                                   pack_bf16(acc[rq][2] * scale, acc[rq][3] * scale)};
}

// Parts of the lists of key blocks: as many as give every CU a workgroup, of 4
// query tiles or more where the lists are as long as on average.
static int plan_kparts(int64_t kitems, int64_t group, int64_t nq, int64_t nk, int64_t count) {
  const int64_t tiles = std::min(group * nq, (group * nq * count + nk - 1) / nk);
  const int64_t parts = std::min<int64_t>(device_cu_count() / std::max<int64_t>(kitems, 1), tiles / 4);
  return (int)std::max<int64_t>(1, parts);
}

struct BwdPlan {
  int64_t nq, nk, nqw, items, kitems;
  int qparts, kparts;
  size_t stats, turned, sums, means, recs;  // bytes
  size_t total() const { return stats + turned + sums + means + recs; }
};

static BwdPlan plan_bwd(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk, int64_t count) {
  BwdPlan r = {};
  r.nq = (Sq + kB - 1) / kB;
  r.nk = (Sk + kB - 1) / kB;
  r.nqw = (r.nq + 63) / 64;
  r.items = B * H * r.nq;
  r.kitems = B * Hk * r.nk;
  r.qparts = plan_split(r.items, count);
  r.kparts = plan_kparts(r.kitems, H / Hk, r.nq, r.nk, count);
  r.stats = (size_t)r.items * bwd::kStat * sizeof(float);
  r.turned = ((size_t)(B * H * r.nk * r.nqw) * sizeof(uint64_t) + 15) / 16 * 16;
  const size_t q = r.qparts > 1 ? (size_t)r.items * r.qparts * kQTiles : 0;
  const size_t k = r.kparts > 1 ? (size_t)r.kitems * r.kparts * kKTiles : 0;
  r.sums = std::max(q, k) * 256 * sizeof(f32x4);  // one after the other
  r.means = (size_t)r.kitems * kD * sizeof(float);
  r.recs = r.qparts > 1 ? (size_t)r.items * r.qparts * kRec * sizeof(float) : 0;
  return r;
}

}  // namespace sparse
}  // namespace aa

using namespace aa;

extern "C" size_t aa_sparse_bwd_workspace(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk, int64_t count) {
  if (B <= 0 || Sq <= 0 || Sk <= 0 || H <= 0 || Hk <= 0 || H % Hk || count < 1) return 0;
  const sparse::BwdPlan plan = sparse::plan_bwd(B, Sq, Sk, H, Hk, count);
  return plan.total();
}

extern "C" int aa_sparse_bwd(const aa_sparse_bwd_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sparse;
  clear_error();
  if (!a) return fail(AA_EINVAL, "sparse_bwd: null args");
  if (a->dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, "sparse_bwd: only bf16 is implemented");
  if (a->hd != sparse::kD) return fail(AA_EUNSUPPORTED, "sparse_bwd: head_dim must be 128");
  if (a->B < 0 || a->Sq < 0 || a->Sk < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk)
    return fail(AA_EINVAL, "sparse_bwd: bad sizes (H must be a multiple of Hk)");
  if (a->count < 1 || a->count > kMaxCount) return fail(AA_EUNSUPPORTED, "sparse_bwd: count must be 1 to 4096");
  if (a->Sk > kMaxBlocks * kB) return fail(AA_EUNSUPPORTED, "sparse_bwd: at most 262144 keys");
  const int64_t nq = (a->Sq + kB - 1) / kB, nk = (a->Sk + kB - 1) / kB;
  if (a->Sq > 0x7fffffc0 || a->B > 0x7fffffff || a->H > 65535 || !backward_fits(a->B, a->Sq, a->Sk, a->H, a->Hk))
    return fail(AA_EUNSUPPORTED, "sparse_bwd: too many blocks");
  if (a->B == 0 || a->Sq == 0 || a->Sk == 0) return AA_OK;
  const void* all[] = {a->dout, a->q, a->k, a->v, a->out, a->lse, a->blocks, a->dq, a->dk, a->dv};
  for (const void* ptr : all)
    if (!ptr) return fail(AA_EINVAL, "sparse_bwd: null pointer");
  const void* rows[] = {a->dout, a->q, a->k, a->v, a->out, a->dq, a->dk, a->dv};
  for (const void* ptr : rows)
    if (!aligned16(ptr)) return fail(AA_EINVAL, "sparse_bwd: tensors must be 16-byte aligned");
  const int64_t* strides[] = {a->dout_stride, a->q_stride, a->k_stride, a->v_stride, a->out_stride, a->dq_stride, a->dk_stride, a->dv_stride};
  for (const int64_t* st : strides)
    for (int i = 0; i < 3; ++i)
      if (st[i] % 8) return fail(AA_EINVAL, "sparse_bwd: strides must be multiples of 8 elements");
  for (int i = 0; i < 4; ++i)
    if (strides[i][1] < 0 || strides[i][1] >= kMaxRowStride)
      return fail(AA_EUNSUPPORTED, "sparse_bwd: sequence stride of dout, q, k or v out of range");
  const BwdPlan plan = plan_bwd(a->B, a->Sq, a->Sk, a->H, a->Hk, a->count);
  const int64_t lists = turn_lists(a->B, a->H, nq), means = turn_means(plan.kitems);
  if (!workspace || !aligned16(workspace) || workspace_bytes < plan.total())
    return fail(AA_EINVAL, "sparse_bwd: workspace too small or misaligned");

  BwdParams sp = {};
  bwd::Params& p = sp.a;
  p.dout = (const bf16*)a->dout;
  p.q = (const bf16*)a->q;
  p.k = (const bf16*)a->k;
  p.v = (const bf16*)a->v;
  p.o = (const bf16*)a->out;
  p.lse = a->lse;
  p.dq = (bf16*)a->dq;
  p.dk = (bf16*)a->dk;
  p.dv = (bf16*)a->dv;
  for (int i = 0; i < 3; ++i) {
    p.s_do[i] = a->dout_stride[i];
    p.s_q[i] = a->q_stride[i];
    p.s_k[i] = a->k_stride[i];
    p.s_v[i] = a->v_stride[i];
    p.s_o[i] = a->out_stride[i];
    p.s_dq[i] = a->dq_stride[i];
    p.s_dk[i] = a->dk_stride[i];
    p.s_dv[i] = a->dv_stride[i];
  }
  p.H = (int)a->H;
  p.Sq = (int)a->Sq;
  p.Sk = (int)a->Sk;
  p.ntq = (int)nq;
  p.ntk = (int)nk;
  p.c = a->softmax_scale * kLog2e;
  p.scale = a->softmax_scale;
  p.stats = (float*)workspace;
  sp.seqused = a->seqused_k;
  sp.blocks = a->blocks;
  sp.group = (int)(a->H / a->Hk);
  sp.count = (int)a->count;
  sp.nqw = (int)plan.nqw;
  sp.items = (int)plan.items;
  sp.kitems = (int)plan.kitems;
  sp.qparts = plan.qparts;
  sp.kparts = plan.kparts;
  char* at = (char*)workspace + plan.stats;
  sp.turned = (uint64_t*)at;
  sp.sums = (f32x4*)(at += plan.turned);
  sp.means = (float*)(at += plan.sums);
  sp.recs = (float*)(at += plan.means);
  hipStream_t st = (hipStream_t)stream;
  sparse_turn_kernel<<<(unsigned)(lists + means), kTurnThreads, (size_t)nk * 8, st>>>(sp, (int)lists);
  sparse_dq_kernel<<<grid_of(plan.items * sp.qparts), 64, 0, st>>>(sp);
  if (sp.qparts > 1) sparse_sum_kernel<true><<<(unsigned)(plan.items * kQTiles / 4), 256, 0, st>>>(sp);
  kv::sparse_dkdv_kernel<<<grid_of(plan.kitems * sp.kparts), kv::kWaves * 64, 0, st>>>(sp);
  if (sp.kparts > 1) sparse_sum_kernel<false><<<(unsigned)(plan.kitems * kKTiles / 4), 256, 0, st>>>(sp);
  return check_launch("sparse_bwd");
}
