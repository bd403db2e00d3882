// dQ of the attention backward for short query ranges (gfx950): one workgroup
// = 64 queries of one (batch, head), its keys split over the 4 waves inside
// the workgroup, as the forward does it (attn_fwd_ks.hip).
//
// Why: dq_kernel takes 256 queries per workgroup, so 1024 tokens x 16 heads
// are 64 workgroups on 256 CUs, and a key split over workgroups would move
// fp32 partials of four times dQ's size through memory. Here wave w takes the
// 32-key blocks w, w + 4, ..., all waves hold the same 64 queries' Q^T and
// dO^T in registers, and the four fp32 partial dQ^T are summed in wave order
// through LDS: deterministic, no workspace, 256 workgroups for that call.
// A wave's schedule and DMA: attn_bwd_dq_wave.h.
#include <type_traits>

#include "attn_bwd.h"
#include "attn_bwd_dq_wave.h"

namespace aa {
namespace bwd {
namespace dqks {

constexpr int kWaves = 4;

__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void dq_ks_kernel(Params p, int first_item, int nqitem, int total_blocks) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * kWaveBytes];

  // A quarter of one of dq_kernel's items of 256 queries.
  const int logical = xcd_remap(blockIdx.x, total_blocks);
  const int item = first_item + logical / 4;
  const int bh = item / nqitem;
  const int qblk = 4 * (item - bh * nqitem) + (logical & 3);
  if (qblk >= p.ntq) return;
  const int b = bh / p.H, h = bh - b * p.H;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int li = lane & 31, hh = lane >> 5;
  const int qrow0 = qblk * kT;

  // Q, dO and O rows (64 each) into places of the rings that the first blocks
  // leave free: the third K place of waves 0-1, 2-3 and the second V place of
  // waves 0-1, as areas of 32 rows (row staging, tile_io.h). Each wave moves
  // 16 rows of each tensor.
  auto area = [&](int w, uint32_t off) { return reinterpret_cast<bf16*>(lds + w * kWaveBytes + off); };
  auto stage_in = [&](const bf16* base, int64_t rs, bf16* a0, bf16* a1) {
    bf16* a = (wave & 2) ? a1 : a0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * (wave & 1) + 4 * i + (lane >> 4);
      const int row = min(qrow0 + 32 * (wave >> 1) + r, p.Sq - 1);
      dma16(base + (int64_t)row * rs + 8 * ((lane & 15) ^ (r & 15)), a + (16 * (wave & 1) + 4 * i) * 128);
    }
  };
  bf16* aq[2] = {area(0, 2 * kBlock), area(1, 2 * kBlock)};
  bf16* ado[2] = {area(2, 2 * kBlock), area(3, 2 * kBlock)};
  bf16* ao[2] = {area(0, kVRing + kBlock), area(1, kVRing + kBlock)};
  stage_in(p.q + b * p.s_q[0] + h * p.s_q[2], p.s_q[1], aq[0], aq[1]);
  stage_in(p.dout + b * p.s_do[0] + h * p.s_do[2], p.s_do[1], ado[0], ado[1]);
  stage_in(p.o + b * p.s_o[0] + h * p.s_o[2], p.s_o[1], ao[0], ao[1]);

  // The wave's i-th block is key block wave + 4 i; one that would reach past
  // Sk is moved back to end there, its keys below lo_of (counted by the
  // blocks before it) masked. Past the wave's last, the last one is fetched
  // again into places that nothing reads.
  const int nblk = (p.Sk + kKeys - 1) / kKeys;
  const int n = (nblk - wave + kWaves - 1) / kWaves;  // 0 if the wave has none
  auto lo_of = [&](int i) { return (wave + kWaves * i) * kKeys; };
  auto row_of = [&](int i) { return min(lo_of(i), max(p.Sk - kKeys, 0)); };
  const bf16* kp = p.k + b * p.s_k[0] + h * p.s_k[2];
  const bf16* vp = p.v + b * p.s_v[0] + h * p.s_v[2];
  const uint32_t mine = lds_addr(lds) + (uint32_t)wave * kWaveBytes;
  BlockDma dma;
  dma.setup(p.s_k[1], p.s_v[1], p.Sk, lane);
  auto k_job = [&](int i) {
    dma.kt = kp + (int64_t)row_of(min(i, n - 1)) * p.s_k[1];
    dma.kdst = mine + (uint32_t)(i % 3) * kBlock;
  };
  auto ka_job = [&](int i) {
    dma.ka = kp + (int64_t)row_of(min(i, n - 1)) * p.s_k[1];
    dma.kadst = mine + (uint32_t)(i % 3) * kBlock;
  };
  auto v_job = [&](int i) {
    dma.vt = vp + (int64_t)row_of(min(i, n - 1)) * p.s_v[1];
    dma.vdst = mine + kVRing + (uint32_t)(i & 1) * kBlock;
  };
  if (n > 0) {
    k_job(0);
    dma.all_k();
    v_job(0);
    dma.all_v();
    k_job(1);
    dma.all_k();
    wait_vm<8>();  // all but K of block 1
  } else {
    wait_dma();
  }
  __syncthreads();

  DqWave w;
  w.li = li;
  w.hh = hh;
  w.c = p.c;
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
  // Operands, and each query's stats: lse2 = lse log2(e) and -D, D =
  // rowsum(dO o O) (this lane's 64 values, then the partner lane's half).
  // Queries past Sq: lse2 = +inf (P = 0) and D = 0.
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = qrow0 + 32 * qb + li;
    float nd = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      w.qop[qb][kk] = staged_operand(aq[qb], lane, kk);
      w.dop[qb][kk] = staged_operand(ado[qb], lane, kk);
      float x[8], y[8];
      unpack8(__builtin_bit_cast(u32x4, staged_operand(ao[qb], lane, kk)), x);
      unpack8(__builtin_bit_cast(u32x4, w.dop[qb][kk]), y);
#pragma unroll
      for (int i = 0; i < 8; ++i) nd = fmaf(y[i], x[i], nd);
      asm volatile("" : "+a"(w.qop[qb][kk]));
    }
    nd = pair_sum(nd);
    nd = q < p.Sq ? -nd : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) w.nd[qb][r] = nd;
    w.lse2[qb] = q < p.Sq ? p.lse[(int64_t)bh * p.Sq + q] * kLog2e : INFINITY;
  }
  // The record that the dK/dV kernel reads: lse2, -D, zero pad.
  if (wave == 0 && hh == 0) {
    float* st = p.stats + ((int64_t)bh * p.ntq + qblk) * kStat;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      st[32 * qb + li] = w.lse2[qb];
      st[kT + 32 * qb + li] = w.nd[qb][0];
      st[2 * kT + 32 * qb + li] = 0.f;
      st[3 * kT + 32 * qb + li] = 0.f;
    }
  }
  // The record's stores and the lse loads leave the vmcnt counts to the DMA.
  wait_dma();
  __syncthreads();  // every wave has read the staged rows

  if (n > 0) {
    v_job(1);
    dma.all_v();
    const int b0 = (n - 1) & 1;  // the last block's S^T is in buffer 0
    const bool m0 = lo_of(0) + kKeys > p.Sk;
    if (b0) {
      w.first<1>();
      if (m0) w.mask<1>(row_of(0), lo_of(0), p.Sk);
    } else {
      w.first<0>();
      if (m0) w.mask<0>(row_of(0), lo_of(0), p.Sk);
    }
    v_job(2);
    dma.all_v();
    ka_job(2);
    static_for<0, 4>([&](auto I) { dma.template issue_ka<decltype(I)::value>(); });
    // Once as the blocks' own counts do not hold yet: all but those 12, that
    // is K and V of block 1.
    wait_vm<12>();

    auto run = [&](auto sb, auto next, int i) {
      constexpr int SB = decltype(sb)::value;
      constexpr bool NEXT = decltype(next)::value;
      if constexpr (NEXT) {
        wait_vm<20>();  // V of block i + 1
        w.advance_rows((i + 1) % 3 == 0 ? 0u - 2u * kBlock : kBlock, (i + 1) & 1 ? kBlock : 0u - kBlock);
        k_job(i + 2);
        ka_job(i + 3);
        v_job(i + 3);
      }
      const int lo = lo_of(i + 1);
      w.block<SB, NEXT>(lo + kKeys > p.Sk, row_of(i + 1), lo, p.Sk, dma);
      w.advance_tr((i + 1) % 3 == 0 ? 0u - 2u * kBlock : kBlock);
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
  // Keeps dQ in AGPRs up to here and orders the reads after its MFMAs.
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
               : "+a"(w.dq[0][0]), "+a"(w.dq[1][0]), "+a"(w.dq[2][0]), "+a"(w.dq[3][0]),
                 "+a"(w.dq[0][1]), "+a"(w.dq[1][1]), "+a"(w.dq[2][1]), "+a"(w.dq[3][1]));
  __syncthreads();  // every wave is done with its rings

  // Sum over the waves in order: wave d takes head-dims 32 d .. 32 d + 31.
  // Block (dt, source wave, qb, rq) of 1 KB: one float4 per lane.
  f32x4* xch = reinterpret_cast<f32x4*>(lds);
  bf16* stage = reinterpret_cast<bf16*>(lds + 128 * 1024);
  auto at = [&](int dt, int src, int qb, int rq) { return (((dt * kWaves + src) * 2 + qb) * 4 + rq) * 64 + lane; };
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const f32x16& v = w.dq[dt][qb];
        xch[at(dt, wave, qb, rq)] = f32x4{v[4 * rq], v[4 * rq + 1], v[4 * rq + 2], v[4 * rq + 3]};
      }
  __syncthreads();
#pragma unroll
  for (int qb = 0; qb < 2; ++qb)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      f32x4 v = xch[at(wave, 0, qb, rq)];
#pragma unroll
      for (int src = 1; src < kWaves; ++src) v += xch[at(wave, src, qb, rq)];
      const u32x2 o2 = {pack_bf16(v[0] * p.scale, v[1] * p.scale), pack_bf16(v[2] * p.scale, v[3] * p.scale)};
      *reinterpret_cast<u32x2*>(stage + qb * 4096 + stage_at(li, 4 * wave + rq) + 4 * hh) = o2;
    }
  __syncthreads();
  bf16* ob = p.dq + b * p.s_dq[0] + h * p.s_dq[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * wave + 4 * i + (lane >> 4), cc = lane & 15;
    const u32x4 v = *reinterpret_cast<const u32x4*>(stage + (r >> 5) * 4096 + stage_at(r & 31, cc));
    if (qrow0 + r < p.Sq) st16_nt(ob + (int64_t)(qrow0 + r) * p.s_dq[1] + 8 * cc, v);
  }
}

}  // namespace dqks

void launch_dq_ks(const Params& p, int first_item, int items, int nqitem, hipStream_t stream) {
  dqks::dq_ks_kernel<<<dim3((unsigned)(4 * items)), dqks::kWaves * 64, 0, stream>>>(p, first_item, nqitem,
                                                                                  4 * items);
}

}  // namespace bwd
}  // namespace aa
