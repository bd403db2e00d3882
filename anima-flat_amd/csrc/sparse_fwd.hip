// Forward of the attention over selected blocks, head_dim 128, bf16 in / fp32
// accumulate (gfx950).
//
//   out = softmax over the keys of the listed blocks (scores q.k * scale) v,
//
// for each block of 64 queries over its own list of blocks of 64 keys.
//
// One wave is one workgroup and takes one query block (or a part of its list,
// below): 64 queries are what one wave can hold with one wave per SIMD, and a
// key block is the 64-key tile of FwdWave's slot schedule (attn_fwd_wave.h), so
// the dense forward's inner loop runs here on tiles whose places in memory come
// from the list. Nothing is shared between waves: lists differ in what they
// name and in how long they are, and a workgroup of several waves would wait
// for its longest at each barrier. Each wave has its own K and V tile in LDS
// (attn_fwd_wave_dma.h), 4 workgroups fill a CU, and as one of them starts or
// ends its neighbours compute.
//
// Work list order: query blocks of one head are neighbours on one XCD, so the
// keys that they have in common come from its L2.
//
// What bounds it: one wave's issue beside its MFMAs, as in the dense forward (1.9 us
// a tile), and what a round of lists does together, start and end: 13 of 43 us for
// 4096 tokens of 16 heads over 16 blocks each, one round. The matrix pipe is busy in 50% of
// the cycles, 21% are waits. 2 x 4096 tokens 82 us (840 TFLOP/s), 16384 tokens over 32
// blocks 280 us (980); 9216 over 24 blocks 158 us (730), 2.25 rounds of which the last
// leaves three of four SIMDs idle. Over one block each it is bound by HBM (4096 tokens
// 15.6 us, 4.3 TB/s).
//
// Few query blocks (fewer than the chip's SIMDs): each list is cut into
// `nsplit` parts of whole blocks, the parts write O and their row statistics
// in fp32 and a second launch merges them (one query, 16 heads, 32 blocks:
// 9.7 + 4.0 us; unsplit the list alone would take 60).
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <string>
#include <type_traits>

#include "attn_fwd_wave_dma.h"
#include "sparse.h"

namespace aa {
namespace sparse {

using ks::WaveDma;

constexpr uint32_t kTileBytes = kTileElems * sizeof(bf16);

// One work item: query block and part of its list. TRACK: with a running
// maximum; without, each row keeps the maximum of its first tile, and `again` is
// set, with nothing written, if a sum left the exponent range by that.
template <bool LSE, bool SPLIT, bool TRACK>
__device__ __forceinline__ void run_item(int item, int split, uint8_t* lds, uint32_t* bits, uint32_t& again) {
  // The kernel's arguments and the lane, as if unknown before: what two bodies
  // of a kernel have in common would be kept in registers through the first.
  constexpr bool FSUM = LSE || TRACK;
  typedef const __attribute__((address_space(4))) SparseParams* Args;
  Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  int lane = threadIdx.x;
  asm volatile("" : "+s"(args), "+s"(item), "+v"(lane));
  const __attribute__((address_space(4))) SparseParams& p = *args;
  const int qblk = item % p.nq;
  const int bh = item / p.nq;
  const int b = bh / p.H, h = bh - b * p.H, hk = h / p.group;
  const int li = lane & 31, hh = lane >> 5;
  const int qrow0 = qblk * kB;
  const int klen = key_length(p.seqused, b, p.Sk);

  // Q: 64 rows (two areas of 32, tile_io.h) into the V tile's place, which the
  // first V tile reaches after the first scores.
  const bf16* qb = p.q + b * p.qs[0] + h * p.qs[2];
  auto stage_q = [&](bf16* to) {
    stage_rows_in(qb, p.qs[1], qrow0, p.Sq, lane, to);
    stage_rows_in(qb, p.qs[1], qrow0 + 32, p.Sq, lane, to + 32 * kD);
  };
  bf16* ktile = reinterpret_cast<bf16*>(lds);
  bf16* vtile = reinterpret_cast<bf16*>(lds + kTileBytes);
  stage_q(vtile);

  BlockWalk walk;
  auto read_list = [&]() {
    walk.read(p.blocks + (int64_t)item * p.count, p.count, (klen + kB - 1) / kB, bits, lane);
    if constexpr (SPLIT) walk.part(split, p.nsplit, lane);
    walk.start();
  };
  read_list();
  const int n = walk.n;

  // The block that klen ends in (-1: it ends with one): the last one of any
  // list that has it.
  const int part = klen % kB ? klen / kB : -1;
  const int last = klen % kB - 1;  // its last row
  const bf16* kp = p.k + b * p.ks[0] + hk * p.ks[2];
  const bf16* vp = p.v + b * p.vs[0] + hk * p.vs[2];
  const uint32_t mine = lds_addr(lds);
  WaveDma dma;
  dma.setup(kp, vp, p.ks[1], p.vs[1], lane, mine);
  auto k_tile = [&](int x) {
    dma.kt = kp + (int64_t)x * kB * p.ks[1];
    if (x == part) dma.rows_k(lane, last);
  };
  auto v_tile = [&](int x) {  // chunks 0-2
    dma.vt = vp + (int64_t)x * kB * p.vs[1];
    if (x == part) dma.rows_v<0, 6>(lane, last);
  };
  auto v3_tile = [&](int x) {
    dma.v3 = vp + (int64_t)x * kB * p.vs[1];
    if (x == part) dma.rows_v<6, 8>(lane, last);
  };
  // Blocks of tiles i, i + 1, i + 2; past the list its last one again, into
  // places that nothing reads (every tile issues the same number of DMAs).
  int x = 0, left = n;
  auto next_block = [&]() {
    if (left > 0) {
      x = walk.next();
      --left;
    }
    return x;
  };

  FwdWave w;
  w.setup(lane, p.c, mine);
  w.lf[0][0] = w.lf[0][1] = w.lf[1][0] = w.lf[1][1] = 0.f;
  if (n > 0) {
    int x0 = next_block(), x1 = next_block(), x2 = next_block();
    k_tile(x0);
    static_for<0, 16>([&](auto I) {
      constexpr int i = decltype(I)::value;
      dma.template issue_k<(i >> 2), (i & 3)>();
    });
    ks::wait_vm<16>();  // the Q rows
    w.read_q(vtile, lane);
    wait_dma();
    // As if a tile -1 came before: the K quarters of tile 1, then V chunks
    // 0-2 of tile 0.
    k_tile(x1);
    const int b0 = (n - 1) & 1;  // the last tile's S^T is in buffer 0
    if (b0) {
      w.qk_first<1>(dma);
      if (x0 == part) dma.template mask<1>(w, x0 * kB, klen);
    } else {
      w.qk_first<0>(dma);
      if (x0 == part) dma.template mask<0>(w, x0 * kB, klen);
    }
    static_for<0, 4>([&](auto I) { dma.template issue_k<3, decltype(I)::value>(); });
    v_tile(x0);
    static_for<0, 12>([&](auto I) {
      constexpr int i = decltype(I)::value;
      dma.template issue_v<(i >> 2), (i & 3)>();
    });
    if (b0) w.max_plain<1>();
    else w.max_plain<0>();
    // Finite also where every score of the first tile is -inf: s - m would be
    // NaN there and the later tiles lost to it.
    w.m_raw[0] = fmaxf(w.mt[0], -FLT_MAX);
    w.m_raw[1] = fmaxf(w.mt[1], -FLT_MAX);

    auto run = [&](auto sb, auto next) {
      constexpr int SB = decltype(sb)::value;
      constexpr bool NEXT = decltype(next)::value;
      k_tile(x2);
      v3_tile(x0);
      v_tile(x1);
      w.tile<SB, NEXT, TRACK, FSUM>(0, x1 == part, x1 * kB, klen, dma);
      if constexpr (NEXT) {
        if constexpr (TRACK) w.update_max<FSUM>();
        x0 = x1;
        x1 = x2;
        x2 = next_block();
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    int i = 0;
    if (b0) {
      run(I1{}, std::true_type{});
      i = 1;
    }
    for (; i + 1 < n; i += 2) {
      run(I0{}, std::true_type{});
      run(I1{}, std::true_type{});
    }
    run(I0{}, std::false_type{});
  }
  wait_dma();
  w.fence_o();
  if constexpr (!TRACK) {
    const uint64_t out = __builtin_amdgcn_ballot_w64(!w.sums_in_range());
    again = (uint32_t)(out | (out >> 32));
    if (again) return;
  }
  // The fp32 probabilities' sum stands in for the rounded ones' where that took
  // in another row's NaN or infinity on the matrix pipe (FwdWave::setup; O did
  // not).
  float lsum[2] = {w.lsum[0][0], w.lsum[1][0]}, lf[2] = {0.f, 0.f};
  if constexpr (FSUM) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      lf[q] = pair_sum(w.lf[q][0] + w.lf[q][1]);
      if (TRACK && !(lsum[q] <= FLT_MAX)) lsum[q] = lf[q];
    }
  }

  if constexpr (SPLIT) {
    const int64_t rec = ((int64_t)item * p.nsplit + split) * kB;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int row = 32 * q + li;
      if (qrow0 + row >= p.Sq) continue;
      if (hh == 0) p.part_stat[rec + row] = f32x4{w.m_raw[q], lsum[q], lf[q], 0.f};
      if (n == 0) continue;  // the combine kernel reads no O of a part without keys
      float* to = p.part_o + (rec + row) * kD;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const f32x16& o = w.o[dt][q];
          *reinterpret_cast<f32x4*>(to + 32 * dt + 8 * rq + 4 * hh) =
              f32x4{o[4 * rq], o[4 * rq + 1], o[4 * rq + 2], o[4 * rq + 3]};
        }
    }
    return;
  }
  // O is normalised by the sum of the bf16 probabilities that weighted V, the
  // LSE is that of the fp32 ones. No key, or none with a weight: O = 0, LSE =
  // -inf (a NaN sum goes on).
  const int64_t at = b * p.os[0] + h * p.os[2];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const bool any = lsum[q] != 0.f;
    const f32x16 o[4] = {w.o[0][q], w.o[1][q], w.o[2][q], w.o[3][q]};
    bf16* area = ktile + q * 32 * kD;
    stage_acc_rows(o, any ? 1.0f / lsum[q] : 0.f, lane, area);
    stage_rows_out(p.o + at, p.os[1], qrow0 + 32 * q, p.Sq, lane, area);
    if constexpr (LSE) {
      const int row = qrow0 + 32 * q + li;
      if (hh == 0 && row < p.Sq)
        p.lse[(int64_t)bh * p.Sq + row] = any ? (w.m_raw[q] * p.c + __log2f(lf[q])) * kLn2 : -INFINITY;
    }
  }
}

// LSE: something reads the log-sum-exp, so the fp32 probabilities are summed
// too (attn_fwd_ks_kernel's comment).
template <bool LSE, bool SPLIT>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void sparse_fwd_kernel(SparseParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kTileBytes];
  __shared__ __attribute__((aligned(16))) uint32_t bits[2 * 64];
  int item = item_of(blockIdx.x, gridDim.x, p.items * (SPLIT ? p.nsplit : 1));
  if (item < 0) return;
  int split = 0;
  if constexpr (SPLIT) {
    split = item % p.nsplit;
    item = item / p.nsplit;
  }
  // (Opaque: joined to the first body, the second one's code spilled registers.)
  uint32_t again = 0;
  run_item<LSE, SPLIT, false>(item, split, lds, bits, again);
  again = __builtin_amdgcn_readfirstlane(again);
  asm volatile("" : "+s"(again)::"memory");
  if (again) run_item<LSE, SPLIT, true>(item, split, lds, bits, again);
}

// One workgroup per query: wave w takes the parts w, w + 4, ..., two head dims a
// lane, and the waves' sums meet in LDS in order. (The parts come from other
// XCDs' workgroups, a long way; 8 loads a lane are on it at once.)
constexpr int kCombineWaves = 4;
__global__ __launch_bounds__(64 * kCombineWaves) void sparse_combine_kernel(SparseParams p) {
  __shared__ float sums[kCombineWaves][4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x;
  const int64_t bh = r / p.Sq;
  const int q = (int)(r - bh * p.Sq);
  const int64_t b = bh / p.H, h = bh - b * p.H;
  const int64_t rec = (bh * p.nq + q / kB) * p.nsplit * kB + q % kB;
  float mx = -INFINITY;
  for (int s = lane; s < p.nsplit; s += 64) mx = fmaxf(mx, p.part_stat[rec + (int64_t)s * kB][0]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
  float sum = 0.f, fsum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 8
  for (int s = wave; s < p.nsplit; s += kCombineWaves) {
    const f32x4 st = p.part_stat[rec + (int64_t)s * kB];
    const float2 o = *reinterpret_cast<const float2*>(p.part_o + (rec + (int64_t)s * kB) * kD + 2 * lane);
    // The O of a part without keys was never written and does not count.
    const bool keys = st[0] != -INFINITY;
    const float a = keys ? fast_exp2((st[0] - mx) * p.c) : 0.f;
    sum += st[1] * a;
    fsum += st[2] * a;
    o0 += keys ? o.x * a : 0.f;
    o1 += keys ? o.y * a : 0.f;
  }
  sums[wave][0][lane] = sum;
  sums[wave][1][lane] = fsum;
  sums[wave][2][lane] = o0;
  sums[wave][3][lane] = o1;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kCombineWaves; ++w) {
    sum += sums[w][0][lane];
    fsum += sums[w][1][lane];
    o0 += sums[w][2][lane];
    o1 += sums[w][3][lane];
  }
  const bool any = sum != 0.f;
  const float scale = any ? 1.0f / sum : 0.f;
  const int64_t at = b * p.os[0] + q * p.os[1] + h * p.os[2] + 2 * lane;
  *reinterpret_cast<uint32_t*>(p.o + at) = pack_bf16(o0 * scale, o1 * scale);
  if (p.lse && lane == 0) p.lse[r] = any ? (mx * p.c + __log2f(fsum)) * kLn2 : -INFINITY;
}

}  // namespace sparse
}  // namespace aa

using namespace aa;

static size_t split_bytes(int64_t items, int nsplit) {
  return nsplit > 1 ? (size_t)(items * nsplit * sparse::kB * (sparse::kD + 4) * (int64_t)sizeof(float)) : 0;
}

extern "C" size_t aa_sparse_fwd_workspace(int64_t B, int64_t Sq, int64_t H, int64_t count) {
  if (B <= 0 || Sq <= 0 || H <= 0 || count < 1) return 0;
  const int64_t items = B * H * ((Sq + sparse::kB - 1) / sparse::kB);
  return split_bytes(items, sparse::plan_split(items, count));
}

extern "C" int aa_sparse_fwd(const aa_sparse_fwd_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sparse;
  using sparse::kD;
  clear_error();
  if (!a) return fail(AA_EINVAL, "sparse_fwd: null args");
  if (a->dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, "sparse_fwd: only bf16 is implemented");
  if (a->hd != kD) return fail(AA_EUNSUPPORTED, "sparse_fwd: head_dim must be 128");
  if (a->B < 0 || a->Sq < 0 || a->Sk < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk)
    return fail(AA_EINVAL, "sparse_fwd: bad sizes (H must be a multiple of Hk)");
  if (a->count < 1 || a->count > kMaxCount) return fail(AA_EUNSUPPORTED, "sparse_fwd: count must be 1 to 4096");
  if (a->Sk > kMaxBlocks * kB) return fail(AA_EUNSUPPORTED, "sparse_fwd: at most 262144 keys");
  const int64_t nq = (a->Sq + kB - 1) / kB;
  if (a->Sq > 0x7fffffc0 || a->B > 0x7fffffff || a->H > 65535 || (nq && a->B * a->H > 0x1fffff0 / nq))
    return fail(AA_EUNSUPPORTED, "sparse_fwd: too many query blocks");
  if (a->lse && a->Sk && !backward_fits(a->B, a->Sq, a->Sk, a->H, a->Hk))
    return fail(AA_EUNSUPPORTED, "sparse_fwd: too many blocks for a backward pass (without lse there is none)");
  if (a->B == 0 || a->Sq == 0) return AA_OK;
  if (!a->q || !a->out || !a->blocks || (a->Sk && (!a->k || !a->v))) return fail(AA_EINVAL, "sparse_fwd: null pointer");
  for (const void* ptr : {a->q, a->k, a->v, (const void*)a->out})
    if (!aligned16(ptr)) return fail(AA_EINVAL, "sparse_fwd: tensors must be 16-byte aligned");
  for (const int64_t* st : {a->q_stride, a->k_stride, a->v_stride, a->out_stride})
    for (int i = 0; i < 3; ++i)
      if (st[i] % 8) return fail(AA_EINVAL, "sparse_fwd: strides must be multiples of 8 elements");
  for (const int64_t st : {a->k_stride[1], a->v_stride[1]})
    if (st < 0 || st >= kMaxRowStride) return fail(AA_EUNSUPPORTED, "sparse_fwd: sequence stride of k or v out of range");
  SparseParams p = {};
  p.q = (const bf16*)a->q;
  p.k = (const bf16*)a->k;
  p.v = (const bf16*)a->v;
  p.o = (bf16*)a->out;
  p.lse = a->lse;
  p.seqused = a->seqused_k;
  p.blocks = a->blocks;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_stride[i];
    p.ks[i] = a->k_stride[i];
    p.vs[i] = a->v_stride[i];
    p.os[i] = a->out_stride[i];
  }
  p.H = (int)a->H;
  p.group = (int)(a->H / a->Hk);
  p.Sq = (int)a->Sq;
  p.Sk = (int)a->Sk;
  p.nq = (int)nq;
  p.count = (int)a->count;
  p.items = (int)(a->B * a->H * nq);
  p.c = a->softmax_scale * kLog2e;
  p.nsplit = plan_split(p.items, a->count);
  const size_t bytes = split_bytes(p.items, p.nsplit);
  if (bytes && (workspace_bytes < bytes || !workspace || !aligned16(workspace)))
    return fail(AA_EINVAL, "sparse_fwd: workspace too small or misaligned");
  hipStream_t st = (hipStream_t)stream;
  if (p.nsplit == 1) {
    const unsigned grid = grid_of(p.items);
    if (p.lse) sparse_fwd_kernel<true, false><<<grid, 64, 0, st>>>(p);
    else sparse_fwd_kernel<false, false><<<grid, 64, 0, st>>>(p);
    return check_launch("sparse_fwd");
  }
  p.part_stat = (f32x4*)workspace;
  p.part_o = (float*)(p.part_stat + (int64_t)p.items * p.nsplit * kB);
  const unsigned grid = grid_of((int64_t)p.items * p.nsplit);
  if (p.lse) sparse_fwd_kernel<true, true><<<grid, 64, 0, st>>>(p);
  else sparse_fwd_kernel<false, true><<<grid, 64, 0, st>>>(p);
  sparse_combine_kernel<<<(unsigned)(a->B * a->H * a->Sq), 64 * kCombineWaves, 0, st>>>(p);
  return check_launch("sparse_fwd");
}
