// Selection of key blocks for the sparse attention (gfx950): for each block of
// 64 queries the `count` blocks of 64 keys with the largest
//   score = mean(q of the block) . mean(k of the block),
// ties to the lower index, in ascending order.
//
// The result is discrete: a rounding that reorders two nearly equal scores
// gives another attention. So means and scores are fp64: sums of bf16 values
// are exact there (as long as they span less than 2^39 of each other), and a
// score's own error, about 2^-50 of its summands, is below any difference that
// means something. That costs 1/16 of the inputs' bytes for the means and, at
// 16384 tokens, 134 M fp64 FMAs beside the attention's 137 G.
//
//   means_kernel   one wave per block of rows: HBM-bound, q and k once (2 x 4096
//                  tokens of 16 + 16 heads 14.8 us, 4.5 TB/s)
//   select_kernel  one workgroup per 4 query blocks of one head: scores into LDS,
//                  a key block per lane (k's means are transposed for that, q's
//                  are scalars), then a wave per row finds the count-th largest
//                  score bit by bit
#include <string>

#include "sparse.h"

namespace aa {
namespace sparse {

struct SelectParams {
  const bf16 *q, *k;
  const int32_t* seqused;
  int32_t* blocks;
  double* qm;  // [B H][nq][128]
  double* km;  // [B Hk][128][nk]
  int64_t qs[3], ks[3];
  int B, H, Hk, Sq, Sk, nq, nk, count;
};

constexpr int kMeanWaves = 4;

// Four consecutive blocks of rows of one (batch, head) per workgroup; heads
// of q first, then those of k.
__global__ __launch_bounds__(64 * kMeanWaves) void means_kernel(SelectParams p, int qgroups, int kgroups, int qtotal) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const bool key = (int)blockIdx.x >= qtotal;
  const int idx = key ? blockIdx.x - qtotal : blockIdx.x;
  const int heads = key ? p.Hk : p.H;
  // Heads are the fastest: neighbouring workgroups read neighbouring bytes.
  const int h = idx % heads, rest = idx / heads;
  const int groups = key ? kgroups : qgroups;
  const int b = rest / groups, blk = (rest - b * groups) * kMeanWaves + wave;
  const int rows = key ? key_length(p.seqused, b, p.Sk) : p.Sq;
  const int n = min(rows - blk * kB, kB);
  if (n <= 0) return;  // nothing reads the mean of no rows
  const int64_t* st = key ? p.ks : p.qs;
  const bf16* base = (key ? p.k : p.q) + b * st[0] + h * st[2] + (int64_t)blk * kB * st[1];

  // 16 lanes a row, 4 rows an instruction.
  const int c = lane & 15, r0 = lane >> 4;
  u32x4 raw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 4 * i + r0;
    raw[i] = r < n ? ld16(base + (int64_t)r * st[1] + 8 * c) : u32x4{0, 0, 0, 0};
  }
  double sum[8] = {};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float x[8];
    unpack8(raw[i], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += (double)x[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    sum[e] += __shfl_xor(sum[e], 16);
    sum[e] += __shfl_xor(sum[e], 32);
  }
  // Lane group r0 writes two of the eight.
  const double inv = (double)n;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if ((e >> 1) != r0) continue;
    const double m = sum[e] / inv;
    const int d = 8 * c + e;
    if (key) p.km[((int64_t)(b * p.Hk + h) * kD + d) * p.nk + blk] = m;
    else p.qm[((int64_t)(b * p.H + h) * p.nq + blk) * kD + d] = m;
  }
}

// Order of doubles as that of unsigned numbers: NaN above everything (it goes
// on to the attention's output), zeros equal. Never 0.
__device__ __forceinline__ uint64_t order_of(double x) {
  if (x != x) return ~uint64_t{0};
  if (x == 0) x = 0;
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | (uint64_t{1} << 63);
}

constexpr int kSelectThreads = 512;
constexpr int kRows = 4;  // query blocks of a workgroup

// A row's scores for one wave: score 64 j + lane of lane `lane`, j < nj. Up to 1024
// stay in registers; more are read from LDS again for every bit (at 4096 they
// would take 128 registers a lane, and their ballots the scalar ones).
template <int NV>
struct Held {
  uint64_t v[NV];
  __device__ __forceinline__ Held(const uint64_t* row, int have, int lane) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = 64 * j + lane < have ? row[64 * j + lane] : 0;
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) f(j, v[j]);
  }
};
struct Kept {
  const uint64_t* row;
  int have, lane;
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 2
    for (int j = 0; j < (have + 63) / 64; ++j) f(j, 64 * j + lane < have ? row[64 * j + lane] : 0);
  }
};

// The list of one row, by one wave: the count-th largest score bit by bit, then
// every score above it and, in order, as many equal ones as are missing.
template <class Scores>
__device__ __forceinline__ void pick(const Scores& scores, int have, int count, int32_t* out, int lane) {
  uint64_t t = 1;       // the largest value that at least `count` scores reach (no score is 0)
  int ties = have;      // of the scores equal to t, how many are taken
  if (have > count) {
    t = 0;
    bool exact = false;
    for (int bit = 63; bit >= 0 && !exact; --bit) {
      const uint64_t trial = t | (uint64_t{1} << bit);
      int reach = 0;
      scores.each([&](int, uint64_t v) { reach += __popcll(__builtin_amdgcn_ballot_w64(v >= trial)); });
      if (reach >= count) t = trial;
      exact = reach == count;
    }
    if (!exact) {
      int above = 0;
      scores.each([&](int, uint64_t v) { above += __popcll(__builtin_amdgcn_ballot_w64(v > t)); });
      ties = count - above;
    }
  }
  const uint64_t below = (uint64_t{1} << lane) - 1;
  int at = 0;
  scores.each([&](int j, uint64_t v) {
    const uint64_t same = __builtin_amdgcn_ballot_w64(v == t);
    const bool take = v > t || (v == t && __popcll(same & below) < ties);
    ties -= __popcll(same);
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    if (take) out[at + __popcll(taken & below)] = 64 * j + lane;
    at += __popcll(taken);
  });
  for (int i = at + lane; i < count; i += 64) out[i] = -1;
}

// Scores of the workgroup's query blocks against the blocks of keys: the former's
// means are scalar operands, the latter's are read once for all of them. The
// waves share the blocks of keys and, with few of them, the head dims (PARTS
// parts, which meet in LDS in a fixed order): latency bounds it, so many loads
// are on their way at once and 512 threads take 4 rows (2048 query blocks x 64 of
// keys: 256 threads 10.1 us, 512 6.8; 4096 x 256 24 us, 7 of them the search.
// 16 rows a workgroup by fp64 matrix instructions: 8.9 and 22).
template <int PARTS>
__device__ __forceinline__ void dot_rows(const double* qm, const double* km, int nk, int have, int rows, double* partial,
                                         uint64_t* score) {
  constexpr int kWidth = kSelectThreads / PARTS, kSpan = kD / PARTS;
  // Written by the launch before: constant here, so that the uniform reads of
  // qm are scalar loads.
  typedef const __attribute__((address_space(4))) double* Const;
  const int part = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWidth);
  for (int j = threadIdx.x - part * kWidth; j < have; j += kWidth) {
    double acc[kRows] = {};
#pragma unroll 1
    for (int d0 = 0; d0 < kSpan; d0 += 16) {
      double x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = km[(int64_t)(part * kSpan + d0 + i) * nk + j];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        // Opaque: the scalar loads of all rows at once would spill.
        uint64_t at = (uint64_t)(uintptr_t)(qm + min(r, rows - 1) * kD + part * kSpan + d0);
        asm volatile("" : "+s"(at));
        const Const q = (Const)at;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[r] = fma(q[i], x[i], acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if constexpr (PARTS == 1) score[r * nk + j] = order_of(acc[r]);
      else partial[(part * kRows + r) * kWidth + j] = acc[r];
    }
  }
  __syncthreads();
  if constexpr (PARTS > 1) {
    for (int i = threadIdx.x; i < kRows * kWidth; i += kSelectThreads) {
      const int r = i / kWidth, j = i % kWidth;
      if (j >= have) continue;
      double sum = 0;
#pragma unroll
      for (int s = 0; s < PARTS; ++s) sum += partial[(s * kRows + r) * kWidth + j];
      score[r * nk + j] = order_of(sum);
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kSelectThreads) void select_kernel(SelectParams p, int rgroups, int items) {
  extern __shared__ __attribute__((aligned(16))) uint64_t score[];  // [kRows][nk]
  __shared__ double partial[kRows * kSelectThreads];
  const int item = item_of(blockIdx.x, gridDim.x, items);
  if (item < 0) return;
  const int bh = item / rgroups, r0 = (item - bh * rgroups) * kRows;
  const int b = bh / p.H, h = bh - b * p.H;
  const int rows = min(kRows, p.nq - r0);
  const int have = (key_length(p.seqused, b, p.Sk) + kB - 1) / kB;
  const double* qm = p.qm + ((int64_t)bh * p.nq + r0) * kD;
  const double* km = p.km + (int64_t)(b * p.Hk + h / (p.H / p.Hk)) * kD * p.nk;
  if (have <= 64) dot_rows<8>(qm, km, p.nk, have, rows, partial, score);
  else if (have <= 128) dot_rows<4>(qm, km, p.nk, have, rows, partial, score);
  else if (have <= 256) dot_rows<2>(qm, km, p.nk, have, rows, partial, score);
  else dot_rows<1>(qm, km, p.nk, have, rows, partial, score);
  const int lane = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < rows; r += kSelectThreads / 64) {
    int32_t* out = p.blocks + ((int64_t)bh * p.nq + r0 + r) * p.count;
    const uint64_t* row = score + r * p.nk;
    if (have <= 64) pick(Held<1>(row, have, lane), have, p.count, out, lane);
    else if (have <= 256) pick(Held<4>(row, have, lane), have, p.count, out, lane);
    else if (have <= 1024) pick(Held<16>(row, have, lane), have, p.count, out, lane);
    else pick(Kept{row, have, lane}, have, p.count, out, lane);
  }
}

}  // namespace sparse
}  // namespace aa

using namespace aa;

static bool select_sizes(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk, int64_t* nq, int64_t* nk) {
  *nq = (Sq + sparse::kB - 1) / sparse::kB;
  *nk = (Sk + sparse::kB - 1) / sparse::kB;
  return B >= 0 && Sq >= 0 && Sk >= 0 && H >= 1 && Hk >= 1 && H % Hk == 0;
}

extern "C" size_t aa_block_select_workspace(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk) {
  int64_t nq, nk;
  if (!select_sizes(B, Sq, Sk, H, Hk, &nq, &nk)) return 0;
  return (size_t)(B * (H * nq + Hk * nk) * sparse::kD * (int64_t)sizeof(double));
}

extern "C" int aa_block_select(const aa_block_select_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (!a) return fail(AA_EINVAL, "block_select: null args");
  if (a->dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, "block_select: only bf16 is implemented");
  if (a->hd != sparse::kD) return fail(AA_EUNSUPPORTED, "block_select: head_dim must be 128");
  int64_t nq, nk;
  if (!select_sizes(a->B, a->Sq, a->Sk, a->H, a->Hk, &nq, &nk))
    return fail(AA_EINVAL, "block_select: bad sizes (H must be a multiple of Hk)");
  if (a->count < 1 || a->count > sparse::kMaxCount) return fail(AA_EUNSUPPORTED, "block_select: count must be 1 to 4096");
  if (nk > sparse::kMaxBlocks) return fail(AA_EUNSUPPORTED, "block_select: at most 262144 keys");
  if (a->Sq > 0x7fffffc0 || a->B > 0x7fffffff || a->H > 65535 || (nq && a->B * a->H > 0x7ffffff0 / nq))
    return fail(AA_EUNSUPPORTED, "block_select: too many query blocks");
  if (a->B == 0 || a->Sq == 0) return AA_OK;
  if (!a->q || (a->Sk && !a->k) || !a->blocks) return fail(AA_EINVAL, "block_select: null pointer");
  if (!aligned16(a->q) || !aligned16(a->k)) return fail(AA_EINVAL, "block_select: q and k must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (a->q_stride[i] % 8 || a->k_stride[i] % 8)
      return fail(AA_EINVAL, "block_select: strides must be multiples of 8 elements");
  if (workspace_bytes < aa_block_select_workspace(a->B, a->Sq, a->Sk, a->H, a->Hk) || !workspace || !aligned16(workspace))
    return fail(AA_EINVAL, "block_select: workspace too small or misaligned");

  using namespace sparse;
  SelectParams p = {};
  p.q = (const bf16*)a->q;
  p.k = (const bf16*)a->k;
  p.seqused = a->seqused_k;
  p.blocks = a->blocks;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_stride[i];
    p.ks[i] = a->k_stride[i];
  }
  p.B = (int)a->B;
  p.H = (int)a->H;
  p.Hk = (int)a->Hk;
  p.Sq = (int)a->Sq;
  p.Sk = (int)a->Sk;
  p.nq = (int)nq;
  p.nk = (int)nk;
  p.count = (int)a->count;
  p.qm = (double*)workspace;
  p.km = p.qm + a->B * a->H * nq * kD;
  hipStream_t st = (hipStream_t)stream;
  const int64_t qg = (nq + kMeanWaves - 1) / kMeanWaves, kg = (nk + kMeanWaves - 1) / kMeanWaves;
  const int64_t qtotal = a->B * a->H * qg, total = qtotal + a->B * a->Hk * kg;
  if (!grid_fits(total, 64 * kMeanWaves)) return fail(AA_EUNSUPPORTED, "block_select: too many blocks");
  means_kernel<<<(unsigned)total, 64 * kMeanWaves, 0, st>>>(p, (int)qg, (int)kg, (int)qtotal);
  if (!grid_fits(grid_of(a->B * a->H * nq), kSelectThreads)) return fail(AA_EUNSUPPORTED, "block_select: too many query blocks");
  const int64_t rg = (nq + kRows - 1) / kRows, items = a->B * a->H * rg;
  select_kernel<<<grid_of(items), kSelectThreads, (size_t)(kRows * nk) * sizeof(uint64_t), st>>>(p, (int)rg, (int)items);
  return check_launch("block_select");
}
