// Activations kept in 8 bits for the backward pass, and the operators whose
// backward reads them: GELU, and the low-rank product of a LoRA projection.
//
// Checkpoint of a row x[K]: int8 codes and one power of two per group of 32
// channels. With amax the group's largest magnitude, 2^(k-1) <= amax < 2^k,
// the step is 2^(k - 7) (at least 2^-126), code = round-to-nearest-even(x /
// step) clamped to +-127, and the value kept is code * step. A bf16 amax / step
// is at most 127.5, so the clamp moves a value by no more than rounding does:
// |x - kept| <= step / 2, at most 2^-7 of amax. The step being a power of two,
// code * step is exact in bf16: a backward product over kept values rounds
// nothing on the way in. The group's byte is the step's biased exponent
// (1 .. 248); 255 marks a group with a value that is not finite, all of which
// read back as NaN. 33/32 bytes a value against bf16's 2.
//
// gelu8: y = GELU(x) in bf16 from x itself; dx = dy GELU'(kept x). HBM bound:
//   2 + 2 + 33/32 bytes a value forward, 33/32 + 2 + 2 backward.
// lora_down8: t = x A^T for A [R, K], R <= 64; dx = dt A; dA = dt^T kept(x).
//   HBM bound: 2 + 33/32 bytes a value forward, 2 (dx) + 33/32 (dA) backward.
#include <algorithm>
#include <type_traits>

#include "aa_common.h"
#include "block_math.h"

namespace aa {

constexpr int kGroup = 32;          // channels per step
constexpr uint32_t kNotFinite = 255;

// The biased exponent of the step of a group whose largest magnitude has these
// bits.
__device__ __forceinline__ uint32_t step_exp(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 6;  // amax in [2^(e' - 127), 2^(e' - 126))
  return amax_bits >= kInfBits ? kNotFinite : (uint32_t)max(e, 1);
}
// step, and 1 / step (both exact: 1 <= exponent <= 248).
__device__ __forceinline__ float step_of(uint32_t e) {
  return __uint_as_float(e == kNotFinite ? 0x7fc00000u : e << 23);
}
__device__ __forceinline__ float inv_step_of(uint32_t e) { return __uint_as_float((254u - e) << 23); }

// Codes of 8 values. An exponent above 253 needs an inverse step below the
// normal range, which cannot occur for finite values (e <= 248); for a marked
// group the codes are never read as numbers.
__device__ __forceinline__ u32x2 codes8(const float* v, float inv) {
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    c[i] = round_bits(__builtin_amdgcn_fmed3f(v[i] * inv, -127.0f, 127.0f));
  return u32x2{low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
}
// Signed byte i (0..3) of a word as a float.
template <int kByte>
__device__ __forceinline__ float byte_f(uint32_t w) {
  return (float)((int)(w << (24 - 8 * kByte)) >> 24);
}

// -------------------------------------------------------------------- GELU --

constexpr int kGeThreads = 256;

// Sixteen values per lane: a group of 32 is two neighbouring lanes. Rows are
// cut into 2 G units of 16 (G = ceil(K / 32)); codes have the row stride 32 G.
// With kFlat (K % 32 == 0) rows follow one another without gaps and a unit's
// index is its place.
struct GeluFwd {
  const bf16* x;
  bf16* y;
  uint8_t* codes;  // [rows][32 G], or null: no checkpoint
  uint8_t* exps;   // [rows][G]
  int64_t units;
  int K, upr;  // units per row
};

template <bool kFlat>
__global__ __launch_bounds__(kGeThreads) void gelu8_fwd_kernel(GeluFwd p) {
  const int64_t u = (int64_t)blockIdx.x * kGeThreads + threadIdx.x;
  if (u >= p.units) return;  // units come in pairs: both lanes of a group stay
  int64_t at = 16 * u;
  int have = 2;  // 8-value halves of this unit that are inside the row
  if constexpr (!kFlat) {
    const int64_t row = u / p.upr;
    const int k = 16 * (int)(u - row * p.upr);
    at = row * p.K + k;
    have = k + 16 <= p.K ? 2 : k + 8 <= p.K ? 1 : 0;
  }
  u32x4 raw[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h < have) raw[h] = ld16(p.x + at + 8 * h);
  float v[16];
  unpack8(raw[0], v);
  unpack8(raw[1], v + 8);
  if (p.codes) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, mag_bits(v[i]));
    top = max(top, dpp_mov<kDppXor1>(top));
    const uint32_t e = step_exp(top);
    const float inv = inv_step_of(e);
    const u32x2 a = codes8(v, inv), b = codes8(v + 8, inv);
    st16(p.codes + 16 * u, u32x4{a[0], a[1], b[0], b[1]});
    if ((threadIdx.x & 1) == 0) p.exps[u >> 1] = (uint8_t)e;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = gelu(v[i]);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h < have) st16(p.y + at + 8 * h, pack8(v + 8 * h));
}

struct GeluBwd {
  const bf16* dy;
  const uint8_t* codes;
  const uint8_t* exps;
  bf16* dx;
  int64_t units;
  int K, upr;
};

template <bool kFlat>
__global__ __launch_bounds__(kGeThreads) void gelu8_bwd_kernel(GeluBwd p) {
  const int64_t u = (int64_t)blockIdx.x * kGeThreads + threadIdx.x;
  if (u >= p.units) return;
  int64_t at = 16 * u;
  int have = 2;
  if constexpr (!kFlat) {
    const int64_t row = u / p.upr;
    const int k = 16 * (int)(u - row * p.upr);
    at = row * p.K + k;
    have = k + 16 <= p.K ? 2 : k + 8 <= p.K ? 1 : 0;
  }
  const u32x4 c = ld16(p.codes + 16 * u);
  const float step = step_of(p.exps[u >> 1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h >= have) continue;
    float g[8];
    unpack8(ld16(p.dy + at + 8 * h), g);
    static_for<0, 8>([&](auto I) {
      constexpr int i = decltype(I)::value;
      g[i] *= gelu_slope(byte_f<i & 3>(c[2 * h + (i >> 2)]) * step);
    });
    st16(p.dx + at + 8 * h, pack8(g));
  }
}

// -------------------------------------------------------------------- LoRA --

constexpr int kLoMaxR = 64;

// t = x A^T and the checkpoint of x, in one pass over x. A workgroup takes 16
// RT rows; its waves take slices of 256 channels in turn. A slice's 16 rows are
// loaded as whole lines (two rows of 512 bytes per instruction, lane l: row
// i + 8 (l / 32), channels 8 (l % 32)), so a group of 32 channels is four
// neighbouring lanes; they are coded and stored from there, and cross to the
// MFMA's operand layout through a tile of LDS that the wave has to itself
// (row r's 16-byte chunk c in slot c ^ r). The waves' partial sums are added in
// LDS in a fixed order.
struct LoraFwd {
  const bf16* x;  // [M, K]
  const bf16* a;  // [R, K]
  bf16* t;        // [M, R]
  uint8_t* codes;  // [M][32 G], or null
  uint8_t* exps;   // [G][Mp], Mp = M up to a multiple of 16
  int64_t M, Mp;
  int K, R, G;
};

constexpr int kLoWaves = 8;
constexpr int kLoThreads = 64 * kLoWaves;
constexpr int kLoSlice = 256;

typedef float f32x4v __attribute__((ext_vector_type(4)));

template <int NR, int RT>
__global__ __launch_bounds__(kLoThreads) void lora8_fwd_kernel(LoraFwd p) {
  // The waves' x tiles, then their sums.
  constexpr int kTile = 16 * kLoSlice * 2;
  constexpr int kSums = NR * RT * 16 * 16 * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLoWaves * (kTile > kSums ? kTile : kSums)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * (16 * RT);
  uint8_t* tile = lds + wave * kTile;
  f32x4v acc[RT][NR];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[t][n] = f32x4v{0.f, 0.f, 0.f, 0.f};
  for (int k0 = kLoSlice * wave; k0 < p.K; k0 += kLoSlice * kLoWaves) {
    const int col = k0 + 8 * (lane & 31);
    const bool in = col < p.K;  // K is a multiple of 8
    u32x4 raw[RT][8];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        raw[t][i] = u32x4{0, 0, 0, 0};
        const int64_t row = min(row0 + 16 * t + i + 8 * (lane >> 5), p.M - 1);
        if (in) raw[t][i] = ld16(p.x + row * p.K + col);
      }
    bf16x8 w[8][NR];
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int rank = 16 * n + li, k = k0 + 32 * s + 8 * g;
        u32x4 v = u32x4{0, 0, 0, 0};
        if (rank < p.R && k < p.K) v = ld16(p.a + (int64_t)rank * p.K + k);
        w[s][n] = __builtin_bit_cast(bf16x8, v);
      }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      uint32_t ex[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i + 8 * (lane >> 5);
        *reinterpret_cast<u32x4*>(tile + r * 512 + (((lane & 31) ^ r) * 16)) = raw[t][i];
        if (p.codes) {
          float v[8];
          unpack8(raw[t][i], v);
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max(top, mag_bits(v[j]));
          top = max(top, dpp_mov<kDppXor1>(top));
          top = max(top, dpp_mov<kDppXor2>(top));
          const uint32_t e = step_exp(top);
          const int64_t row = row0 + 16 * t + r;
          if (row < p.M && col < kGroup * p.G)
            *reinterpret_cast<u32x2*>(p.codes + row * (kGroup * p.G) + col) = codes8(v, inv_step_of(e));
          ex[i >> 2] |= e << (8 * (i & 3));
        }
      }
      // Rows r0 .. r0 + 7 of this lane's group; rows past M, up to Mp, too.
      if (p.codes && (lane & 3) == 0 && col < kGroup * p.G && row0 + 16 * t < p.Mp)
        *reinterpret_cast<u32x2*>(p.exps + (int64_t)(col / kGroup) * p.Mp + row0 + 16 * t + 8 * (lane >> 5)) =
            u32x2{ex[0], ex[1]};
      // The wave's own tile: its writes are in order with its reads.
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const bf16x8 xv = *reinterpret_cast<const bf16x8*>(tile + li * 512 + (((4 * s + g) ^ li) * 16));
#pragma unroll
        for (int n = 0; n < NR; ++n)
          acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[s][n], xv, acc[t][n], 0, 0, 0);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  // acc[t][n]: lane li is token 16 t + li, element i is rank 16 n + 4 g + i.
  __syncthreads();
  f32x4v* sums = reinterpret_cast<f32x4v*>(lds);
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int n = 0; n < NR; ++n) sums[(wave * RT * NR + t * NR + n) * 64 + lane] = acc[t][n];
  __syncthreads();
  for (int o = threadIdx.x; o < RT * NR * 64; o += kLoThreads) {
    f32x4v s = sums[o];
#pragma unroll
    for (int w = 1; w < kLoWaves; ++w) s += sums[w * RT * NR * 64 + o];
    const int l = o & 63, n = (o >> 6) % NR, t = (o >> 6) / NR;
    const int64_t row = row0 + 16 * t + (l & 15);
    const int rank = 16 * n + 4 * (l >> 4);
    if (row < p.M && rank < p.R)  // R is a multiple of 8
      *reinterpret_cast<u32x2*>(p.t + row * p.R + rank) = u32x2{pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3])};
  }
}

// dx = dt A: a wave takes 128 channels and 16 rows at a time. A's columns are
// the MFMA's row operand, gathered once per wave (A^T is not in memory);
// channel 32 j + 8 g + 4 h + i is row 4 g + i of product (j, h), so that a lane
// ends with 8 neighbouring channels of its row.
struct LoraDx {
  const bf16* dt;  // [M, R]
  const bf16* a;
  bf16* dx;
  int64_t M;
  int K, R, rows;  // rows per workgroup
};

template <int NS>  // 32 ranks per step
__global__ __launch_bounds__(256) void lora8_dx_kernel(LoraDx p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int k0 = blockIdx.x * 128;
  bf16x8 w[4][2][NS];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 32 * j + 8 * (li >> 2) + 4 * h + (li & 3);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        bf16x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int rank = 32 * s + 8 * g + e;
          v[e] = rank < p.R && k < p.K ? p.a[(int64_t)rank * p.K + k] : (bf16)0.f;
        }
        w[j][h][s] = v;
      }
    }
  const int64_t begin = (int64_t)blockIdx.y * p.rows, end = min(p.M, begin + p.rows);
  for (int64_t r0 = begin + 16 * wave; r0 < end; r0 += 64) {
    const int64_t row = min(r0 + li, p.M - 1);
    bf16x8 d[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int rank = 32 * s + 8 * g;
      u32x4 v = u32x4{0, 0, 0, 0};
      if (rank < p.R) v = ld16(p.dt + row * p.R + rank);
      d[s] = __builtin_bit_cast(bf16x8, v);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4v o[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        o[h] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s)
          o[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j][h][s], d[s], o[h], 0, 0, 0);
      }
      const int k = k0 + 32 * j + 8 * g;
      if (r0 + li < end && k < p.K)
        st16(p.dx + (r0 + li) * p.K + k, u32x4{pack_bf16(o[0][0], o[0][1]), pack_bf16(o[0][2], o[0][3]),
                                               pack_bf16(o[1][0], o[1][1]), pack_bf16(o[1][2], o[1][3])});
    }
  }
}

// dA = dt^T kept(x): a workgroup takes 256 channels and a range of rows, its
// four waves 32 rows each in turn. Lane l reads 16 channels (16 (l % 16)) of
// rows 8 (l / 16) .. + 7: product j of 16 takes channel 16 li + j of every
// lane, the rows as the contracted index. dt comes transposed through LDS,
// 128 rows at a time. Partial sums per range of rows, in fp32, are added by
// lora8_da_sum_kernel (or, of one range, written as they are).
struct LoraDa {
  const bf16* dt;
  const uint8_t* codes;
  const uint8_t* exps;
  float* part;  // [splits][R][K]
  bf16* da;     // [R][K], written here when splits == 1
  int64_t M, Mp;
  int K, R, G, rows, splits;
};

constexpr int kDaWaves = 4;
constexpr int kDaThreads = 64 * kDaWaves;
constexpr int kDaRows = 32 * kDaWaves;  // rows of a turn
constexpr int kDaPitch = kDaRows + 8;   // bf16 elements per rank in LDS

template <int NR>
__global__ __launch_bounds__(kDaThreads) void lora8_da_kernel(LoraDa p) {
  constexpr int kDt = 16 * NR * kDaPitch * 2;
  constexpr int kSum = kDaWaves * 64 * 16 * NR * 4;  // one rank row i of every wave at a time
  __shared__ __attribute__((aligned(16))) uint8_t lds[kDt > kSum ? kDt : kSum];
  bf16* dts = reinterpret_cast<bf16*>(lds);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int col = blockIdx.x * 256 + 16 * li;
  const int grp = min(col / kGroup, p.G - 1);
  const bool in = col < kGroup * p.G;  // the codes' rows are padded to whole groups
  const int64_t begin = (int64_t)blockIdx.y * p.rows, end = min(p.M, begin + p.rows);
  f32x4v acc[16][NR];
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[j][n] = f32x4v{0.f, 0.f, 0.f, 0.f};
  for (int64_t r0 = begin; r0 < end; r0 += kDaRows) {
    const int64_t mine = r0 + 32 * wave + 8 * g;  // this lane's 8 rows
    u32x4 c[8];
    uint32_t ex[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = u32x4{0, 0, 0, 0};
      if (in && mine + e < end) c[e] = ld16(p.codes + (mine + e) * (kGroup * p.G) + col);
    }
    if (mine < end) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p.exps + (int64_t)grp * p.Mp + mine);
      ex[0] = v[0];
      ex[1] = v[1];
    }
    __syncthreads();  // the turn before has read its dt
    for (int o = tid; o < kDaRows * 2 * NR; o += kDaThreads) {
      const int r = o / (2 * NR), rank = 8 * (o % (2 * NR));
      u32x4 v = u32x4{0, 0, 0, 0};
      if (r0 + r < end && rank < p.R) v = ld16(p.dt + (r0 + r) * p.R + rank);
      const bf16x8 b = __builtin_bit_cast(bf16x8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) dts[(rank + e) * kDaPitch + r] = b[e];
    }
    __syncthreads();
    float step[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // Rows past the range count nothing, whatever their group's mark.
      step[e] = mine + e < end ? step_of((ex[e >> 2] >> (8 * (e & 3))) & 255u) : 0.f;
    }
    bf16x8 d[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
      d[n] = *reinterpret_cast<const bf16x8*>(dts + (16 * n + li) * kDaPitch + 32 * wave + 8 * g);
    static_for<0, 16>([&](auto J) {
      constexpr int j = decltype(J)::value;
      u32x4 v;
      static_for<0, 4>([&](auto E) {
        constexpr int e = 2 * decltype(E)::value;
        v[e / 2] = pack_bf16(byte_f<j & 3>(c[e][j >> 2]) * step[e], byte_f<j & 3>(c[e + 1][j >> 2]) * step[e + 1]);
      });
      const bf16x8 xv = __builtin_bit_cast(bf16x8, v);
#pragma unroll
      for (int n = 0; n < NR; ++n) acc[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(d[n], xv, acc[j][n], 0, 0, 0);
    });
  }
  // acc[j][n]: lane li is channel 16 li + j, element i is rank 16 n + 4 g + i.
  // Added over the waves one element i at a time: sums[wave][n][g][256 channels].
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4v*>(sums + ((wave * NR + n) * 4 + g) * 256 + 16 * li + 4 * q) =
            f32x4v{acc[4 * q][n][i], acc[4 * q + 1][n][i], acc[4 * q + 2][n][i], acc[4 * q + 3][n][i]};
    __syncthreads();
    const int k = blockIdx.x * 256 + tid;
    if (k < p.K) {
#pragma unroll
      for (int m = 0; m < NR * 4; ++m) {
        const int rank = 16 * (m >> 2) + 4 * (m & 3) + i;
        if (rank >= p.R) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kDaWaves; ++w) s += sums[(w * NR * 4 + m) * 256 + tid];
        if (p.splits == 1) p.da[(int64_t)rank * p.K + k] = (bf16)s;
        else p.part[((int64_t)blockIdx.y * p.R + rank) * p.K + k] = s;
      }
    }
  }
}

// Adds the ranges' partial sums in order, eight values per lane.
__global__ __launch_bounds__(64) void lora8_da_sum_kernel(const float* part, bf16* da, int64_t n, int splits) {
  const int64_t at = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 4;
  if (at >= n) return;  // n = R K is a multiple of 64
  f32x4v s = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < splits; ++i) s += *reinterpret_cast<const f32x4v*>(part + i * n + at);
  *reinterpret_cast<u32x2*>(da + at) = u32x2{pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3])};
}

// Ranges of rows of the dA product: enough workgroups for the device, but at
// least 256 rows each (a partial sum is 4 R bytes a channel, 256 rows' codes
// are 256).
static int da_splits(int64_t M, int64_t K) {
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t tiles = (K + 255) / 256;
  const int64_t want = (2 * cus + tiles - 1) / tiles;
  return (int)std::clamp<int64_t>(std::min(want, (M + 255) / 256), 1, 65535);
}

static int check_rows(const char* what, int64_t M, int64_t K, int dtype) {
  const std::string w = what;
  if (dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, w + ": only bf16 activations are implemented");
  if (M < 0 || K <= 0) return fail(AA_EINVAL, w + ": bad rows/K");
  if (K % 8 != 0 || K > 65536)
    return fail(AA_EUNSUPPORTED, w + ": K must be a multiple of 8 and at most 65536");
  if (M > 0x7fffff00) return fail(AA_EUNSUPPORTED, w + ": too many rows");
  return AA_OK;
}

static int check_rank(const char* what, int64_t R) {
  if (R <= 0 || R % 8 != 0 || R > kLoMaxR)
    return fail(AA_EUNSUPPORTED, std::string(what) + ": the rank must be a multiple of 8 and at most 64");
  return AA_OK;
}

}  // namespace aa

using namespace aa;

extern "C" int aa_gelu8_fwd(const void* x, void* y, void* codes, void* exps, int64_t rows, int64_t K,
                            int dtype, void* stream) {
  clear_error();
  if (int rc = check_rows("gelu8", rows, K, dtype)) return rc;
  if (rows == 0) return AA_OK;
  if (!x || !y || (codes && !exps)) return fail(AA_EINVAL, "gelu8: null pointer");
  if (!aligned16(x) || !aligned16(y) || !aligned16(codes))
    return fail(AA_EINVAL, "gelu8: pointers must be 16-byte aligned");
  GeluFwd p;
  p.x = (const bf16*)x;
  p.y = (bf16*)y;
  p.codes = (uint8_t*)codes;
  p.exps = (uint8_t*)exps;
  p.K = (int)K;
  p.upr = 2 * (int)((K + kGroup - 1) / kGroup);
  p.units = rows * p.upr;
  const int64_t blocks = (p.units + kGeThreads - 1) / kGeThreads;
  if (blocks > 0x7fffffff) return fail(AA_EUNSUPPORTED, "gelu8: too many values");
  hipStream_t st = (hipStream_t)stream;
  if (K % kGroup == 0) gelu8_fwd_kernel<true><<<dim3((unsigned)blocks), kGeThreads, 0, st>>>(p);
  else gelu8_fwd_kernel<false><<<dim3((unsigned)blocks), kGeThreads, 0, st>>>(p);
  return check_launch("gelu8");
}

extern "C" int aa_gelu8_bwd(const void* dy, const void* codes, const void* exps, void* dx, int64_t rows,
                            int64_t K, int dtype, void* stream) {
  clear_error();
  if (int rc = check_rows("gelu8_bwd", rows, K, dtype)) return rc;
  if (rows == 0) return AA_OK;
  if (!dy || !codes || !exps || !dx) return fail(AA_EINVAL, "gelu8_bwd: null pointer");
  if (!aligned16(dy) || !aligned16(dx) || !aligned16(codes))
    return fail(AA_EINVAL, "gelu8_bwd: pointers must be 16-byte aligned");
  GeluBwd p;
  p.dy = (const bf16*)dy;
  p.codes = (const uint8_t*)codes;
  p.exps = (const uint8_t*)exps;
  p.dx = (bf16*)dx;
  p.K = (int)K;
  p.upr = 2 * (int)((K + kGroup - 1) / kGroup);
  p.units = rows * p.upr;
  const int64_t blocks = (p.units + kGeThreads - 1) / kGeThreads;
  if (blocks > 0x7fffffff) return fail(AA_EUNSUPPORTED, "gelu8_bwd: too many values");
  hipStream_t st = (hipStream_t)stream;
  if (K % kGroup == 0) gelu8_bwd_kernel<true><<<dim3((unsigned)blocks), kGeThreads, 0, st>>>(p);
  else gelu8_bwd_kernel<false><<<dim3((unsigned)blocks), kGeThreads, 0, st>>>(p);
  return check_launch("gelu8_bwd");
}

template <int RT>
static void launch_lora_fwd(dim3 grid, hipStream_t st, const LoraFwd& p) {
  if (p.R <= 16) lora8_fwd_kernel<1, RT><<<grid, kLoThreads, 0, st>>>(p);
  else if (p.R <= 32) lora8_fwd_kernel<2, RT><<<grid, kLoThreads, 0, st>>>(p);
  else if constexpr (RT == 1) {
    if (p.R <= 48) lora8_fwd_kernel<3, RT><<<grid, kLoThreads, 0, st>>>(p);
    else lora8_fwd_kernel<4, RT><<<grid, kLoThreads, 0, st>>>(p);
  }
}

extern "C" int aa_lora8_fwd(const void* x, const void* a, void* t, void* codes, void* exps, int64_t M,
                            int64_t K, int64_t R, int dtype, void* stream) {
  clear_error();
  if (int rc = check_rows("lora8", M, K, dtype)) return rc;
  if (int rc = check_rank("lora8", R)) return rc;
  if (M == 0) return AA_OK;
  if (!x || !a || !t || (codes && !exps)) return fail(AA_EINVAL, "lora8: null pointer");
  if (!aligned16(x) || !aligned16(a) || !aligned16(t) || !aligned16(codes) || !aligned16(exps))
    return fail(AA_EINVAL, "lora8: pointers must be 16-byte aligned");
  LoraFwd p;
  p.x = (const bf16*)x;
  p.a = (const bf16*)a;
  p.t = (bf16*)t;
  p.codes = (uint8_t*)codes;
  p.exps = (uint8_t*)exps;
  p.M = M;
  p.Mp = (M + 15) / 16 * 16;
  p.K = (int)K;
  p.R = (int)R;
  p.G = (int)((K + kGroup - 1) / kGroup);
  const int64_t cus = std::max(1, device_cu_count());
  hipStream_t st = (hipStream_t)stream;
  if (M >= 32 * cus && R <= 32) launch_lora_fwd<2>(dim3((unsigned)((M + 31) / 32)), st, p);
  else launch_lora_fwd<1>(dim3((unsigned)((M + 15) / 16)), st, p);
  return check_launch("lora8");
}

extern "C" size_t aa_lora8_bwd_workspace(int64_t M, int64_t K, int64_t R) {
  if (M <= 0 || K <= 0 || R <= 0) return 0;
  const int64_t splits = da_splits(M, K);
  return splits == 1 ? 0 : (size_t)(splits * R * K) * sizeof(float);
}

extern "C" int aa_lora8_bwd(const void* dt, const void* a, const void* codes, const void* exps, void* dx,
                            void* da, void* workspace, size_t workspace_bytes, int64_t M, int64_t K,
                            int64_t R, int dtype, void* stream) {
  clear_error();
  if (int rc = check_rows("lora8_bwd", M, K, dtype)) return rc;
  if (int rc = check_rank("lora8_bwd", R)) return rc;
  if (M == 0) return da ? fail(AA_EINVAL, "lora8_bwd: no rows to sum over") : AA_OK;
  if (!dt || (dx && !a) || (da && (!codes || !exps))) return fail(AA_EINVAL, "lora8_bwd: null pointer");
  for (const void* q : {dt, a, codes, exps, (const void*)dx, (const void*)da, (const void*)workspace})
    if (!aligned16(q)) return fail(AA_EINVAL, "lora8_bwd: pointers must be 16-byte aligned");
  const size_t need = da ? aa_lora8_bwd_workspace(M, K, R) : 0;
  if (need && (!workspace || workspace_bytes < need)) return fail(AA_EINVAL, "lora8_bwd: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  const int64_t cus = std::max(1, device_cu_count());
  if (dx) {
    LoraDx p;
    p.dt = (const bf16*)dt;
    p.a = (const bf16*)a;
    p.dx = (bf16*)dx;
    p.M = M;
    p.K = (int)K;
    p.R = (int)R;
    const int64_t tiles = (K + 127) / 128;
    const int64_t per = (M * tiles + 4 * cus - 1) / (4 * cus);
    p.rows = (int)((std::clamp<int64_t>(per, std::max<int64_t>(64, (M + 65534) / 65535), 1 << 20) + 63) / 64 * 64);
    const dim3 grid((unsigned)tiles, (unsigned)((M + p.rows - 1) / p.rows));
    if (R <= 32) lora8_dx_kernel<1><<<grid, 256, 0, st>>>(p);
    else lora8_dx_kernel<2><<<grid, 256, 0, st>>>(p);
    if (int rc = check_launch("lora8_bwd")) return rc;
  }
  if (!da) return AA_OK;
  LoraDa p;
  p.dt = (const bf16*)dt;
  p.codes = (const uint8_t*)codes;
  p.exps = (const uint8_t*)exps;
  p.part = (float*)workspace;
  p.da = (bf16*)da;
  p.M = M;
  p.Mp = (M + 15) / 16 * 16;
  p.K = (int)K;
  p.R = (int)R;
  p.G = (int)((K + kGroup - 1) / kGroup);
  p.splits = da_splits(M, K);
  // Ranges of whole turns' rows; the last ones may be empty and write zeros.
  p.rows = (int)(((M + p.splits - 1) / p.splits + kDaRows - 1) / kDaRows * kDaRows);
  const dim3 grid((unsigned)((K + 255) / 256), (unsigned)p.splits);
  if (R <= 16) lora8_da_kernel<1><<<grid, kDaThreads, 0, st>>>(p);
  else if (R <= 32) lora8_da_kernel<2><<<grid, kDaThreads, 0, st>>>(p);
  else if (R <= 48) lora8_da_kernel<3><<<grid, kDaThreads, 0, st>>>(p);
  else lora8_da_kernel<4><<<grid, kDaThreads, 0, st>>>(p);
  if (int rc = check_launch("lora8_bwd")) return rc;
  if (p.splits == 1) return AA_OK;
  const int64_t n = R * K;
  lora8_da_sum_kernel<<<dim3((unsigned)((n / 4 + 63) / 64)), 64, 0, st>>>(p.part, p.da, n, p.splits);
  return check_launch("lora8_bwd");
}
