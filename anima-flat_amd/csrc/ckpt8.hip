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
//   2 + 2 + 33/32 bytes a value forward, 33/32 + 2 + 2 backward. 4096 x 8192: 33 and
//   34 us, 5.1 and 5.0 TB/s, a copy's rate.
// lora_down8: t = x A^T for A [R, K], R <= 64; dx = dt A; dA = dt^T kept(x).
//   HBM bound: 2 + 33/32 bytes a value forward, 2 (dx) + 33/32 (dA) backward, the
//   latter beside the vector instructions that unpack the codes.
#include <algorithm>
#include <type_traits>

#include "aa_common.h"
#include "block_math.h"
#include "tile_io.h"

namespace aa {

constexpr int kGroup = 32;          // channels per step
constexpr uint32_t kNotFinite = 255;

// The biased exponent of the step of a group whose largest magnitude has these
// bits.
__device__ __forceinline__ uint32_t step_exp(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 6;  // amax in [2^(e' - 127), 2^(e' - 126))
  return amax_bits >= kInfBits ? kNotFinite : (uint32_t)max(e, 1);
}
// The bits of the largest magnitude of a group that four neighbouring lanes hold
// 8 values each of, from the packed bf16: as 16-bit integers, magnitudes keep
// their order and NaN stands above infinity.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t packed_max(uint32_t a, uint32_t b) {
  const u16x2 x = __builtin_bit_cast(u16x2, a), y = __builtin_bit_cast(u16x2, b);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}
__device__ __forceinline__ uint32_t lane_amax(u32x4 w) {
  const uint32_t m = 0x7fff7fffu;
  return packed_max(packed_max(w[0] & m, w[1] & m), packed_max(w[2] & m, w[3] & m));
}
// The larger of a packed pair, as the bits of a float.
__device__ __forceinline__ uint32_t pair_amax(uint32_t top) { return max(top << 16, top & 0xffff0000u); }
__device__ __forceinline__ uint32_t group_amax(u32x4 w) {
  uint32_t top = pair_amax(lane_amax(w));
  top = max(top, dpp_mov<kDppXor1>(top));
  return max(top, dpp_mov<kDppXor2>(top));
}

// step, and 1 / step (both exact: 1 <= exponent <= 248).
__device__ __forceinline__ float step_of(uint32_t e) {
  return __uint_as_float(e == kNotFinite ? 0x7fc00000u : e << 23);
}
__device__ __forceinline__ float inv_step_of(uint32_t e) { return __uint_as_float((254u - e) << 23); }

// Codes of 8 values: v * inv is exact (a power of two), so the FMA's one
// rounding is that to an integer. An exponent above 253 needs an inverse step below the
// normal range, which cannot occur for finite values (e <= 248); for a marked
// group the codes are never read as numbers.
__device__ __forceinline__ u32x2 codes8(const float* v, float inv) {
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    c[i] = __float_as_uint(__builtin_amdgcn_fmed3f(fmaf(v[i], inv, kRoundMagic), kRoundMagic - 127.0f, kRoundMagic + 127.0f));
  return u32x2{low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
}
// 127 less each of four codes, as unsigned bytes, which one instruction each converts:
// all but a byte's sign flipped. The empty asm keeps that on the word: left alone, the
// compiler flips every byte by itself.
__device__ __forceinline__ uint32_t below_top(uint32_t w) {
  w ^= 0x7f7f7f7fu;
  asm("" : "+v"(w));
  return w;
}
// The value of a code of 127: finite for every step (128 of the largest, 2^121, are not).
__device__ __forceinline__ float top_of(float step) { return 127.0f * step; }
// code * step of byte kByte of below_top(codes), with top = top_of(step): 127 step -
// (127 - code) step, exact in the FMA since code * step has at most 7 significant bits.
template <int kByte>
__device__ __forceinline__ float kept_value(uint32_t below, float step, float top) {
  return fmaf((float)((below >> (8 * kByte)) & 255u), -step, top);
}

// -------------------------------------------------------------------- GELU --

constexpr int kGeThreads = 256;
constexpr int kGeChunks = 4;  // per lane

// Chunks of 8 values, a lane's kGeChunks at a stride of the workgroup, so that
// every load and store of a wave covers whole cache lines (with 16 neighbouring
// values a lane, each store half of every other 32 bytes, nontemporal stores
// took twice the time); a group of 32 is four neighbouring lanes. Rows are cut
// into 4 G chunks (G = ceil(K / 32)); codes have the row stride 32 G. With kFlat
// (K % 32 == 0) rows follow one another without gaps and a chunk's index is its
// place.
struct GeluFwd {
  const bf16* x;
  bf16* y;
  uint8_t* codes;  // [rows][32 G], or null: no checkpoint
  uint8_t* exps;   // [rows][G]
  int64_t chunks;
  int K, cpr;  // chunks per row
};

// Element index of chunk c, or -1 past its row's end.
template <bool kFlat>
__device__ __forceinline__ int64_t chunk_at(int64_t c, int K, int cpr) {
  if constexpr (kFlat) return 8 * c;
  const int64_t row = c / cpr;
  const int k = 8 * (int)(c - row * cpr);
  return k < K ? row * K + k : -1;
}

template <bool kFlat>
__global__ __launch_bounds__(kGeThreads) void gelu8_fwd_kernel(GeluFwd p) {
  const int64_t first = (int64_t)blockIdx.x * (kGeThreads * kGeChunks) + threadIdx.x;
  u32x4 raw[kGeChunks];
  int64_t at[kGeChunks];
#pragma unroll
  for (int i = 0; i < kGeChunks; ++i) {
    const int64_t c = first + kGeThreads * i;
    at[i] = c < p.chunks ? chunk_at<kFlat>(c, p.K, p.cpr) : -1;
    raw[i] = u32x4{0, 0, 0, 0};
    if (at[i] >= 0) raw[i] = ld16(p.x + at[i]);
  }
#pragma unroll
  for (int i = 0; i < kGeChunks; ++i) {
    const int64_t c = first + kGeThreads * i;
    float v[8];
    unpack8(raw[i], v);
    if (p.codes) {
      const uint32_t e = step_exp(group_amax(raw[i]));
      if (c < p.chunks) {  // chunks come in fours: all lanes of a group
        __builtin_nontemporal_store(codes8(v, inv_step_of(e)), reinterpret_cast<u32x2*>(p.codes + 8 * c));
        if ((threadIdx.x & 3) == 0) p.exps[c >> 2] = (uint8_t)e;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = gelu(v[j]);
    if (at[i] >= 0) st16_nt(p.y + at[i], pack8(v));
  }
}

struct GeluBwd {
  const bf16* dy;
  const uint8_t* codes;
  const uint8_t* exps;
  bf16* dx;
  int64_t chunks;
  int K, cpr;
};

template <bool kFlat>
__global__ __launch_bounds__(kGeThreads) void gelu8_bwd_kernel(GeluBwd p) {
  const int64_t first = (int64_t)blockIdx.x * (kGeThreads * kGeChunks) + threadIdx.x;
  u32x4 raw[kGeChunks];
  u32x2 code[kGeChunks];
  uint32_t e[kGeChunks];
  int64_t at[kGeChunks];
#pragma unroll
  for (int i = 0; i < kGeChunks; ++i) {
    const int64_t c = first + kGeThreads * i;
    at[i] = c < p.chunks ? chunk_at<kFlat>(c, p.K, p.cpr) : -1;
    if (at[i] >= 0) {
      raw[i] = ld16(p.dy + at[i]);
      code[i] = *reinterpret_cast<const u32x2*>(p.codes + 8 * c);
      e[i] = p.exps[c >> 2];
    }
  }
#pragma unroll
  for (int i = 0; i < kGeChunks; ++i) {
    if (at[i] < 0) continue;
    const float step = step_of(e[i]), top = top_of(step);
    float g[8];
    unpack8(raw[i], g);
    const uint32_t c[2] = {below_top(code[i][0]), below_top(code[i][1])};
    static_for<0, 8>([&](auto J) {
      constexpr int j = decltype(J)::value;
      g[j] *= gelu_slope(kept_value<j & 3>(c[j >> 2], step, top));
    });
    st16_nt(p.dx + at[i], pack8(g));
  }
}

// -------------------------------------------------------------------- LoRA --

constexpr int kLoMaxR = 64;

// t = x A^T and the checkpoint of x, in one pass over x. A workgroup takes 2048
// channels (1024 above rank 48), its 16 (8) waves 128 each, and tiles of 16 rows in turn. A wave keeps
// its part of A in registers, loads its 16 x 128 part of x as whole lines (lane
// l: row i + 4 (l / 16), channels 8 (l % 16)), so that a group of 32 channels is
// four neighbouring lanes, and codes and stores it from there; x crosses to the
// MFMA's operand layout through a tile of LDS that the wave has to itself (row
// r's 16-byte chunk c in slot c ^ r). The waves' 16 x R sums then go to the same
// place, and after a barrier four waves, others from tile to tile, add them in a
// fixed order. Two such places in turn, so one barrier a tile. With more channels
// than one workgroup takes, the sums of the ranges leave in fp32 for lora8_sum_kernel.
// Forms measured before, 7904 x 8192 at rank 40 (floor 28 us): every wave with
// rows and channels of its own and A from memory in the operand layout 79 us
// (A's traffic, 16 ranks x 64 bytes an instruction); A's part of a step through
// LDS, shared by 32 rows, 58 us (LDS and vector work between barriers). This one: 42
// (38 at rank 16; 196 MB: 4.7 and 5.2 TB/s, a copy's rate 5.1).
struct LoraFwd {
  const bf16* x;  // [M, K]
  const bf16* a;  // [R, K]
  bf16* t;        // [M, R], written here when splits == 1
  float* part;    // [splits][M][R]
  uint8_t* codes;  // [M][32 G], or null
  uint8_t* exps;   // [G][Mp], Mp = M up to a multiple of 16
  int64_t M, Mp;
  int K, R, G;
  int splits;  // ranges of channels
  int tiles;   // tiles of 16 rows per workgroup
};

constexpr int kLoSlice = 128;
// Waves of a workgroup: A's part takes 16 registers per 16 ranks, and 64 do not
// fit beside the rest of 16 waves' 128.
constexpr int lora_waves(int64_t R) { return R <= 48 ? 16 : 8; }
constexpr int lora_splits(int64_t K, int64_t R) {
  return (int)((K + kLoSlice * lora_waves(R) - 1) / (kLoSlice * lora_waves(R)));
}

typedef float f32x4v __attribute__((ext_vector_type(4)));

template <int NR>
__global__ __launch_bounds__(64 * lora_waves(16 * NR)) void lora8_fwd_kernel(LoraFwd p) {
  constexpr int kLoWaves = lora_waves(16 * NR);
  constexpr int kLoRange = kLoSlice * kLoWaves;
  constexpr int kTile = 16 * kLoSlice * 2;  // >= NR KiB of sums
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][kLoWaves][kTile];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int k0 = blockIdx.y * kLoRange + kLoSlice * wave;  // the wave's channels
  const int col = k0 + 8 * li;                             // this lane's
  const bool in = col < p.K;
  const bool keep = p.codes && col < kGroup * p.G;

  bf16x8 a[4][NR];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int rank = 16 * n + li, k = k0 + 32 * s + 8 * g;
      u32x4 v = u32x4{0, 0, 0, 0};
      if (rank < p.R && k < p.K) v = ld16(p.a + (int64_t)rank * p.K + k);
      a[s][n] = __builtin_bit_cast(bf16x8, v);
    }
  const int64_t first = (int64_t)blockIdx.x * p.tiles;
  const int tiles = (int)min<int64_t>(p.tiles, p.Mp / 16 - first);
  u32x4 x[4];
  // Addresses: a uniform base per tile and 32-bit offsets (15 rows of at most 65536).
  const uint32_t pitch = kGroup * p.G;
  auto load = [&](int64_t row0) {  // rows past M re-read the last
    const bf16* base = p.x + row0 * p.K;
    const int last = (int)min<int64_t>(15, p.M - 1 - row0);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = u32x4{0, 0, 0, 0};
    if (in) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = ld16(base + ((uint32_t)(min(i + 4 * g, last) * p.K) + (uint32_t)col));
    }
  };
  load(16 * first);
  for (int it = 0; it < tiles; ++it) {
    const int64_t row0 = 16 * (first + it);
    uint8_t* tile = lds[it & 1][wave];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i + 4 * g;
      *reinterpret_cast<u32x4*>(tile + r * 256 + ((li ^ r) * 16)) = x[i];
    }
    if (p.codes) {
      uint8_t* codes = p.codes + row0 * pitch;
      const int rows = keep ? (int)min<int64_t>(16, p.M - row0) : 0;
      uint32_t ex = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t e = step_exp(group_amax(x[i]));
        float v[8];
        unpack8(x[i], v);
        const u32x2 c = codes8(v, inv_step_of(e));
        if (i + 4 * g < rows) *reinterpret_cast<u32x2*>(codes + ((uint32_t)(i + 4 * g) * pitch + (uint32_t)col)) = c;
        ex |= e << (8 * i);
      }
      // Four rows' exponents; rows past M, up to Mp, are written too.
      if (keep && (lane & 3) == 0)
        *reinterpret_cast<uint32_t*>(p.exps + row0 + ((int64_t)(col / kGroup) * p.Mp + 4 * g)) = ex;
    }
    if (it + 1 < tiles) load(row0 + 16);
    f32x4v acc[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[n] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bf16x8 xv = *reinterpret_cast<const bf16x8*>(tile + li * 256 + (((4 * s + g) ^ li) * 16));
#pragma unroll
      for (int n = 0; n < NR; ++n) acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[s][n], xv, acc[n], 0, 0, 0);
    }
    // acc[n]: lane li is row li, element i is rank 16 n + 4 g + i. The wave's reads
    // of its tile come before these writes.
#pragma unroll
    for (int n = 0; n < NR; ++n) reinterpret_cast<f32x4v*>(tile)[n * 64 + lane] = acc[n];
    __syncthreads();
    const int turn = (wave - 4 * it) & (kLoWaves - 1);
    if (turn < NR) {  // this wave adds rank block `turn`
      f32x4v s = reinterpret_cast<const f32x4v*>(lds[it & 1][0])[turn * 64 + lane];
#pragma unroll
      for (int w = 1; w < kLoWaves; ++w) s += reinterpret_cast<const f32x4v*>(lds[it & 1][w])[turn * 64 + lane];
      const int64_t row = row0 + li;
      const int rank = 16 * turn + 4 * g;
      if (row < p.M && rank < p.R) {  // R is a multiple of 8
        if (p.splits == 1)
          *reinterpret_cast<u32x2*>(p.t + row * p.R + rank) = u32x2{pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3])};
        else
          *reinterpret_cast<f32x4v*>(p.part + ((int64_t)blockIdx.y * p.M + row) * p.R + rank) = s;
      }
    }
  }
}

// Workgroups of a tiles x groups grid (tiles along the channels), numbered so
// that an XCD (blocks go to the 8 in turn) takes whole runs of tiles of a few
// groups of rows. With the tiles in turn over the XCDs, an XCD wrote or read only
// every eighth piece of each row, and with rows of a power of two of bytes
// those lie in 2 to 4 of its L2's 16 channels.
static unsigned grid_blocks(int64_t n) { return (unsigned)((n + 7) / 8 * 8); }
struct Block {
  int at, of;  // this workgroup among those of its work
};
__device__ __forceinline__ bool grid_place(Block b, int tiles, int groups, int* tile, int* group) {
  const int n = (b.at & 7) * (b.of >> 3) + (b.at >> 3);
  *group = n / tiles;
  *tile = n - *group * tiles;
  return *group < groups;
}

// dx = dt A: a workgroup takes 512 channels, its four waves 128 each, and 128 rows
// of dt in LDS at a time. Product j of 8 takes channel 8 li + j of every lane as
// its column (A's rows are loaded as 256-byte pieces, eight ranks' 8 channels a
// lane, and transposed in registers) and 16 rows of dt, so that a lane ends with
// 8 neighbouring channels of rows 4 g .. 4 g + 3 and the 16 lanes of a quarter
// wave store 256 bytes of one row. With dt's rows along the lanes instead, the
// quarter waves of a store spread over 8 rows, four times as many pieces of
// lines: the CU's address unit was busy 80% of the time, 33 us at 7904 x 8192
// and rank 40 against 25.5 to 28 (4.6 to 5.1 TB/s of writes; a fill of that size
// reaches 6.2).
struct LoraDx {
  const bf16* dt;  // [M, R]
  const bf16* a;
  bf16* dx;
  int64_t M;
  int K, R, rows;  // rows per workgroup
  int tiles, groups;
};

constexpr int kDxCols = 512;
constexpr int kDxRows = 128;

template <int NS>
constexpr int dx_lds() { return kDxRows * 32 * NS * 2; }

template <int NS>  // 32 ranks per step
__device__ __forceinline__ void lora8_dx(const LoraDx& p, uint8_t* lds, Block block) {
  // dt's rows, 16-byte chunk c (8 ranks) of row r at slot c ^ (r & (4 NS - 1)).
  bf16* dts = reinterpret_cast<bf16*>(lds);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  int bx, by;
  if (!grid_place(block, p.tiles, p.groups, &bx, &by)) return;
  const int k = bx * kDxCols + 128 * wave + 8 * li;  // this lane's channels
  const bool in = k < p.K;
  bf16x8 w[8][NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    u32x4 v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int rank = 32 * s + 8 * g + e;
      v[e] = u32x4{0, 0, 0, 0};
      if (rank < p.R && in) v[e] = ld16(p.a + (int64_t)rank * p.K + k);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u32x4 t;
#pragma unroll
      for (int e = 0; e < 8; e += 2)  // the bf16 j of ranks e and e + 1
        t[e / 2] = __builtin_amdgcn_perm(v[e + 1][j / 2], v[e][j / 2], (j & 1) ? 0x07060302u : 0x05040100u);
      w[j][s] = __builtin_bit_cast(bf16x8, t);
    }
  }
  const int64_t begin = (int64_t)by * p.rows, end = min(p.M, begin + p.rows);
  for (int64_t c0 = begin; c0 < end; c0 += kDxRows) {
    const int rows = (int)min<int64_t>(kDxRows, end - c0);
    __syncthreads();  // the rows before have been read
    for (int o = tid; o < kDxRows * 4 * NS; o += 256) {
      const int r = o / (4 * NS), c = o % (4 * NS);
      u32x4 v = u32x4{0, 0, 0, 0};
      if (r < rows && 8 * c < p.R) v = ld16(p.dt + (c0 + r) * p.R + 8 * c);
      *reinterpret_cast<u32x4*>(dts + (r * 4 * NS + (c ^ (r & (4 * NS - 1)))) * 8) = v;
    }
    __syncthreads();
    for (int r0 = 0; r0 < rows; r0 += 16) {
      bf16x8 d[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int r = r0 + li, c = 4 * s + g;
        d[s] = *reinterpret_cast<const bf16x8*>(dts + (r * 4 * NS + (c ^ (r & (4 * NS - 1)))) * 8);
      }
      f32x4v q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        q[j] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s) q[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(d[s], w[j][s], q[j], 0, 0, 0);
      }
      // q[j]: lane li is channel 8 li + j, element i is row 4 g + i.
      if (in) {
        bf16* out = p.dx + (c0 + r0 + 4 * g) * p.K + k;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r0 + 4 * g + i < rows)
            st16_nt(out + (int64_t)i * p.K, u32x4{pack_bf16(q[0][i], q[1][i]), pack_bf16(q[2][i], q[3][i]),
                                                  pack_bf16(q[4][i], q[5][i]), pack_bf16(q[6][i], q[7][i])});
      }
    }
  }
}

// dA = dt^T kept(x): a workgroup takes 128 channels and a range of rows, its
// four waves 32 rows each in turn. Lane l reads 8 channels (8 (l % 16)) of rows
// 8 (l / 16) .. + 7: product j of 8 takes channel 8 li + j of every lane, the
// rows as the contracted index. dt lies in LDS as it is in memory, 128 rows at
// a time, and is read transposed. The codes, steps and dt of two turns ahead are
// loaded before this turn's products. Partial sums per range of rows, in fp32,
// are added by lora8_sum_kernel (or, of one range, written as they are). Bound by
// vector instructions: per 8 codes 8 conversions, 8 FMAs and 4 packs, with the rest
// of a turn 2.5 times a read of the codes at the memory's rate (7904 x 8192: 22 us at
// rank 16, 24 at 32, 28 at 40, 37 at 64; 67 MB in 13). Three sets of a turn's
// registers in turn, copied, and pointers per lane: 24, 26, 31, 39.
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
constexpr int kDaCols = 128;

// Row pitch in LDS: a multiple of 8 bytes whose 16-row stride spreads over the
// banks (the transposed reads take 4 rows x 32 bytes per 16 lanes).
constexpr int da_pitch(int NR) { return 16 * NR + 4; }
template <int NR>
constexpr int da_lds() {  // two turns' dt, or one element i of every wave's sums
  return std::max(2 * kDaRows * da_pitch(NR) * 2, kDaWaves * NR * 4 * kDaCols * 4);
}

template <int NR>
__device__ __forceinline__ void lora8_da(const LoraDa& p, uint8_t* lds, Block block) {
  constexpr int kPitch = da_pitch(NR);
  bf16* dts = reinterpret_cast<bf16*>(lds);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  // The codes' rows are padded to whole groups; channels past them read the last.
  int bx, by;
  if (!grid_place(block, (p.K + kDaCols - 1) / kDaCols, p.splits, &bx, &by)) return;
  const int col = min(bx * kDaCols + 8 * li, kGroup * p.G - 8);
  const int grp = col / kGroup;
  const int64_t begin = (int64_t)by * p.rows, end = min(p.M, begin + p.rows);
  f32x4v acc[8][NR];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[j][n] = f32x4v{0.f, 0.f, 0.f, 0.f};

  constexpr int kPieces = kDaRows * 4 * NR / kDaThreads;  // 8-byte pieces of dt per thread
  const uint32_t pitch = kGroup * p.G;
  struct Turn {
    u32x2 c[8];  // codes of this lane's 8 rows
    u32x2 ex;    // their groups' exponents
    u32x2 dt[kPieces];
  } even, odd;
  const int mine = 32 * wave + 8 * g;  // this lane's 8 rows
  uint32_t piece[kPieces];  // bytes of dt, in a whole turn
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int o = tid + kDaThreads * i;
    piece[i] = 2u * (uint32_t)(o / (4 * NR) * p.R + min(4 * (o % (4 * NR)), p.R - 4));
  }
  const uint32_t whole = (uint32_t)mine * pitch + (uint32_t)col;  // of this lane's first row
  auto load = [&](Turn& t, int64_t r0) {
    // Addresses: a uniform row base and 32-bit offsets in the turn's 128 rows. (The
    // empty asm keeps r0 in a scalar register: left alone, the compiler carries a
    // pointer per lane and load through the loop, 60 registers.)
    asm("" : "+s"(r0));
    const uint8_t* codes = p.codes + r0 * pitch;
    const uint8_t* exps = p.exps + (int64_t)grp * p.Mp + r0;
    const uint8_t* dt = reinterpret_cast<const uint8_t*>(p.dt + r0 * p.R);
    // Every load is in bounds and made: rows past the range re-read its last, and
    // count nothing below; channels and ranks past theirs are not written.
    if (end - r0 >= kDaRows) {
#pragma unroll
      for (int e = 0; e < 8; ++e) t.c[e] = *reinterpret_cast<const u32x2*>(codes + (int64_t)e * pitch + whole);
      t.ex = *reinterpret_cast<const u32x2*>(exps + mine);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) t.dt[i] = *reinterpret_cast<const u32x2*>(dt + piece[i]);
    } else {
      const int last = (int)(end - r0) - 1;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        t.c[e] = *reinterpret_cast<const u32x2*>(codes + ((uint32_t)min(mine + e, last) * pitch + (uint32_t)col));
      t.ex = *reinterpret_cast<const u32x2*>(exps + min(mine, last & ~7));
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int r = (tid + kDaThreads * i) / (4 * NR);
        const u32x2 v = *reinterpret_cast<const u32x2*>(dt + (piece[i] - 2u * (uint32_t)(max(r - last, 0) * p.R)));
        t.dt[i] = r <= last ? v : u32x2{0, 0};
      }
    }
  };
  // One turn of t's rows from r0; t is free for the turn after the next as soon as its
  // codes and steps are unpacked and its dt is in LDS.
  auto turn = [&](Turn& t, int64_t r0, bf16* mydt) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int o = tid + kDaThreads * i, r = o / (4 * NR), rank = 4 * (o % (4 * NR));
      *reinterpret_cast<u32x2*>(mydt + r * kPitch + rank) = t.dt[i];
    }
    float step[8], top[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) step[e] = step_of((t.ex[e >> 2] >> (8 * (e & 3))) & 255u);
    if (r0 + kDaRows > end) {  // rows past the range count nothing, whatever their group's mark
      const int left = (int)(end - r0) - mine;
#pragma unroll
      for (int e = 0; e < 8; ++e) step[e] = e < left ? step[e] : 0.f;
    }
    uint32_t code[8][2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top[e] = top_of(step[e]);
      code[e][0] = below_top(t.c[e][0]);
      code[e][1] = below_top(t.c[e][1]);
    }
    if (r0 + 2 * kDaRows < end) load(t, r0 + 2 * kDaRows);
    // One barrier a turn: these places are written again two turns on, behind the
    // next turn's barrier, which every wave reaches after its reads here.
    __syncthreads();
    // Lanes 4 r + q of a group of 16 give the piece of four ranks at 4 q of row
    // 8 g + r (+ 4 for the second read); lane li receives rank li of four rows.
    const bf16* from = mydt + (mine + (li >> 2)) * kPitch + 4 * (li & 3);
    bf16x8 d[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const s16x4 lo = ds_read_tr(from + 16 * n);
      const s16x4 hi = ds_read_tr(from + 4 * kPitch + 16 * n);
      d[n] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    static_for<0, 8>([&](auto J) {
      constexpr int j = decltype(J)::value;
      u32x4 v;
      static_for<0, 4>([&](auto E) {
        constexpr int e = 2 * decltype(E)::value;
        v[e / 2] = pack_bf16(kept_value<j & 3>(code[e][j >> 2], step[e], top[e]),
                             kept_value<j & 3>(code[e + 1][j >> 2], step[e + 1], top[e + 1]));
      });
      const bf16x8 xv = __builtin_bit_cast(bf16x8, v);
#pragma unroll
      for (int n = 0; n < NR; ++n) acc[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(d[n], xv, acc[j][n], 0, 0, 0);
    });
  };
  if (begin < end) load(even, begin);
  if (begin + kDaRows < end) load(odd, begin + kDaRows);
  for (int64_t r0 = begin; r0 < end; r0 += 2 * kDaRows) {
    turn(even, r0, dts);
    if (r0 + kDaRows < end) turn(odd, r0 + kDaRows, dts + kDaRows * kPitch);
  }
  // acc[j][n]: lane li is channel 8 li + j, element i is rank 16 n + 4 g + i.
  // Added over the waves one element i at a time: sums[wave][n][g][channel].
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        *reinterpret_cast<f32x4v*>(sums + ((wave * NR + n) * 4 + g) * kDaCols + 8 * li + 4 * q) =
            f32x4v{acc[4 * q][n][i], acc[4 * q + 1][n][i], acc[4 * q + 2][n][i], acc[4 * q + 3][n][i]};
    __syncthreads();
    const int at = tid & (kDaCols - 1), k = bx * kDaCols + at;
    if (k < p.K) {
#pragma unroll
      for (int m0 = 0; m0 < NR * 4; m0 += 2) {
        const int m = m0 + (tid >> 7);  // rank 16 n + 4 g + i with m = 4 n + g
        const int rank = 4 * m + i;
        if (rank >= p.R) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kDaWaves; ++w) s += sums[(w * NR * 4 + m) * kDaCols + at];
        if (p.splits == 1) p.da[(int64_t)rank * p.K + k] = (bf16)s;
        else p.part[((int64_t)by * p.R + rank) * p.K + k] = s;
      }
    }
  }
}

template <int NS>
__global__ __launch_bounds__(256) void lora8_dx_kernel(LoraDx p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[dx_lds<NS>()];
  lora8_dx<NS>(p, lds, {(int)blockIdx.x, (int)gridDim.x});
}
template <int NR>
__global__ __launch_bounds__(kDaThreads, NR < 4 ? 2 : 1) void lora8_da_kernel(LoraDa p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[da_lds<NR>()];
  lora8_da<NR>(p, lds, {(int)blockIdx.x, (int)gridDim.x});
}
// Both in one launch, eight workgroups (one an XCD) of each in turn: dx is bound by
// its stores and dA by the vector instructions that unpack the codes, so that a CU
// with workgroups of both does better than one after the other. 7904 x 8192, one
// launch against two: rank 16 37 against 48 us (128 MB out and 67 in: 5.3 TB/s), rank
// 32 41 against 48, rank 40 46 to 48 against 54. Above rank 48 dA's registers leave a
// CU one workgroup, of either (rank 64: 84 against 62), and two launches are made.
template <int NR>
__global__ __launch_bounds__(kDaThreads, 2) void lora8_both_kernel(LoraDx x, LoraDa a, int nx, int na) {
  constexpr int NS = (NR + 1) / 2;
  __shared__ __attribute__((aligned(16))) uint8_t lds[std::max(dx_lds<NS>(), da_lds<NR>())];
  const int u = blockIdx.x >> 3, xcd = blockIdx.x & 7;
  const int pairs = min(nx, na) >> 3;  // units of eight of each
  const bool dx = u < 2 * pairs ? (u & 1) == 0 : nx > na;
  const int at = 8 * (u < 2 * pairs ? u >> 1 : u - pairs) + xcd;
  if (dx) lora8_dx<NS>(x, lds, {at, nx});
  else lora8_da<NR>(a, lds, {at, na});
}

// Adds the ranges' partial sums of t or dA in order, four values per lane. 4 us for 5 MB
// of them: the latency of a dependent launch.
__global__ __launch_bounds__(64) void lora8_sum_kernel(const float* part, bf16* out, int64_t n, int splits) {
  const int64_t at = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 4;
  if (at >= n) return;  // n, R times K or M, is a multiple of 8
  f32x4v s = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < splits; ++i) s += *reinterpret_cast<const f32x4v*>(part + i * n + at);
  *reinterpret_cast<u32x2*>(out + at) = u32x2{pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3])};
}

// Ranges of rows of the dA product: two workgroups a CU (one above rank 48, where no
// more fit), but at least 256 rows each (a partial sum is 4 R bytes a channel, 256
// rows' codes are 256). 7904 x 8192 with an earlier form of the loop, one, two and
// four a CU: rank 16 28, 24 and 27 us; rank 40 35, 31 and (two at a time) 32; rank
// 64, one and two: 39 and 47.
static int da_splits(int64_t M, int64_t K, int64_t R) {
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t tiles = (K + kDaCols - 1) / kDaCols;
  const int64_t want = std::max<int64_t>(1, (R <= 48 ? 2 : 1) * cus / tiles);
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
  p.cpr = 4 * (int)((K + kGroup - 1) / kGroup);
  p.chunks = rows * p.cpr;
  const int64_t blocks = (p.chunks + kGeThreads * kGeChunks - 1) / (kGeThreads * kGeChunks);
  if (!grid_fits(blocks, kGeThreads)) return fail(AA_EUNSUPPORTED, "gelu8: too many values");
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
  p.cpr = 4 * (int)((K + kGroup - 1) / kGroup);
  p.chunks = rows * p.cpr;
  const int64_t blocks = (p.chunks + kGeThreads * kGeChunks - 1) / (kGeThreads * kGeChunks);
  if (!grid_fits(blocks, kGeThreads)) return fail(AA_EUNSUPPORTED, "gelu8_bwd: too many values");
  hipStream_t st = (hipStream_t)stream;
  if (K % kGroup == 0) gelu8_bwd_kernel<true><<<dim3((unsigned)blocks), kGeThreads, 0, st>>>(p);
  else gelu8_bwd_kernel<false><<<dim3((unsigned)blocks), kGeThreads, 0, st>>>(p);
  return check_launch("gelu8_bwd");
}

extern "C" size_t aa_lora8_fwd_workspace(int64_t M, int64_t K, int64_t R) {
  if (M <= 0 || K <= 0 || R <= 0) return 0;
  const int64_t splits = lora_splits(K, R);
  return splits == 1 ? 0 : (size_t)(splits * M * R) * sizeof(float);
}

extern "C" int aa_lora8_fwd(const void* x, const void* a, void* t, void* codes, void* exps,
                            void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t R,
                            int dtype, void* stream) {
  clear_error();
  if (int rc = check_rows("lora8", M, K, dtype)) return rc;
  if (int rc = check_rank("lora8", R)) return rc;
  if (M == 0) return AA_OK;
  if (!x || !a || !t || (codes && !exps)) return fail(AA_EINVAL, "lora8: null pointer");
  for (const void* q : {x, a, (const void*)t, (const void*)codes, (const void*)exps, (const void*)workspace})
    if (!aligned16(q)) return fail(AA_EINVAL, "lora8: pointers must be 16-byte aligned");
  const size_t need = aa_lora8_fwd_workspace(M, K, R);
  if (need && (!workspace || workspace_bytes < need)) return fail(AA_EINVAL, "lora8: workspace too small");
  LoraFwd p;
  p.x = (const bf16*)x;
  p.a = (const bf16*)a;
  p.t = (bf16*)t;
  p.part = (float*)workspace;
  p.codes = (uint8_t*)codes;
  p.exps = (uint8_t*)exps;
  p.M = M;
  p.Mp = (M + 15) / 16 * 16;
  p.K = (int)K;
  p.R = (int)R;
  p.G = (int)((K + kGroup - 1) / kGroup);
  p.splits = lora_splits(K, R);
  // One workgroup a CU (16 waves, 128 KiB of LDS), each with its share of the tiles.
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t tiles = p.Mp / 16, groups = std::clamp<int64_t>(cus / p.splits, 1, tiles);
  p.tiles = (int)((tiles + groups - 1) / groups);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((tiles + p.tiles - 1) / p.tiles), (unsigned)p.splits);
  if (R <= 16) lora8_fwd_kernel<1><<<grid, 64 * lora_waves(16 * 1), 0, st>>>(p);
  else if (R <= 32) lora8_fwd_kernel<2><<<grid, 64 * lora_waves(16 * 2), 0, st>>>(p);
  else if (R <= 48) lora8_fwd_kernel<3><<<grid, 64 * lora_waves(16 * 3), 0, st>>>(p);
  else lora8_fwd_kernel<4><<<grid, 64 * lora_waves(16 * 4), 0, st>>>(p);
  if (int rc = check_launch("lora8")) return rc;
  if (p.splits == 1) return AA_OK;
  const int64_t n = M * R;
  lora8_sum_kernel<<<dim3((unsigned)((n / 4 + 63) / 64)), 64, 0, st>>>(p.part, p.t, n, p.splits);
  return check_launch("lora8");
}

extern "C" size_t aa_lora8_bwd_workspace(int64_t M, int64_t K, int64_t R) {
  if (M <= 0 || K <= 0 || R <= 0) return 0;
  const int64_t splits = da_splits(M, K, R);
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
  LoraDx x;
  LoraDa p;
  unsigned nx = 0, na = 0;
  if (dx) {
    x.dt = (const bf16*)dt;
    x.a = (const bf16*)a;
    x.dx = (bf16*)dx;
    x.M = M;
    x.K = (int)K;
    x.R = (int)R;
    const int64_t tiles = (K + kDxCols - 1) / kDxCols;
    // Two workgroups a CU (one to six: within 3 us of each other at 7904 x 8192), each
    // with at least 32 rows to spend the reading of its part of A on.
    const int64_t per = (M * tiles + 2 * cus - 1) / (2 * cus);
    x.rows = (int)((std::clamp<int64_t>(per, 32, 1 << 20) + 15) / 16 * 16);
    x.tiles = (int)tiles;
    x.groups = (int)((M + x.rows - 1) / x.rows);
    nx = grid_blocks(tiles * x.groups);
  }
  if (da) {
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
    p.splits = da_splits(M, K, R);
    // Ranges of whole turns' rows; the last ones may be empty and write zeros.
    p.rows = (int)(((M + p.splits - 1) / p.splits + kDaRows - 1) / kDaRows * kDaRows);
    na = grid_blocks((K + kDaCols - 1) / kDaCols * p.splits);
  }
  const bool both = nx && na && R <= 48;
  if (both) {
    if (R <= 16) lora8_both_kernel<1><<<nx + na, kDaThreads, 0, st>>>(x, p, nx, na);
    else if (R <= 32) lora8_both_kernel<2><<<nx + na, kDaThreads, 0, st>>>(x, p, nx, na);
    else lora8_both_kernel<3><<<nx + na, kDaThreads, 0, st>>>(x, p, nx, na);
  }
  if (nx && !both) {
    if (R <= 32) lora8_dx_kernel<1><<<nx, 256, 0, st>>>(x);
    else lora8_dx_kernel<2><<<nx, 256, 0, st>>>(x);
  }
  if (na && !both) {
    if (R <= 16) lora8_da_kernel<1><<<na, kDaThreads, 0, st>>>(p);
    else if (R <= 32) lora8_da_kernel<2><<<na, kDaThreads, 0, st>>>(p);
    else if (R <= 48) lora8_da_kernel<3><<<na, kDaThreads, 0, st>>>(p);
    else lora8_da_kernel<4><<<na, kDaThreads, 0, st>>>(p);
  }
  if (int rc = check_launch("lora8_bwd")) return rc;
  if (!da) return AA_OK;
  if (p.splits == 1) return AA_OK;
  const int64_t n = R * K;
  lora8_sum_kernel<<<dim3((unsigned)((n / 4 + 63) / 64)), 64, 0, st>>>(p.part, p.da, n, p.splits);
  return check_launch("lora8_bwd");
}
