// Tokens to int8 with a scale per token, and the product of such tokens with
// int8 weights that have a scale per output channel:
//
//   s[t] = max(max_k |x[t, k]|, 1e-12) / 127, q[t, k] = round(x[t, k] / s[t])
//   y[t, n] = s[t] ws[n] sum_k q[t, k] wq[n, k]
//
// The sum is exact: int8 MFMA accumulates in int32, and K <= 65536 products of
// at most 2^14 stay below 2^31. It is then one fp32 conversion, two fp32
// products and one rounding to bf16.
//
// Tiled product (int8_linear_kernel): the projections' main loop
// (qkv_proj.hip) with 128 bytes of K per row and stage: an operand of
// v_mfma_i32_32x32x32_i8 is 16 bytes per lane, as bf16's is, with twice the K,
// so LDS blocks, XOR, DMA and k-steps are the same in bytes, at twice the
// operations per MFMA cycle.
// Many tokens (int8_linear_big_kernel): 256 x 256 tiles, for whole rounds of them.
// Some tokens (int8_mid_kernel): 64 x 64 tiles with K split over the waves.
// Few tokens (int8_skinny_kernel, up to 64): bound by reading the weights once.
#include <algorithm>
#include <type_traits>

#include "aa_common.h"
#include "block_math.h"
#include "tile_io.h"

namespace aa {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ------------------------------------------------------------------ tokens --

constexpr int kQ8Threads = 256;
constexpr int kQ8Rows = kQ8Threads / 64;  // one wave per row
constexpr int kQ8MaxK = 8192;

// One wave per row, the row in registers between its one read and the store of
// its codes: unit lane + 64 p of U values (16 where K allows 16-byte stores). HBM
// bound, 3 bytes a value; with GELU as much by its vector instructions (block_math.h).
// 18432 x 8192 with GELU 84 to 97 us (453 MB: 4.7 to 5.4 TB/s; a copy 5.1), vector
// instructions issued in 97% of a CU's cycles, 17 a value; with the GELU of two
// transcendental instructions 95 to 107; with a division per value and plain stores 131.
template <int NU, int U, bool kGelu>
__global__ __launch_bounds__(kQ8Threads) void rowquant_int8_kernel(const bf16* __restrict__ x,
                                                                   uint8_t* __restrict__ q,
                                                                   float* __restrict__ s, int rows,
                                                                   int K) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kQ8Rows + (threadIdx.x >> 6);
  if (row >= rows) return;  // whole waves; no barrier here
  const int nunit = K / U;
  const bf16* xr = x + row * K;
  u32x4 raw[NU][U / 8];
#pragma unroll
  for (int p = 0; p < NU; ++p)
    if (lane + 64 * p < nunit) {
#pragma unroll
      for (int w = 0; w < U / 8; ++w) raw[p][w] = ld16(xr + U * (lane + 64 * p) + 8 * w);
    }
  float v[NU][U];
  float top = 0.f;
#pragma unroll
  for (int p = 0; p < NU; ++p)
    if (lane + 64 * p < nunit) {
#pragma unroll
      for (int w = 0; w < U / 8; ++w) unpack8(raw[p][w], &v[p][8 * w]);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if constexpr (kGelu) v[p][i] = gelu_coarse(v[p][i]);
#pragma unroll
      for (int i = 0; i < U; i += 2) top = max3abs_nan(top, v[p][i], v[p][i + 1]);
    }
  const RowScale rs = row_scale(wave_umax(mag_bits(top)));
#pragma unroll
  for (int p = 0; p < NU; ++p)
    if (lane + 64 * p < nunit) {
      uint8_t* to = q + row * K + U * (lane + 64 * p);
      const u32x2 a = int8_codes8(&v[p][0], rs);
      if constexpr (U == 16) {
        const u32x2 b = int8_codes8(&v[p][8], rs);
        st16_nt(to, u32x4{a[0], a[1], b[0], b[1]});
      } else {
        *reinterpret_cast<u32x2*>(to) = a;
      }
    }
  if (lane == 0) s[row] = rs.s;
}

template <int NU, int U>
static void launch_rowquant(dim3 grid, hipStream_t st, const bf16* x, uint8_t* q, float* s, int rows,
                            int K, bool gelu) {
  if (gelu) rowquant_int8_kernel<NU, U, true><<<grid, kQ8Threads, 0, st>>>(x, q, s, rows, K);
  else rowquant_int8_kernel<NU, U, false><<<grid, kQ8Threads, 0, st>>>(x, q, s, rows, K);
}

// ----------------------------------------------------------------- product --

constexpr int kIK = 128;      // bytes of K per stage
// Rows of LDS of the kernels that choose k-steps by bits 5 and 6 of an address: their
// offsets alone decide these only if the array starts at a row of 128 bytes.
constexpr int kRowsAlign = 1024;
constexpr int kIGroupM = 4;   // token tiles per work-order group

struct I8Params {
  const uint8_t* x;  // [M, K]
  const float* xs;   // [M]
  const uint8_t* w;  // [N, K]
  const float* ws;   // [N]
  bf16* y;           // [M, N]
  int64_t M;
  int N, K, mtiles;
};

template <int MT, int NT, int WN, int RING>
struct I8Tile {
  static constexpr int kMT = MT;  // tokens per workgroup, 64 per wave
  static constexpr int kNT = NT;  // output channels per workgroup, WN per wave
  static constexpr int kWN = WN;
  static constexpr int kWaves = (MT / 64) * (NT / WN);
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kStage = (MT + NT) * kIK;      // bytes
  static constexpr int kBPW = (MT + NT) / 8 / kWaves;  // 8-row DMA blocks per wave and stage
  static constexpr int kCB = WN / 32;
  static constexpr int kRing = RING;
  static constexpr int kRingBytes = RING * kStage;
  static constexpr int kDmaParts = 2;
  static_assert((MT + NT) / 8 % kWaves == 0 && kBPW % 2 == 0, "DMA blocks split evenly, in pairs");
  static_assert(kRingBytes <= 160 * 1024 && MT * 256 <= kRingBytes, "LDS");
  static_assert(NT % 128 == 0 && 128 % WN == 0 || WN == 128, "128-channel sections");
};
// 64 KiB ring, two workgroups per CU, where each runs beside the other's waits: 20 to
// 23.5 us for both at K = 2048. 128 KiB ring, one per CU, bound by the latency of its
// stages: 14.4 us at K = 2048, 9.4 for 666 x 1024 -> 4096.
using I8TileC = I8Tile<128, 128, 64, 2>;
using I8TileD = I8Tile<128, 128, 64, 4>;

__device__ __forceinline__ i32x16 mfma_i8(i32x4 a, i32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

template <class T>
__global__ __launch_bounds__(T::kThreads) void int8_linear_kernel(I8Params p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::kRingBytes];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ntn = (p.N + T::kNT - 1) / T::kNT;
  const int total = p.mtiles * ntn;
  const int L = xcd_remap(blockIdx.x, total);
  const int group = L / (kIGroupM * ntn);
  const int within = L - group * kIGroupM * ntn;
  const int gm = min(kIGroupM, p.mtiles - group * kIGroupM);
  const int mt = group * kIGroupM + within % gm;
  const int nt = within / gm;
  const int64_t row0 = (int64_t)mt * T::kMT;
  const int nrows = (int)min<int64_t>(T::kMT, p.M - row0);
  const int ncols = min(T::kNT, p.N - T::kNT * nt);
  const uint8_t* xbase = p.x + row0 * p.K;
  const uint8_t* wbase = p.w + (int64_t)nt * T::kNT * p.K;

  // DMA roles as in the projections: row lane >> 3 of an 8-row block, LDS slot
  // lane & 7, which holds 16-byte chunk slot ^ (row & 7) ^ (block & 1). Rows
  // past the last re-read it.
  const int drow = lane >> 3;
  const int dchunk0 = (lane & 7) ^ drow;
  const int dchunk1 = dchunk0 ^ 1;
  const uint8_t* sbase[T::kBPW];
  uint32_t voff[T::kBPW];
#pragma unroll
  for (int i = 0; i < T::kBPW; ++i) {
    const int b = wave * T::kBPW + i;
    const bool is_x = b < T::kMT / 8;
    const int last = (is_x ? nrows : ncols) - 1;
    const int b0 = min(8 * (is_x ? b : b - T::kMT / 8), last);
    sbase[i] = (is_x ? xbase : wbase) + (int64_t)b0 * p.K;
    voff[i] = (uint32_t)(min(drow, last - b0) * p.K + 16 * ((i & 1) ? dchunk1 : dchunk0));
  }
  const uint32_t ring = lds_addr(lds) + (uint32_t)(wave * T::kBPW) * 1024u;
  // The last stage of a K that is no multiple of 128 has `tail` chunks; the
  // lanes of the chunks past them load chunk 0 instead (in bounds; their
  // products are left out or multiplied by zero below).
  const int tail = (p.K % kIK) / 16;
  const uint32_t back0 = dchunk0 >= tail ? 16u * dchunk0 : 0u;
  const uint32_t back1 = dchunk1 >= tail ? 16u * dchunk1 : 0u;
  auto issue = [&](int s, auto lo, auto hi) {
    constexpr int LO = decltype(lo)::value, HI = decltype(hi)::value;
    const int k0 = s * kIK;
    const uint32_t dst = ring + (uint32_t)((s % T::kRing) * T::kStage);
    const bool whole = p.K - k0 >= kIK;
    const uint32_t a0 = whole ? 0u : back0, a1 = whole ? 0u : back1;
    static_for<LO, HI>([&](auto I) {
      constexpr int i = decltype(I)::value;
      dma16_sva_off<0, 1024 * i>(sbase[i] + k0, voff[i] - ((i & 1) ? a1 : a0), dst);
    });
  };
  const int nk = (p.K + kIK - 1) / kIK;
  const int nfull = p.K / kIK;
  constexpr int kLead = T::kRing - 1;
  for (int s = 0; s < kLead && s < nk; ++s)
    issue(s, std::integral_constant<int, 0>{}, std::integral_constant<int, T::kBPW>{});

  constexpr int kWavesM = T::kMT / 64;
  const int wm = wave % kWavesM;
  const int wn = wave / kWavesM;
  const int li = lane & 31;
  const int hh = lane >> 5;
  const int kbase = (li >> 3) * 1024 + (li & 7) * 128 + (hh ^ (li & 7) ^ ((li >> 3) & 1)) * 16;

  i32x16 acc[T::kCB][2];
#pragma unroll
  for (int c = 0; c < T::kCB; ++c)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[c][t][e] = 0;

  constexpr int kPre = 2;
  auto stage = [&](int s, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    // This wave's DMAs of stage s are done (the kLead - 1 stages after it may be
    // in flight); the barrier publishes every wave's and retires all reads of
    // stage s - 1, whose slot stage s + kLead reuses.
    if (kLead > 1 && s + kLead - 1 < nk)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kLead - 1) * T::kBPW) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const uint8_t* stg = lds + (s % T::kRing) * T::kStage;
    const uint8_t* xs = stg + wm * 8192;
    const uint8_t* ws = stg + T::kMT * kIK + wn * T::kWN * kIK;
    i32x4 a[4][T::kCB], b[4][2];
    auto read = [&](int kk) {
      const int ko = kbase ^ (32 * kk);
#pragma unroll
      for (int c = 0; c < T::kCB; ++c) a[kk][c] = *reinterpret_cast<const i32x4*>(ws + 4096 * c + ko);
#pragma unroll
      for (int t = 0; t < 2; ++t) b[kk][t] = *reinterpret_cast<const i32x4*>(xs + 4096 * t + ko);
      if constexpr (!kWhole) {  // chunk 2 kk + hh past the row's end
        if (2 * kk + hh >= tail) b[kk][0] = b[kk][1] = i32x4{0, 0, 0, 0};
      }
    };
#pragma unroll
    for (int kk = 0; kk < kPre; ++kk) read(kk);
    auto part = [&](auto jj) {
      constexpr int j = decltype(jj)::value;
      if (s + kLead < nk)
        issue(s + kLead, std::integral_constant<int, j * T::kBPW / T::kDmaParts>{},
              std::integral_constant<int, (j + 1) * T::kBPW / T::kDmaParts>{});
    };
    part(std::integral_constant<int, 0>{});
    static_for<0, 4>([&](auto KK) {
      constexpr int kk = decltype(KK)::value;
      if constexpr (kk >= 1 && kk < T::kDmaParts) part(KK);
      if constexpr (kk + kPre < 4) read(kk + kPre);
#pragma unroll
      for (int c = 0; c < T::kCB; ++c)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[c][t] = mfma_i8(a[kk][c], b[kk][t], acc[c][t]);
    });
  };
  for (int s = 0; s < nfull; ++s) stage(s, std::true_type{});
  if (nk > nfull) stage(nfull, std::false_type{});

  // acc[c][t]: lane li is token 64 wm + 32 t + li, element e is channel
  // WN wn + 32 c + 8 (e / 4) + 4 hh + e % 4 of the tile. Scaled to bf16 and
  // staged 128 channels at a time as 256-byte rows, chunk ch of row r in slot
  // ch ^ (r & 15), for whole-line stores.
  float rs[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) rs[t] = p.xs[row0 + min(64 * wm + 32 * t + li, nrows - 1)];
  const int j = tid & 15;
  const int grp = tid >> 4;
#pragma unroll
  for (int sec = 0; sec < T::kNT / 128; ++sec) {
    __syncthreads();  // the ring (or the section before) is free
    if (T::kWN * wn / 128 == sec) {
#pragma unroll
      for (int c = 0; c < T::kCB; ++c) {
        const int col = T::kWN * wn + 32 * c;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          // N is a multiple of 8: four channels are all there or all past it.
          const int ch = min(col + 8 * e4 + 4 * hh, ncols - 4);
          const float* wsc = p.ws + nt * T::kNT + ch;
          const float w0 = wsc[0], w1 = wsc[1], w2 = wsc[2], w3 = wsc[3];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int r = 64 * wm + 32 * t + li;
            u32x2 v;
            v[0] = pack_bf16((float)acc[c][t][4 * e4] * rs[t] * w0, (float)acc[c][t][4 * e4 + 1] * rs[t] * w1);
            v[1] = pack_bf16((float)acc[c][t][4 * e4 + 2] * rs[t] * w2, (float)acc[c][t][4 * e4 + 3] * rs[t] * w3);
            const int chunk = ((col & 127) >> 3) + e4;
            *reinterpret_cast<u32x2*>(lds + r * 256 + ((chunk ^ (r & 15)) * 16) + 8 * hh) = v;
          }
        }
      }
    }
    __syncthreads();
    const int col = 128 * sec + 8 * j;
    if (col < ncols) {
      bf16* out = p.y + row0 * p.N + nt * T::kNT + col;
      for (int r = grp; r < nrows; r += T::kThreads / 16)
        st16(out + (int64_t)r * p.N, *reinterpret_cast<const u32x4*>(lds + r * 256 + ((j ^ (r & 15)) * 16)));
    }
  }
}

// The large tile: 256 tokens x 256 channels, one wave per SIMD, each with 128 x
// 128 outputs in 256 accumulator registers. Per 32 bytes of K a wave reads 8
// operands for 16 MFMAs (the 64 x 128 waves of the tiles above: 6 for 8), which
// halves the LDS reads that two waves per SIMD could not hide behind each
// other's MFMAs.
// A stage is four k-steps of 16 slots: an MFMA, and in the first eight an
// operand read of the k-step after it, in the others a DMA of a stage ahead.
// The ring holds three stages of X and two of W, 32 KiB each. The one barrier
// stands before the last k-step of stage s, whose operands are read by then: it
// publishes stage s + 1 (whose first operands are read in that k-step) and frees
// stage s's places, for W of s + 2 (its DMA goes out behind the barrier) and X of
// s + 3 (in the k-step after; it may be in flight still at the next barrier).
// K % 128 != 0: the first stage is the short one; its lanes past the rest load
// zeros.
// One workgroup a CU takes its tiles in turn. The next tile's first two stages are
// sent for behind the last operand reads of this one, ahead of its epilogue, whose
// stores then run beside the next tile's first two stages: 16384 x 8192 x 2048 (M,
// N, K; four rounds) 265 -> 252 us, two rounds 76.7 -> 75.7 and 261 -> 258.
// At K = 8192 the matrix pipe is busy for 79% of a CU's cycles, at a clock of 1.55 GHz:
// the power limit. At K = 2048 60% at 1.6 GHz: some 15000 cycles a tile go by outside
// the main loop's 33000: the epilogue's 1200 vector instructions a lane, the next tile's
// addresses and first DMAs, and the stores of all CUs at once (33 MB a round).
// 4096 x 8192 x 2048 64 to 68 us (2.0 to 2.15 POPS), 7904 x 6144 x 2048 92 to 95 (2.1),
// 18432 x 2048 x 8192 245 to 265 (2.3 to 2.5, with the rest rows' launch). Two waves per SIMD of
// 64 x 128 each, per wave two barriers a stage, 76, 102 and 319 where this form took 73 to
// 78, 98 to 106 and 258 (another box, random codes).
__device__ const u32x4 kZeroChunk = {0, 0, 0, 0};

constexpr int kBigTile = 256;
constexpr int kBigThreads = 256;
constexpr int kBigPart = kBigTile * kIK;  // bytes of X or W per stage

struct NoDma {
  template <class I>
  __device__ void operator()(I) const {}
};

__global__ __launch_bounds__(kBigThreads, 1) void int8_linear_big_kernel(I8Params p) {
  __shared__ __attribute__((aligned(kRowsAlign))) uint8_t lds[5 * kBigPart];  // X's three, W's two
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1;   // tokens 128 wm ..
  const int wn = wave >> 1;  // channels 128 wn ..
  const int ntn = (p.N + kBigTile - 1) / kBigTile;
  const int total = p.mtiles * ntn;
  const int nk = (p.K + kIK - 1) / kIK;
  const int rest = p.K - (nk - 1) * kIK;  // bytes of the first stage, 16 .. 128

  // DMA: 32 blocks of 8 rows x 128 bytes of each matrix; wave w moves blocks 8 w ..
  // 8 w + 7 of both, lane roles as above. Per block its first row's address,
  // per lane the byte offset from there.
  const uint8_t* xbase[8];
  const uint8_t* wbase[8];
  uint32_t xoff[8], woff[8];
  const uint32_t ring = lds_addr(lds);
  const uint32_t mine = ring + (uint32_t)wave * 8192u;
  // Block I of this wave's share of a stage s >= 1, X to the place at byte `at`.
  auto issue_x = [&](auto I, int s, uint32_t at) {
    constexpr int i = decltype(I)::value;
    dma16_sva_off<0, 1024 * i>(xbase[i] + (rest + (s - 1) * kIK), xoff[i], mine + at);
  };
  auto issue_w = [&](auto I, int s) {
    constexpr int i = decltype(I)::value;
    dma16_sva_off<0, 1024 * i>(wbase[i] + (rest + (s - 1) * kIK), woff[i], mine + (uint32_t)(3 + (s & 1)) * kBigPart);
  };
  // Tile `n` of the work order: its place, and its first two stages sent for.
  struct Tile {
    int64_t row0;
    int nt, nrows, ncols;
    float scale[4];  // of tokens and channels lane and lane + 64 of this wave's
  } next;
  // (The empty asm here and below keeps what follows from the lane where it is used:
  // computed once, ahead of the tiles, it would not leave room for the sums.)
  auto start = [&](int n) {
    int l = lane;
    asm volatile("" : "+v"(l));
    const int drow = l >> 3;
    const int chunk0 = (l & 7) ^ drow, chunk1 = chunk0 ^ 1;  // even and odd blocks
    const int L = xcd_remap(n, total);
    const int group = L / (kIGroupM * ntn);
    const int within = L - group * kIGroupM * ntn;
    const int gm = min(kIGroupM, p.mtiles - group * kIGroupM);
    const int mt = group * kIGroupM + within % gm;
    const int nt = within / gm;
    const int64_t row0 = (int64_t)mt * kBigTile;
    const int nrows = (int)min<int64_t>(kBigTile, p.M - row0);
    const int ncols = min(kBigTile, p.N - kBigTile * nt);
    next.row0 = row0;
    next.nt = nt;
    next.nrows = nrows;
    next.ncols = ncols;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      next.scale[h] = p.xs[row0 + min(128 * wm + 64 * h + l, nrows - 1)];
      next.scale[2 + h] = p.ws[(int64_t)nt * kBigTile + min(128 * wn + 64 * h + l, ncols - 1)];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t chunk = 16 * ((i & 1) ? chunk1 : chunk0);
      const int x0 = min(8 * (wave * 8 + i), nrows - 1), w0 = min(8 * (wave * 8 + i), ncols - 1);
      xbase[i] = p.x + (row0 + x0) * p.K;
      wbase[i] = p.w + ((int64_t)nt * kBigTile + w0) * p.K;
      xoff[i] = (uint32_t)(min(drow, nrows - 1 - x0) * p.K) + chunk;
      woff[i] = (uint32_t)(min(drow, ncols - 1 - w0) * p.K) + chunk;
    }
    static_for<0, 8>([&](auto I) {
      constexpr int i = decltype(I)::value;
      const bool in = 16 * ((i & 1) ? chunk1 : chunk0) < rest;
      dma16_a(in ? xbase[i] + xoff[i] : (const uint8_t*)&kZeroChunk, mine + 1024u * i);
      dma16_a(in ? wbase[i] + woff[i] : (const uint8_t*)&kZeroChunk, mine + 3u * kBigPart + 1024u * i);
    });
    static_for<0, 8>([&](auto I) { issue_x(I, 1, kBigPart); });
    static_for<0, 8>([&](auto I) { issue_w(I, 1); });
  };

  const int li = lane & 31, hh = lane >> 5;
  const uint32_t kbase = (li >> 3) * 1024 + (li & 7) * 128 + (hh ^ (li & 7) ^ ((li >> 3) & 1)) * 16;
  // Operand addresses of k-step kk: these ^ 32 kk (the ring and its parts are
  // aligned to 1 KiB, bits 4 to 6 are the slot's), blocks of 32 rows at + 4096.
  const uint32_t xa = ring + wm * 16384 + kbase;
  const uint32_t wa = ring + 3u * kBigPart + wn * 16384 + kbase;

  i32x16 acc[4][4];
  struct Ops {
    i32x4 v[8];  // four channel blocks, four token blocks
  } o0, o1;
  auto read = [&](auto J, Ops& o, uint32_t x, uint32_t w) {
    constexpr int j = decltype(J)::value;
    o.v[j] = __builtin_bit_cast(i32x4, lds_ld16((j < 4 ? w : x) + 4096u * (j & 3)));
  };
  // 16 MFMAs on `cur`, beside them the operands of the next k-step to `next` and
  // eight DMAs: a read and a DMA in turn (four waves' DMAs back to back would hold
  // up their MFMAs: the CU's load path takes one per ~11 cycles), or the reads in
  // the first slots where none go out.
  auto kstep = [&](const Ops& cur, Ops& next, uint32_t x, uint32_t w, auto has_next, auto dma, auto fresh) {
    constexpr int kStride = std::is_same_v<decltype(dma), NoDma> ? 1 : 2;
    static_for<0, 16>([&](auto J) {
      constexpr int j = decltype(J)::value;
      if constexpr (decltype(fresh)::value) acc[j >> 2][j & 3] = mfma_i8(cur.v[j >> 2], cur.v[4 + (j & 3)], i32x16{});
      else acc[j >> 2][j & 3] = mfma_i8(cur.v[j >> 2], cur.v[4 + (j & 3)], acc[j >> 2][j & 3]);
      if constexpr (j % kStride == 0 && j / kStride < 8 && decltype(has_next)::value) {
        // Channel block 0 and the token blocks first: the next k-step's first four MFMAs.
        constexpr int order[8] = {0, 4, 5, 6, 7, 1, 2, 3};
        read(std::integral_constant<int, order[j / kStride]>{}, next, x, w);
      }
      if constexpr (kStride == 2 && j % 2 == 1) dma(std::integral_constant<int, j / 2>{});
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  const NoDma none;
  // Places of X in the ring: of this stage, the next, and the one after, in
  // which X of stage s + 2 is sent for in this stage's first k-step.
  uint32_t px0, px1, px2;
  // The 32 stores of the tile before, made after this tile's first two stages were
  // sent for, may be in flight until the end of its second stage.
  bool stores = false;
  // left: stages after this one, as far as it matters (0, 1, 2). first: the tile's
  // first stage, whose first products start the sums.
  constexpr std::true_type kYes;
  constexpr std::false_type kNo;
  auto stage = [&](int s, auto left, auto first) {
    constexpr int kLeft = decltype(left)::value;
    const uint32_t x = xa + px0, w = wa + (uint32_t)(s & 1) * kBigPart;
    if constexpr (kLeft >= 2)
      kstep(o0, o1, x ^ 32u, w ^ 32u, kYes, [&](auto I) { issue_x(I, s + 2, px2); }, first);
    else
      kstep(o0, o1, x ^ 32u, w ^ 32u, kYes, none, first);
    kstep(o1, o0, x ^ 64u, w ^ 64u, kYes, none, kNo);
    kstep(o0, o1, x ^ 96u, w ^ 96u, kYes, none, kNo);
    if constexpr (kLeft >= 1) {
      // Every read of stage s has arrived, and this wave's DMAs of stage s + 1: only
      // X of s + 2 came after them (and, in the first stage, the stores).
      if constexpr (kLeft >= 2) {
        if (decltype(first)::value && stores) asm volatile("s_waitcnt vmcnt(40) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      const uint32_t x1 = xa + px1, w1 = wa + (uint32_t)((s + 1) & 1) * kBigPart;
      if constexpr (kLeft >= 2)
        kstep(o1, o0, x1, w1, kYes, [&](auto I) { issue_w(I, s + 2); }, kNo);
      else
        kstep(o1, o0, x1, w1, kYes, none, kNo);
      const uint32_t t = px0;
      px0 = px1;
      px1 = px2;
      px2 = t;
    } else {
      // Every wave's reads have arrived: the ring is free behind this barrier.
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      kstep(o1, o0, x, w, kNo, none, kNo);
    }
  };

  int n = blockIdx.x;
  start(n);
  for (;;) {
    const Tile tile = next;
    // This wave's DMAs of stage 0 are done (stage 1's, and the stores of the tile
    // before, may be in flight); the barrier publishes every wave's.
    if (stores) asm volatile("s_waitcnt vmcnt(48)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
    static_for<0, 8>([&](auto J) { read(J, o0, xa, wa); });
    px0 = 0, px1 = kBigPart, px2 = 2 * kBigPart;
    stage(0, std::integral_constant<int, 2>{}, kYes);
    int s = 1;
    for (; s + 2 < nk; ++s) stage(s, std::integral_constant<int, 2>{}, kNo);
    stage(s++, std::integral_constant<int, 1>{}, kNo);
    stage(s, std::integral_constant<int, 0>{}, kNo);
    n += gridDim.x;
    const bool more = n < total;
    if (more) start(n);

    // acc[c][t]: lane li is token 128 wm + 32 t + li, element e channel 128 wn + 32 c
    // + 8 (e / 4) + 4 hh + e % 4. The scales and then 16 tokens at a time go through
    // this wave's 8 KiB of X's third place (the next tile's stages are under way to
    // the others, and this wave's own DMAs are the first to write here): 256-byte
    // rows, chunk ch of row r in slot ch ^ r, stored as whole lines. A wave's LDS
    // accesses are in order.
    int l = lane, N = p.N;
    asm volatile("" : "+v"(l), "+s"(N));
    const int li = l & 31, hh = l >> 5;
    uint8_t* out = lds + 2 * kBigPart + wave * 8192;
    float* scales = reinterpret_cast<float*>(out);
#pragma unroll
    for (int h = 0; h < 4; ++h) scales[64 * h + l] = tile.scale[h];
    __builtin_amdgcn_wave_barrier();
    float rs[4];
    f32x4 ws[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) rs[t] = scales[32 * t + li];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) ws[c][e4] = *reinterpret_cast<const f32x4*>(scales + 128 + 32 * c + 8 * e4 + 4 * hh);
    const int wcols = tile.ncols - 128 * wn, wrows = tile.nrows - 128 * wm;  // what there is of the wave's
    const int j = l & 15, q = l >> 4;
    bf16* y = p.y + (tile.row0 + 128 * wm) * N + (int64_t)tile.nt * kBigTile + 128 * wn + 8 * j;
    static_for<0, 4>([&](auto T) {
      constexpr int t = decltype(T)::value;
      // The sums stay in accumulator registers until their turn.
#pragma unroll
      for (int c = 0; c < 4; ++c) asm volatile("" : "+a"(acc[c][t]));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const i32x16& v = acc[c][t];
          const f32x4 w = ws[c][e4];
          u32x2 b;
          b[0] = pack_bf16((float)v[4 * e4] * rs[t] * w[0], (float)v[4 * e4 + 1] * rs[t] * w[1]);
          b[1] = pack_bf16((float)v[4 * e4 + 2] * rs[t] * w[2], (float)v[4 * e4 + 3] * rs[t] * w[3]);
          *reinterpret_cast<u32x2*>(out + li * 256 + (((4 * c + e4) ^ (li & 15)) * 16) + 8 * hh) = b;
        }
      __builtin_amdgcn_sched_barrier(0);
      u32x4 row[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = q + 4 * i;
        row[i] = *reinterpret_cast<const u32x4*>(out + r * 256 + ((j ^ (r & 15)) * 16));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 32 * t + q + 4 * i;
        if (8 * j < wcols && r < wrows) st16(y + (int64_t)r * N, row[i]);
      }
    });
    if (!more) return;
    stores = tile.nrows == kBigTile && tile.ncols == kBigTile;  // 32 of them, in every wave
  }
}

// Few tokens (M <= 8 XB): bound by reading the weights once. A workgroup takes 16
// channels; its four waves take 128 bytes of K in turn, each through a ring of
// LDS of its own, so nothing waits for another wave until the sums: per step two
// DMAs of 8 channels x 128 bytes and XB of 8 tokens, kDepth steps ahead. 8192 x
// 8192 weights: 14.8 us for 2 tokens (67 MB: 4.5 TB/s), 14.9 for 16, 16.0 for 32,
// 20.8 for 64 (the 128 x 128 tiles: 32). Operands straight from memory (16 rows x 16
// bytes per quarter wave, four times as many pieces of lines as a DMA's two rows x
// 128): 16.2, 18.6, 25.2, 39.0; 32 channels a workgroup: 19.5, 20.1, 20.7, 23.1. In
// v_mfma_i32_16x16x64_i8 lane l holds 16 bytes of row l % 16 (a channel, a token) at
// chunk l / 16 of the 64. The waves' int32 sums are added in LDS.
constexpr int kSkinnyRows = 64;
template <int XB>
struct Skinny {
  static constexpr int kTT = (XB + 1) / 2;         // token tiles of 16
  static constexpr int kBlocks = 2 + XB;      // DMAs per step
  static constexpr int kDepth = 20 / kBlocks;      // two workgroups a CU
  static constexpr int kWaveBytes = kDepth * kBlocks * 1024;
  static constexpr int kSums = 4 * kTT * 1024;
  static constexpr int kLds = 4 * kWaveBytes > kSums ? 4 * kWaveBytes : kSums;
};

template <int XB>
__global__ __launch_bounds__(256) void int8_skinny_kernel(I8Params p) {
  using T = Skinny<XB>;
  __shared__ __attribute__((aligned(kRowsAlign))) uint8_t lds[T::kLds];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int M = (int)p.M;
  // DMA roles as above: row lane >> 3 of a block, chunk (lane & 7) ^ row ^ parity.
  const int drow = lane >> 3;
  const uint8_t* src[T::kBlocks];
#pragma unroll
  for (int i = 0; i < T::kBlocks; ++i) {
    const bool is_w = i < 2;
    const int b = is_w ? i : i - 2;
    const int64_t row = is_w ? min(n0 + 8 * b + drow, p.N - 1) : min(8 * b + drow, M - 1);
    src[i] = (is_w ? p.w : p.x) + row * p.K;
  }
  const int c0 = 16 * ((lane & 7) ^ drow), c1 = c0 ^ 16;  // bytes of even and odd blocks' chunks
  const uint32_t ring = lds_addr(lds) + (uint32_t)wave * T::kWaveBytes;
  const int nk = (p.K + kIK - 1) / kIK;
  const int n = (nk - wave + 3) / 4;  // this wave's steps
  auto issue = [&](int i) {
    const int k0 = (wave + 4 * i) * kIK;
    const uint32_t dst = ring + (uint32_t)(i % T::kDepth) * (T::kBlocks * 1024u);
#pragma unroll
    for (int j = 0; j < T::kBlocks; ++j) {
      const int k = k0 + ((j & 1) ? c1 : c0);
      // Past the row's end: zeros (K is a multiple of 16).
      dma16_a(k < p.K ? src[j] + k : (const uint8_t*)&kZeroChunk, dst + 1024u * j);
    }
  };
#pragma unroll
  for (int i = 0; i < T::kDepth; ++i)
    if (i < n) issue(i);

  i32x4 acc[T::kTT];
#pragma unroll
  for (int t = 0; t < T::kTT; ++t) acc[t] = i32x4{0, 0, 0, 0};
  // Row li of a tile at chunk g: block li >> 3 (a tile of 8 tokens has one; its rows
  // 8 to 15 are no tokens).
  const int half = li >> 3;
  const uint32_t at_w = half * 1024 + (li & 7) * 128 + (g ^ (li & 7) ^ half) * 16;
  const uint32_t at_x = XB == 1 ? (li & 7) * 128 + (g ^ (li & 7)) * 16 : at_w;
  for (int i = 0; i < n; ++i) {
    if (i + T::kDepth <= n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::kDepth - 1) * T::kBlocks) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint32_t slot = ring + (uint32_t)(i % T::kDepth) * (T::kBlocks * 1024u);
    i32x4 a[2], b[2][T::kTT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // chunks 4 h + g: bit 6 of the address
      a[h] = __builtin_bit_cast(i32x4, lds_ld16((slot + at_w) ^ (64u * h)));
#pragma unroll
      for (int t = 0; t < T::kTT; ++t)
        b[h][t] = __builtin_bit_cast(i32x4, lds_ld16((slot + 2048u + 2048u * t + at_x) ^ (64u * h)));
    }
    // The reads are back before the step kDepth on takes their place.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i + T::kDepth < n) issue(i + T::kDepth);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < T::kTT; ++t)
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[h], b[h][t], acc[t], 0, 0, 0);
  }
  __syncthreads();  // every wave is done with its ring
  i32x4* part = reinterpret_cast<i32x4*>(lds);
#pragma unroll
  for (int t = 0; t < T::kTT; ++t) part[(wave * T::kTT + t) * 64 + lane] = acc[t];
  __syncthreads();
  // Tile t: token 16 t + li, channels 4 g .. 4 g + 3.
  for (int t = wave; t < T::kTT; t += 4) {
    i32x4 s = part[t * 64 + lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) s += part[(w * T::kTT + t) * 64 + lane];
    const int tok = 16 * t + li, ch = n0 + 4 * g;
    if (tok < M && ch < p.N) {
      const float rs = p.xs[tok];
      u32x2 v;
      v[0] = pack_bf16((float)s[0] * rs * p.ws[ch], (float)s[1] * rs * p.ws[ch + 1]);
      v[1] = pack_bf16((float)s[2] * rs * p.ws[ch + 2], (float)s[3] * rs * p.ws[ch + 3]);
      *reinterpret_cast<u32x2*>(p.y + (int64_t)tok * p.N + ch) = v;
    }
  }
}

// Too few tokens or channels to fill the device with 128 x 128 tiles: 64 x 64 ones,
// whose four waves take 128 bytes of K in turn, each all 64 x 64 outputs, through 16 KiB
// of LDS of its own (8 blocks of X and of W), so that a quarter of the steps stand one
// behind another and nothing waits for another wave until the sums, which are added in
// LDS, in int32: exact. Bound by latency: a step's operands are read into registers, the
// next step's DMAs go out, and the products run beside them and beside the CU's other
// workgroup. 333 tokens, N x K = 2048 x 2048: 6.5 us (the 128 x 128 tiles 10.9), 4096 x
// 1024 7.1 (7.8), 1024 x 4096 8.0 (17.4), 2048 x 8192 15 (32); with two steps' LDS, one
// workgroup a CU: 6.8, 9.2, 8.5, 15. More than two workgroups a CU lose: 1500 tokens,
// 2048 x 2048 15.8 against 12.4.
constexpr int kMidTile = 64;
constexpr int kMidBlocks = 2 * kMidTile / 8;  // DMAs per step
constexpr int kMidStep = kMidBlocks * 1024;   // bytes

__global__ __launch_bounds__(256) void int8_mid_kernel(I8Params p) {
  __shared__ __attribute__((aligned(kRowsAlign))) uint8_t lds[4 * kMidStep];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ntn = (p.N + kMidTile - 1) / kMidTile;
  const int L = xcd_remap(blockIdx.x, p.mtiles * ntn);
  const int group = L / (kIGroupM * ntn);
  const int within = L - group * kIGroupM * ntn;
  const int gm = min(kIGroupM, p.mtiles - group * kIGroupM);
  const int64_t row0 = (int64_t)(group * kIGroupM + within % gm) * kMidTile;
  const int n0 = within / gm * kMidTile;
  const int nrows = (int)min<int64_t>(kMidTile, p.M - row0), ncols = min(kMidTile, p.N - n0);
  // DMA roles as above; rows past the last re-read it.
  const int drow = lane >> 3;
  const uint32_t c0 = 16 * ((lane & 7) ^ drow), c1 = c0 ^ 16;  // bytes of even and odd blocks' chunks
  const uint8_t* base[kMidBlocks];
  uint32_t off[kMidBlocks];
#pragma unroll
  for (int i = 0; i < kMidBlocks; ++i) {
    const bool is_x = i < kMidBlocks / 2;
    const int last = (is_x ? nrows : ncols) - 1, b0 = min(8 * (is_x ? i : i - kMidBlocks / 2), last);
    base[i] = is_x ? p.x + (row0 + b0) * p.K : p.w + (int64_t)(n0 + b0) * p.K;
    off[i] = (uint32_t)(min(drow, last - b0) * p.K) + ((i & 1) ? c1 : c0);
  }
  const uint32_t mine = lds_addr(lds) + (uint32_t)wave * kMidStep;
  const int nk = (p.K + kIK - 1) / kIK;
  const int n = (nk - wave + 3) / 4;  // this wave's steps
  auto issue = [&](int i) {
    const int k0 = (wave + 4 * i) * kIK;
    if (k0 + kIK <= p.K) {
      static_for<0, kMidBlocks>([&](auto I) {
        constexpr int j = decltype(I)::value;
        dma16_sva_off<0, 1024 * j>(base[j] + k0, off[j], mine);
      });
    } else {  // past the row's end: zeros
#pragma unroll
      for (int j = 0; j < kMidBlocks; ++j) {
        const int k = k0 + (int)((j & 1) ? c1 : c0);
        dma16_a(k < p.K ? base[j] + k0 + off[j] : (const uint8_t*)&kZeroChunk, mine + 1024u * j);
      }
    }
  };
  if (n > 0) issue(0);

  const int li = lane & 31, hh = lane >> 5;
  const uint32_t kbase = (li >> 3) * 1024 + (li & 7) * 128 + (hh ^ (li & 7) ^ ((li >> 3) & 1)) * 16;
  i32x16 acc[2][2];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[c][t][e] = 0;
  for (int i = 0; i < n; ++i) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint32_t at = mine + kbase;
    i32x4 a[4][2], b[4][2];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        b[kk][h] = __builtin_bit_cast(i32x4, lds_ld16((at ^ (32u * kk)) + 4096u * h));
        a[kk][h] = __builtin_bit_cast(i32x4, lds_ld16((at ^ (32u * kk)) + 8192u + 4096u * h));
      }
    // The reads are back before the next step takes their place.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i + 1 < n) issue(i + 1);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[c][t] = mfma_i8(a[kk][c], b[kk][t], acc[c][t]);
  }
  // acc[c][t]: lane li is token 32 t + li, element e channel 32 c + 8 (e / 4) + 4 hh +
  // e % 4. Each wave's sums as 256-byte rows of int32 in its own LDS, 16-byte chunk ch
  // of row r in slot ch ^ (r & 15); then wave w adds rows 16 w .. + 15.
  uint8_t* sums = lds + wave * kMidStep;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int r = 32 * t + li;
        const i32x16& v = acc[c][t];
        *reinterpret_cast<i32x4*>(sums + r * 256 + (((8 * c + 2 * e4 + hh) ^ (r & 15)) * 16)) =
            i32x4{v[4 * e4], v[4 * e4 + 1], v[4 * e4 + 2], v[4 * e4 + 3]};
      }
  __syncthreads();
  const int j = lane & 7;  // channels 8 j .. 8 j + 7
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * wave + 8 * i + (lane >> 3);
    i32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        s[h] += *reinterpret_cast<const i32x4*>(lds + w * kMidStep + r * 256 + (((2 * j + h) ^ (r & 15)) * 16));
    if (r < nrows && 8 * j < ncols) {
      const float rs = p.xs[row0 + r];
      const float* ws = p.ws + n0 + 8 * j;
      u32x4 v;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          v[2 * h + e] = pack_bf16((float)s[h][2 * e] * rs * ws[4 * h + 2 * e], (float)s[h][2 * e + 1] * rs * ws[4 * h + 2 * e + 1]);
      st16(p.y + (row0 + r) * p.N + n0 + 8 * j, v);
    }
  }
}

}  // namespace aa

using namespace aa;

extern "C" int aa_rowquant_int8(const void* x, int64_t rows, int64_t K, int gelu, void* q, float* s,
                                int dtype, void* stream) {
  clear_error();
  if (dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, "rowquant_int8: only bf16 input is implemented");
  if (rows < 0 || K <= 0) return fail(AA_EINVAL, "rowquant_int8: bad rows/K");
  if (K % 8 != 0 || K > kQ8MaxK)
    return fail(AA_EUNSUPPORTED, "rowquant_int8: K must be a multiple of 8 and at most 8192");
  if (rows > 0x7fffff00 || !grid_fits((rows + kQ8Rows - 1) / kQ8Rows, kQ8Threads))
    return fail(AA_EUNSUPPORTED, "rowquant_int8: too many rows");
  if (rows == 0) return AA_OK;
  if (!x || !q || !s) return fail(AA_EINVAL, "rowquant_int8: null pointer");
  if (!aligned16(x) || ((uintptr_t)q & 7u) != 0)
    return fail(AA_EINVAL, "rowquant_int8: x must be 16-byte and q 8-byte aligned");
  const dim3 grid((unsigned)((rows + kQ8Rows - 1) / kQ8Rows));
  hipStream_t st = (hipStream_t)stream;
  const bf16* xb = (const bf16*)x;
  uint8_t* qb = (uint8_t*)q;
  const int k = (int)K, n = (int)rows;
  const bool g = gelu != 0;
  if (K <= 512) {  // 8 values a lane: with 16 half the lanes or more would have none
    launch_rowquant<1, 8>(grid, st, xb, qb, s, n, k, g);
  } else if (K % 16 == 0 && aligned16(q)) {
    if (K <= 2048) launch_rowquant<2, 16>(grid, st, xb, qb, s, n, k, g);
    else if (K <= 4096) launch_rowquant<4, 16>(grid, st, xb, qb, s, n, k, g);
    else launch_rowquant<8, 16>(grid, st, xb, qb, s, n, k, g);
  } else {
    if (K <= 2048) launch_rowquant<4, 8>(grid, st, xb, qb, s, n, k, g);
    else if (K <= 4096) launch_rowquant<8, 8>(grid, st, xb, qb, s, n, k, g);
    else launch_rowquant<16, 8>(grid, st, xb, qb, s, n, k, g);
  }
  return check_launch("rowquant_int8");
}

// Times of what stands beside the large tiles, in rounds of those (37.5 us at K = 2048,
// 109 at 8192). Measured: up to 64 tokens 4 and 9 us; 64 x 64 tiles, one or two a CU,
// 6.2 and 10 at K = 2048, 11 to 15 and 27 at 8192; 128 x 128 tiles, one or two a CU, 14.4
// and 20 to 23.5 at K = 2048, 40 and 68 at 8192. Below K = 2048 a launch's fixed part weighs
// more in all of them: 64 x 64 tiles two a CU 5.6 at K = 512, 128 x 128 one a CU 6.9 (8.9 at 1024).
constexpr double kFewTime = 0.1, kMidAlone = 0.16, kMidPair = 0.26, kSmallAlone = 0.38, kSmallPair = 0.62;

extern "C" int aa_int8_linear(const void* q, const float* s, const void* weight, const float* weight_scale,
                              void* y, int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  clear_error();
  if (dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, "int8_linear: only bf16 output is implemented");
  if (M < 0 || N <= 0 || K <= 0) return fail(AA_EINVAL, "int8_linear: bad M/N/K");
  if (K % 16 != 0 || K > 65536)
    return fail(AA_EUNSUPPORTED, "int8_linear: K must be a multiple of 16 and at most 65536");
  if (N % 8 != 0 || N > (1 << 24)) return fail(AA_EUNSUPPORTED, "int8_linear: N must be a multiple of 8 and at most 2^24");
  if (M == 0) return AA_OK;
  if (!q || !s || !weight || !weight_scale || !y) return fail(AA_EINVAL, "int8_linear: null pointer");
  if (!aligned16(q) || !aligned16(weight) || !aligned16(y))
    return fail(AA_EINVAL, "int8_linear: pointers must be 16-byte aligned");
  I8Params p;
  p.x = (const uint8_t*)q;
  p.xs = s;
  p.w = (const uint8_t*)weight;
  p.ws = weight_scale;
  p.y = (bf16*)y;
  p.M = M;
  p.N = (int)N;
  p.K = (int)K;
  hipStream_t st = (hipStream_t)stream;
  const int64_t cus = std::max(1, device_cu_count());
  const auto tiles = [&](int64_t rows, int64_t size) { return (rows + size - 1) / size * ((N + size - 1) / size); };
  const auto time_without_large = [&](int64_t rows) {
    if (rows <= kSkinnyRows) return kFewTime;
    if (tiles(rows, kMidTile) <= 2 * cus) return tiles(rows, kMidTile) <= cus ? kMidAlone : kMidPair;
    const int64_t t = tiles(rows, 128);
    return t <= cus ? kSmallAlone : (double)((t + 2 * cus - 1) / (2 * cus)) * kSmallPair;
  };
  // Tokens for the large tiles: all, or what fills whole rounds of them (the rest
  // goes in a launch of its own), or none.
  const int64_t ntn = (N + kBigTile - 1) / kBigTile, mtn = (M + kBigTile - 1) / kBigTile;
  const int64_t whole = mtn * ntn / cus * cus / ntn * kBigTile;
  int64_t big = 0;
  double best = time_without_large(M);
  for (const int64_t rows : {std::min(M, whole), M}) {
    if (rows <= 0 || K <= 2 * kIK) continue;  // the large tiles' ring takes three stages or more
    const double time = (double)((tiles(rows, kBigTile) + cus - 1) / cus) + (rows < M ? time_without_large(M - rows) : 0.0);
    if (time < best) {
      best = time;
      big = rows;
    }
  }
  if (!grid_fits(tiles(M, 128), 256)) return fail(AA_EUNSUPPORTED, "int8_linear: too many tokens");
  if (big > 0) {
    p.M = big;
    p.mtiles = (int)((big + kBigTile - 1) / kBigTile);
    int8_linear_big_kernel<<<dim3((unsigned)std::min(tiles(big, kBigTile), cus)), kBigThreads, 0, st>>>(p);
    if (int rc = check_launch("int8_linear")) return rc;
    p.x += big * K;
    p.xs += big;
    p.y += big * N;
    p.M = M - big;
  }
  if (p.M == 0) return AA_OK;
  if (p.M <= kSkinnyRows) {
    const dim3 grid((unsigned)((N + 15) / 16));
    if (p.M <= 8) int8_skinny_kernel<1><<<grid, 256, 0, st>>>(p);
    else if (p.M <= 16) int8_skinny_kernel<2><<<grid, 256, 0, st>>>(p);
    else if (p.M <= 32) int8_skinny_kernel<4><<<grid, 256, 0, st>>>(p);
    else int8_skinny_kernel<8><<<grid, 256, 0, st>>>(p);
  } else if (tiles(p.M, kMidTile) <= 2 * cus) {
    p.mtiles = (int)((p.M + kMidTile - 1) / kMidTile);
    int8_mid_kernel<<<dim3((unsigned)tiles(p.M, kMidTile)), 256, 0, st>>>(p);
  } else {
    p.mtiles = (int)((p.M + 127) / 128);
    const int64_t t = tiles(p.M, 128);
    // One workgroup a CU: the deeper ring, for weights that are not in a cache (666 x
    // 1024 x 4096: 11.4 -> 9.4 us; where they are, 8.8 against 9.4).
    if (t <= cus) int8_linear_kernel<I8TileD><<<dim3((unsigned)t), I8TileD::kThreads, 0, st>>>(p);
    else int8_linear_kernel<I8TileC><<<dim3((unsigned)t), I8TileC::kThreads, 0, st>>>(p);
  }
  return check_launch("int8_linear");
}
