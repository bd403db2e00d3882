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
// Few tokens (int8_skinny_kernel, M <= 64): bound by reading the weights once.
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
// its codes: unit lane + 64 p of U values (16 where K allows 16-byte stores).
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
        if constexpr (kGelu) v[p][i] = gelu(v[p][i]);
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
using I8TileA = I8Tile<256, 256, 128, 2>;  // 128 KiB ring
using I8TileC = I8Tile<128, 128, 64, 2>;   // 64 KiB ring, two workgroups per CU
using I8TileD = I8Tile<128, 128, 64, 4>;   // 128 KiB ring

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
        st16_nt(out + (int64_t)r * p.N, *reinterpret_cast<const u32x4*>(lds + r * 256 + ((j ^ (r & 15)) * 16)));
    }
  }
}

// Few tokens: a workgroup takes 16 output channels, its four waves a quarter of
// K each (64-byte steps in turn), TT tiles of 16 tokens. Operands go from
// memory to registers: in v_mfma_i32_16x16x64_i8 lane l holds 16 bytes of row
// l % 16 (a channel's weights, a token) at chunk l / 16 of the 64. The waves'
// int32 sums are added in LDS.
template <int TT>
__global__ __launch_bounds__(256) void int8_skinny_kernel(I8Params p) {
  __shared__ i32x4 part[4][TT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int M = (int)p.M;
  const uint8_t* w = p.w + (int64_t)min(n0 + li, p.N - 1) * p.K + 16 * g;
  const uint8_t* x[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) x[t] = p.x + (int64_t)min(16 * t + li, M - 1) * p.K + 16 * g;
  i32x4 acc[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t] = i32x4{0, 0, 0, 0};
  constexpr int kDepth = TT <= 2 ? 8 : 4;  // steps whose loads go out together
  for (int k0 = 64 * wave; k0 < p.K; k0 += 256 * kDepth) {
    i32x4 a[kDepth], b[kDepth][TT];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int k = k0 + 256 * d;
      const bool in = k + 16 * g < p.K;  // K is a multiple of 16
      a[d] = i32x4{0, 0, 0, 0};
      if (in) a[d] = *reinterpret_cast<const i32x4*>(w + k);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        b[d][t] = i32x4{0, 0, 0, 0};
        if (in) b[d][t] = *reinterpret_cast<const i32x4*>(x[t] + k);
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
#pragma unroll
      for (int t = 0; t < TT; ++t)
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[d], b[d][t], acc[t], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // Wave t of the first TT adds tile t: token 16 t + li, channels 4 g .. 4 g + 3.
  for (int t = wave; t < TT; t += 4) {
    const i32x4 s = part[0][t][lane] + part[1][t][lane] + part[2][t][lane] + part[3][t][lane];
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

}  // namespace aa

using namespace aa;

extern "C" int aa_rowquant_int8(const void* x, int64_t rows, int64_t K, int gelu, void* q, float* s,
                                int dtype, void* stream) {
  clear_error();
  if (dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, "rowquant_int8: only bf16 input is implemented");
  if (rows < 0 || K <= 0) return fail(AA_EINVAL, "rowquant_int8: bad rows/K");
  if (K % 8 != 0 || K > kQ8MaxK)
    return fail(AA_EUNSUPPORTED, "rowquant_int8: K must be a multiple of 8 and at most 8192");
  if (rows > 0x7fffff00) return fail(AA_EUNSUPPORTED, "rowquant_int8: too many rows");
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
  if (K % 16 == 0 && aligned16(q)) {
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
  if (M <= 64) {
    const dim3 grid((unsigned)((N + 15) / 16));
    if (M <= 16) int8_skinny_kernel<1><<<grid, 256, 0, st>>>(p);
    else if (M <= 32) int8_skinny_kernel<2><<<grid, 256, 0, st>>>(p);
    else int8_skinny_kernel<4><<<grid, 256, 0, st>>>(p);
    return check_launch("int8_linear");
  }
  const int64_t cus = std::max(1, device_cu_count());
  const auto tiles = [&](int64_t mt, int64_t nt) { return (M + mt - 1) / mt * ((N + nt - 1) / nt); };
  // Whole rounds of workgroups over the CUs times a round's relative time.
  const double big = (double)((tiles(256, 256) + cus - 1) / cus) * 1.93;
  const double small = (double)((tiles(128, 128) + 2 * cus - 1) / (2 * cus)) * 1.24;
  const bool use_big = big <= small;
  const int64_t mt = use_big ? 256 : 128;
  const int64_t total = use_big ? tiles(256, 256) : tiles(128, 128);
  if (total > 0x7fffffff) return fail(AA_EUNSUPPORTED, "int8_linear: too many tokens");
  p.mtiles = (int)((M + mt - 1) / mt);
  if (use_big) int8_linear_kernel<I8TileA><<<dim3((unsigned)total), I8TileA::kThreads, 0, st>>>(p);
  else if (total <= cus) int8_linear_kernel<I8TileD><<<dim3((unsigned)total), I8TileD::kThreads, 0, st>>>(p);
  else int8_linear_kernel<I8TileC><<<dim3((unsigned)total), I8TileC::kThreads, 0, st>>>(p);
  return check_launch("int8_linear");
}
