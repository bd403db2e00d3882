// The norms around a block's sublayers, with its gate, residual scale and
// modulation: one pass forward, one backward.
//
//   n = y                                   (the sublayer's output), or
//   n = y * rsqrt(mean(y^2) + eps) * w      with a norm behind the sublayer
//   r = x + c g n                           gate g, residual scale c
//   h = (r - mean(r)) * rsqrt(var(r) + eps) * (1 + scale) + shift
//
// over rows of D channels; g, scale, shift are one row per batch item (or one
// for all). r and h are each rounded to bf16 once: the norm is taken of the
// fp32 r, not of the rounded one. With kInt8 h leaves as int8 codes with a
// scale per token (block_math.h), rounded from fp32 directly.
//
// Backward, with xh = (r - mean) rstd and u = dh (1 + scale):
//   d  = dr + rstd (u - mean(u) - xh mean(u xh))     = dx
//   dn = c g d;  dy = dn, or ry (dn w - yh mean(dn w yh)) with yh = y ry
//   dg = sum c n d, dscale = sum dh xh, dshift = sum dh, dw = sum dn yh
// r is formed again from x and y in fp32 (reading the bf16 r instead would
// cost the same bytes and put its rounding, 2^-9, into every gradient); mean,
// rstd and ry come from the forward (16 bytes a row).
//
// Bound: HBM. 8 bytes a value forward (x, y in, r, h out), 7 with int8, 12 backward.
// A row lies in the registers of one wave (D <= 2048; backward with a norm on y or
// with sums <= 1024) or of two, four or eight, so it is read once, the variance is
// taken about the mean without a second read, and no barrier stands between loads
// and stores of a wave's own row. Measured at D = 2048 (a copy: 5.1 TB/s): forward
// 8192 tokens 21 to 22 us (6.1 to 6.3 TB/s; with plain in place of nontemporal stores
// 22 to 25), 4096 tokens 12; int8 7904 tokens 23 to 25 (4.5 to 4.9); backward 4096
// tokens 18 (5.5 TB/s; the registers of the norm's form at two waves a SIMD: 26).
// Backward with all gradients, 3 x 1001 tokens of 1544 17.4 (3.2 TB/s, a round of one
// workgroup a CU, held modulation and the next row ahead; without these two 21), and
// 3.9 for the sums' second launch (7.2 with 4 waves a column block in place of 16).
#include <algorithm>

#include "aa_common.h"
#include "block_math.h"

namespace aa {

constexpr int kAdThreads = 256;
constexpr int kAdWaves = kAdThreads / 64;
constexpr int kAdMaxD = 8192;

struct AdFwd {
  const bf16* x;
  const bf16* y;  // null: no residual add, r = x is not written
  const void *gate, *scale, *shift;
  int64_t gs, ss, hs;  // elements between the batch items' rows, 0: one row for all
  const float* w;      // null: no norm behind the sublayer
  bf16* r;
  bf16* h;
  uint8_t* q;
  float* qs;
  float* stats;  // [rows][4]: mean, rstd, ry, 0; or null
  int rows, S, D;
  int rpw;  // rows per wave (per workgroup where four waves share a row)
  float eps, c;
};

// Eight values of a modulation row, bf16 or fp32.
template <bool kF32>
struct Mod8 {
  u32x4 v[kF32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    if constexpr (kF32) {
      v[0] = ld16((const float*)base + at);
      v[1] = ld16((const float*)base + at + 4);
    } else {
      v[0] = ld16((const bf16*)base + at);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (kF32) return __uint_as_float(v[i >> 2][i & 3]);
    else return (i & 1) ? bf16_hi(v[0][i >> 1]) : bf16_lo(v[0][i >> 1]);
  }
};

// Sums (or maxima) over the waves that share a row.
template <int WPR>
struct RowShare {
  float* buf;  // [2][8]: a place per wave
  int wave, turn;
  template <class Op>
  __device__ __forceinline__ uint32_t join(uint32_t x, Op op) {
    if constexpr (WPR == 1) return x;
    uint32_t* at = reinterpret_cast<uint32_t*>(buf) + turn * 8;
    turn ^= 1;
    // Two buffers in turn: a wave that has passed the barrier of one use can
    // be at most at the store of the next, in the other buffer.
    at[wave] = x;
    __syncthreads();
    x = at[wave & ~(WPR - 1)];
#pragma unroll
    for (int i = 1; i < WPR; ++i) x = op(x, at[(wave & ~(WPR - 1)) + i]);
    return x;
  }
  __device__ __forceinline__ float sum(float x) {
    return __uint_as_float(join(__float_as_uint(wave_sum(x)), [](uint32_t a, uint32_t b) {
      return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
  }
  __device__ __forceinline__ uint32_t umax(uint32_t x) {
    return join(wave_umax(x), [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  }
};

// WPR waves per row, NU units of 8 values per lane: unit lane + 64 (wsub + WPR p).
template <int NU, int WPR, bool kModF32, bool kInt8>
__global__ __launch_bounds__(kAdThreads) void adaln_fwd_kernel(AdFwd p) {
  __shared__ float shared[16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wsub = wave % WPR;
  constexpr int kRows = kAdWaves / WPR;
  RowShare<WPR> share{shared, wave, 0};
  const int nunit = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  int unit[NU];
  bool live[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    unit[i] = lane + 64 * (wsub + WPR * i);
    live[i] = unit[i] < nunit;
  }
  int row = blockIdx.x * (kRows * p.rpw) + wave / WPR;
  int b = row / p.S, at = row - b * p.S;  // batch item and place in it
  int have = -1;
  // bf16 modulation rows stay in registers from row to row; fp32 ones, twice as
  // many, are read again (from L1: the workgroup's waves share them).
  constexpr bool kHold = !kModF32;
  Mod8<kModF32> gate[NU], scale[NU], shift[NU];
  for (int it = 0; it < p.rpw && row < p.rows; ++it, row += kRows, at += kRows) {
    while (at >= p.S) {
      at -= p.S;
      ++b;
    }
    u32x4 xr[NU], yr[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      xr[i] = yr[i] = u32x4{0, 0, 0, 0};
      if (live[i]) {
        xr[i] = ld16(p.x + (int64_t)row * p.D + 8 * unit[i]);
        if (p.y) yr[i] = ld16(p.y + (int64_t)row * p.D + 8 * unit[i]);
      }
    }
    if (kHold && b != have) {
      have = b;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (!live[i]) continue;
        if (p.y) gate[i].load(p.gate, b * p.gs + 8 * unit[i]);
        scale[i].load(p.scale, b * p.ss + 8 * unit[i]);
        shift[i].load(p.shift, b * p.hs + 8 * unit[i]);
      }
    }
    float ry = 1.0f;
    if (p.w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        float y[8];
        unpack8(yr[i], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
      }
      ry = 1.0f / sqrtf(share.sum(ss) * inv_d + p.eps);
    }
    float r[NU][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      unpack8(xr[i], r[i]);
      if (p.y && live[i]) {
        float y[8];
        unpack8(yr[i], y);
        if (p.w) {
          const f32x4 w0 = ldf4(p.w + 8 * unit[i]), w1 = ldf4(p.w + 8 * unit[i] + 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= ry * (j < 4 ? w0[j & 3] : w1[j & 3]);
        }
        if constexpr (!kHold) gate[i].load(p.gate, b * p.gs + 8 * unit[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[i][j] = fmaf(p.c * gate[i].get(j), y[j], r[i][j]);
        st16_nt(p.r + (int64_t)row * p.D + 8 * unit[i], pack8(r[i]));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += r[i][j];
    }
    const float mean = share.sum(sum) * inv_d;
    float var = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (!live[i]) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[i][j] -= mean;
        var = fmaf(r[i][j], r[i][j], var);
      }
    }
    const float rstd = 1.0f / sqrtf(share.sum(var) * inv_d + p.eps);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (!live[i]) continue;
      if constexpr (!kHold) {
        scale[i].load(p.scale, b * p.ss + 8 * unit[i]);
        shift[i].load(p.shift, b * p.hs + 8 * unit[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) r[i][j] = fmaf(r[i][j] * rstd, 1.0f + scale[i].get(j), shift[i].get(j));
      if constexpr (kInt8) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) top = max3abs_nan(top, r[i][j], r[i][j + 1]);
      }
      if constexpr (!kInt8) st16_nt(p.h + (int64_t)row * p.D + 8 * unit[i], pack8(r[i]));
    }
    if constexpr (kInt8) {
      const RowScale rs = row_scale(share.umax(mag_bits(top)));
#pragma unroll
      for (int i = 0; i < NU; ++i)
        if (live[i])
          *reinterpret_cast<u32x2*>(p.q + (int64_t)row * p.D + 8 * unit[i]) = int8_codes8(r[i], rs);
      if (lane == 0 && wsub == 0) p.qs[row] = rs.s;
    }
    if (p.stats && lane == 0 && wsub == 0)
      *reinterpret_cast<f32x4*>(p.stats + 4 * (int64_t)row) = f32x4{mean, rstd, ry, 0.f};
  }
}

// ---------------------------------------------------------------- backward --

constexpr int kAdBThreads = 512;
constexpr int kAdBWaves = kAdBThreads / 64;

struct AdBwd {
  const bf16 *dr, *dh;  // either may be null: a gradient of zero
  const bf16 *x, *y;
  const void *gate, *scale;
  int64_t gs, ss;
  const float* w;
  const float* stats;
  bf16 *dx, *dy;
  float* part;  // [B * chunks][NC][D], NC column sums: dscale, dshift, dgate, dw
  int S, D;
  int chunks;  // per batch item
  int rpc;     // rows per chunk
  float c;
};

// One workgroup takes a chunk of a batch item's rows, its waves (groups of WPR)
// one row each in turn. NC > 0: sums over the chunk's rows stay in registers,
// are added over the waves in LDS in a fixed order and leave as one partial
// record, which colsum_kernel adds up.
template <int NU, int WPR, bool kModF32, int NC, bool kPost>
__global__ __launch_bounds__(kAdBThreads) void adaln_bwd_kernel(AdBwd p) {
  constexpr int kGroups = kAdBWaves / WPR;   // rows at a time
  constexpr int kWidth = NU * WPR * 64 * 8;  // columns a group holds (>= D)
  __shared__ __attribute__((aligned(16))) float sums[NC ? kGroups * kWidth : 4];
  __shared__ float shared[16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wsub = wave % WPR, group = wave / WPR;
  RowShare<WPR> share{shared, wave, 0};
  const int nunit = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  const int b = blockIdx.x / p.chunks, chunk = blockIdx.x - b * p.chunks;
  const int64_t row0 = (int64_t)b * p.S;
  const int first = chunk * p.rpc, last = min(p.S, first + p.rpc);
  float acc[NC ? NC : 1][NU][8];
#pragma unroll
  for (int v = 0; v < NC; ++v)
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[v][i][j] = 0.f;

  int unit[NU];
  bool live[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    unit[i] = lane + 64 * (wsub + WPR * i);
    live[i] = unit[i] < nunit;
  }
  struct Row {
    f32x4 st;
    u32x4 x[NU], y[NU], dh[NU], dr[NU];
  };
  auto load = [&](Row& t, int s) {
    const int64_t row = row0 + min(s, last - 1);
    t.st = ldf4(p.stats + 4 * row);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int64_t at = row * p.D + 8 * unit[i];
      t.x[i] = t.y[i] = t.dh[i] = t.dr[i] = u32x4{0, 0, 0, 0};
      if (live[i]) {
        t.x[i] = ld16(p.x + at);
        if (p.y) t.y[i] = ld16(p.y + at);
        if (p.dh) t.dh[i] = ld16(p.dh + at);
        if (p.dr) t.dr[i] = ld16(p.dr + at);
      }
    }
  };
  // c gate, 1 + scale and w of a lane's columns, from registers for all rows where
  // a workgroup is alone on its CU (sums), else as they are needed.
  constexpr bool kHold = NC > 0;
  float hg[kHold ? NU : 1][8], hs[kHold ? NU : 1][8], hw[kHold && kPost ? NU : 1][8];
  auto get_gate = [&](float (&v)[8], int i) {
    Mod8<kModF32> m;
    m.load(p.gate, b * p.gs + 8 * unit[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p.c * m.get(j);
  };
  auto get_scale = [&](float (&v)[8], int i) {
    Mod8<kModF32> m;
    m.load(p.scale, b * p.ss + 8 * unit[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 1.0f + m.get(j);
  };
  auto get_w = [&](float (&v)[8], int i) {
    const f32x4 w0 = ldf4(p.w + 8 * unit[i]), w1 = ldf4(p.w + 8 * unit[i] + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < 4 ? w0[j & 3] : w1[j & 3];
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (live[i]) {
        get_scale(hs[i], i);
        if (p.y) get_gate(hg[i], i);
        if constexpr (kPost) get_w(hw[i], i);
      }
  }
  // Every wave of a row's group makes the same turns, and all groups as many
  // (the barriers of a shared row's sums): a group past its rows computes on
  // the last row and writes nothing.
  const int turns = (last - first + kGroups - 1) / kGroups;
  Row next;
  if constexpr (kHold) load(next, first + group);
  for (int it = 0; it < turns; ++it) {
    const int s = first + it * kGroups + group;
    const bool mine = s < last;
    if (WPR == 1 && !mine) break;
    const int64_t row = row0 + min(s, last - 1);
    Row cur;
    if constexpr (kHold) {
      cur = next;
      if (it + 1 < turns) load(next, s + kGroups);
    } else {
      load(cur, s);
    }
    const auto &rx = cur.x, &rdy = cur.y, &rdh = cur.dh, &rdr = cur.dr;
    const float mean = cur.st[0], rstd = cur.st[1], ry = cur.st[2];
    // xh in place of r, and the two means.
    float xh[NU][8];
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      unpack8(rx[i], xh[i]);
      if (!live[i]) continue;
      float v[8];
      if (p.y) {
        float y[8];
        unpack8(rdy[i], y);
        if constexpr (kPost) {
          if constexpr (!kHold) get_w(v, i);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= ry * (kHold ? hw[kHold ? i : 0][j] : v[j]);
        }
        if constexpr (!kHold) get_gate(v, i);
#pragma unroll
        for (int j = 0; j < 8; ++j) xh[i][j] = fmaf(kHold ? hg[kHold ? i : 0][j] : v[j], y[j], xh[i][j]);
      }
      if constexpr (!kHold) get_scale(v, i);
      float dh[8];
      unpack8(rdh[i], dh);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] = (xh[i][j] - mean) * rstd;
        const float u = dh[j] * (kHold ? hs[kHold ? i : 0][j] : v[j]);
        m1 += u;
        m2 = fmaf(u, xh[i][j], m2);
      }
    }
    m1 = share.sum(m1) * inv_d;
    m2 = share.sum(m2) * inv_d;
    // With a norm on y, dy waits for a third mean: dn w stays until then.
    float m3 = 0.f;
    float dnw[kPost ? NU : 1][8];
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (!live[i]) continue;
      float v[8];
      if constexpr (!kHold) get_scale(v, i);
      float dh[8], d[8];
      unpack8(rdh[i], dh);
      unpack8(rdr[i], d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = dh[j] * (kHold ? hs[kHold ? i : 0][j] : v[j]);
        d[j] = fmaf(rstd, u - m1 - xh[i][j] * m2, d[j]);
        if constexpr (NC > 0) {
          if (mine) {
            acc[0][i][j] = fmaf(dh[j], xh[i][j], acc[0][i][j]);
            acc[1][i][j] += dh[j];
          }
        }
      }
      if (mine) st16_nt(p.dx + row * p.D + 8 * unit[i], pack8(d));
      if (!p.y) continue;
      if constexpr (!kHold) get_gate(v, i);
      float y[8];
      unpack8(rdy[i], y);
      if constexpr (kPost) {
        float w[8];
        if constexpr (!kHold) get_w(w, i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float wj = kHold ? hw[kHold ? i : 0][j] : w[j];
          const float yh = y[j] * ry;
          const float dn = (kHold ? hg[kHold ? i : 0][j] : v[j]) * d[j];
          if constexpr (NC > 3) {
            if (mine) {
              acc[2][i][j] = fmaf(p.c * yh * wj, d[j], acc[2][i][j]);
              acc[3][i][j] = fmaf(dn, yh, acc[3][i][j]);
            }
          }
          dnw[i][j] = dn * wj;
          m3 = fmaf(dnw[i][j], yh, m3);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (NC > 2) {
            if (mine) acc[2][i][j] = fmaf(p.c * y[j], d[j], acc[2][i][j]);
          }
          d[j] *= kHold ? hg[kHold ? i : 0][j] : v[j];
        }
        if (mine) st16_nt(p.dy + row * p.D + 8 * unit[i], pack8(d));
      }
    }
    if constexpr (kPost) {
      m3 = share.sum(m3) * inv_d;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (!live[i]) continue;
        float y[8];
        unpack8(rdy[i], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = ry * (dnw[i][j] - y[j] * ry * m3);
        if (mine) st16_nt(p.dy + row * p.D + 8 * unit[i], pack8(y));
      }
    }
  }
  if constexpr (NC > 0) {
#pragma unroll
    for (int v = 0; v < NC; ++v) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        float* at = sums + group * kWidth + 8 * (lane + 64 * (wsub + WPR * i));
        *reinterpret_cast<f32x4*>(at) = f32x4{acc[v][i][0], acc[v][i][1], acc[v][i][2], acc[v][i][3]};
        *reinterpret_cast<f32x4*>(at + 4) = f32x4{acc[v][i][4], acc[v][i][5], acc[v][i][6], acc[v][i][7]};
      }
      __syncthreads();
      float* out = p.part + ((int64_t)blockIdx.x * NC + v) * p.D;
      for (int col = threadIdx.x; col < p.D; col += kAdBThreads) {
        float s = sums[col];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) s += sums[g * kWidth + col];
        out[col] = s;
      }
    }
  }
}

// Adds the partial records up, in a fixed order: out[b][col] over the chunks of
// batch item b, or out[0][col] over all of them.
struct ColSum {
  const float* part;
  int nc, D, chunks, B;
  struct Out {
    void* out;
    int vec;   // which of the record's sums
    int rows;  // B or 1
    int f32;   // fp32 or bf16
  } out[4];
};

constexpr int kCsParts = 16;  // waves of a workgroup, each with every 16th record

__global__ __launch_bounds__(64 * kCsParts) void colsum_kernel(ColSum p) {
  const ColSum::Out o = p.out[blockIdx.y];
  const int b = blockIdx.z;
  if (b >= o.rows) return;  // whole workgroups
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
  __shared__ float join[kCsParts][64];
  const int c0 = o.rows == 1 ? 0 : b * p.chunks;
  const int n = o.rows == 1 ? p.B * p.chunks : p.chunks;
  float s = 0.f;
  if (col < p.D) {
    const float* at = p.part + ((int64_t)c0 * p.nc + o.vec) * p.D + col;
    const int64_t step = (int64_t)p.nc * p.D;
    // Four running sums: a chain of one would wait for each load's add.
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    int c = part;
    for (; c + 3 * kCsParts < n; c += 4 * kCsParts)
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] += at[(c + kCsParts * i) * step];
    for (; c < n; c += kCsParts) t[0] += at[c * step];
    s = (t[0] + t[1]) + (t[2] + t[3]);
  }
  join[part][threadIdx.x & 63] = s;
  __syncthreads();
  if (part == 0 && col < p.D) {
    const int l = threadIdx.x;
    s = join[0][l];
#pragma unroll
    for (int i = 1; i < kCsParts; ++i) s += join[i][l];
    const int64_t at = (int64_t)b * p.D + col;
    if (o.f32) ((float*)o.out)[at] = s;
    else ((bf16*)o.out)[at] = (bf16)s;
  }
}

// -------------------------------------------------------------------- host --

template <int NU, int WPR>
static void launch_fwd(dim3 grid, hipStream_t st, const AdFwd& p, bool f32, bool int8) {
  if (f32 && int8) adaln_fwd_kernel<NU, WPR, true, true><<<grid, kAdThreads, 0, st>>>(p);
  else if (f32) adaln_fwd_kernel<NU, WPR, true, false><<<grid, kAdThreads, 0, st>>>(p);
  else if (int8) adaln_fwd_kernel<NU, WPR, false, true><<<grid, kAdThreads, 0, st>>>(p);
  else adaln_fwd_kernel<NU, WPR, false, false><<<grid, kAdThreads, 0, st>>>(p);
}

template <int NU, int WPR, int NC, bool kPost>
static void launch_bwd_nc(dim3 grid, hipStream_t st, const AdBwd& p, bool f32) {
  if (f32) adaln_bwd_kernel<NU, WPR, true, NC, kPost><<<grid, kAdBThreads, 0, st>>>(p);
  else adaln_bwd_kernel<NU, WPR, false, NC, kPost><<<grid, kAdBThreads, 0, st>>>(p);
}
template <int NU, int WPR, bool kPlain = true>
static void launch_bwd(dim3 grid, hipStream_t st, const AdBwd& p, bool sums, bool f32) {
  if (sums && p.w) launch_bwd_nc<NU, WPR, 4, true>(grid, st, p, f32);
  else if (sums) launch_bwd_nc<NU, WPR, 3, false>(grid, st, p, f32);
  else if (p.w) launch_bwd_nc<NU, WPR, 0, true>(grid, st, p, f32);
  else if constexpr (kPlain) launch_bwd_nc<NU, WPR, 0, false>(grid, st, p, f32);
}

// Chunks of rows per batch item in the backward: with column sums one
// workgroup per CU (its partial record, NC D floats, is as much as 2 NC rows of
// an input, so no more of them than fill the device), else four rows a wave.
// wave_rows: a wave takes whole rows up to D = 2048 (32 columns a lane, else 16),
// where neither sums nor a norm on y want the registers.
static int bwd_waves_per_row(int64_t D, bool wave_rows) {
  return D <= 1024 || (D <= 2048 && wave_rows) ? 1 : D <= 2048 ? 2 : D <= 4096 ? 4 : 8;
}
static int bwd_rows_per_chunk(int64_t B, int64_t S, int64_t D, bool sums, bool wave_rows) {
  const int64_t groups = kAdBWaves / bwd_waves_per_row(D, wave_rows);
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t per = sums ? (B * S + cus - 1) / cus : std::min<int64_t>(4 * groups, (B * S + 2 * cus - 1) / (2 * cus));
  return (int)std::min<int64_t>(S, std::max<int64_t>(1, (per + groups - 1) / groups) * groups);
}

static int check_sizes(const char* what, int64_t B, int64_t S, int64_t D, int dtype, int mod_dtype) {
  const std::string w = what;
  if (dtype != AA_DTYPE_BF16) return fail(AA_EUNSUPPORTED, w + ": only bf16 activations are implemented");
  if (mod_dtype != AA_DTYPE_BF16 && mod_dtype != AA_DTYPE_FP32)
    return fail(AA_EUNSUPPORTED, w + ": the modulation must be bf16 or fp32");
  if (B < 0 || S < 0 || D <= 0) return fail(AA_EINVAL, w + ": bad B/S/D");
  if (D % 8 != 0 || D > kAdMaxD)
    return fail(AA_EUNSUPPORTED, w + ": D must be a multiple of 8 and at most 8192");
  if (B > 0 && S > 0x7fffff00 / B) return fail(AA_EUNSUPPORTED, w + ": too many tokens");
  return AA_OK;
}

// One modulation row per batch item or for all: 16-byte aligned rows.
static int check_mod(const char* what, const void* t, int64_t stride, int64_t D, int mod_dtype) {
  const std::string w = what;
  if (!t) return fail(AA_EINVAL, w + ": null pointer");
  const int64_t unit = mod_dtype == AA_DTYPE_FP32 ? 4 : 8;
  if (!aligned16(t) || stride % unit != 0)
    return fail(AA_EINVAL, w + ": modulation rows must be 16-byte aligned");
  if (stride < 0 || (stride != 0 && stride < D))
    return fail(AA_EINVAL, w + ": a modulation's batch stride must be 0 or at least D");
  return AA_OK;
}

}  // namespace aa

using namespace aa;

extern "C" int aa_adaln_fwd(const aa_adaln_args* a, void* stream) {
  clear_error();
  const char* what = "adaln";
  if (!a) return fail(AA_EINVAL, "adaln: null args");
  if (int rc = check_sizes(what, a->B, a->S, a->D, a->dtype, a->mod_dtype)) return rc;
  if (a->B * a->S == 0) return AA_OK;
  if (!a->x || (!a->q && !a->h) || (a->q && !a->q_scale) || (a->y && !a->r))
    return fail(AA_EINVAL, "adaln: null pointer");
  if (a->q && a->h) return fail(AA_EINVAL, "adaln: h and q exclude each other");
  if (a->weight && !a->y) return fail(AA_EINVAL, "adaln: weight without y");
  if (a->y)
    if (int rc = check_mod(what, a->gate, a->gate_stride, a->D, a->mod_dtype)) return rc;
  if (int rc = check_mod(what, a->scale, a->scale_stride, a->D, a->mod_dtype)) return rc;
  if (int rc = check_mod(what, a->shift, a->shift_stride, a->D, a->mod_dtype)) return rc;
  for (const void* t : {a->x, a->y, (const void*)a->weight, (const void*)a->r, (const void*)a->h,
                        (const void*)a->stats})
    if (!aligned16(t)) return fail(AA_EINVAL, "adaln: pointers must be 16-byte aligned");
  if (((uintptr_t)a->q & 7u) != 0) return fail(AA_EINVAL, "adaln: q must be 8-byte aligned");
  AdFwd p;
  p.x = (const bf16*)a->x;
  p.y = (const bf16*)a->y;
  p.gate = a->gate;
  p.scale = a->scale;
  p.shift = a->shift;
  p.gs = a->gate_stride;
  p.ss = a->scale_stride;
  p.hs = a->shift_stride;
  p.w = a->weight;
  p.r = (bf16*)a->r;
  p.h = (bf16*)a->h;
  p.q = (uint8_t*)a->q;
  p.qs = a->q_scale;
  p.stats = a->stats;
  p.rows = (int)(a->B * a->S);
  p.S = (int)a->S;
  p.D = (int)a->D;
  p.eps = a->eps;
  p.c = a->branch_scale;
  const int rows_at_once = p.D <= 2048 ? kAdWaves : 1;
  const int64_t cus = std::max(1, device_cu_count());
  p.rpw = (int)std::clamp<int64_t>(p.rows / (cus * 4 * rows_at_once), 1, 4);
  const int64_t per = (int64_t)rows_at_once * p.rpw;
  const int64_t blocks = (p.rows + per - 1) / per;
  if (!grid_fits(blocks, kAdThreads)) return fail(AA_EUNSUPPORTED, "adaln: too many tokens");
  const dim3 grid((unsigned)blocks);
  hipStream_t st = (hipStream_t)stream;
  const bool f32 = a->mod_dtype == AA_DTYPE_FP32, int8 = a->q != nullptr;
  if (p.D <= 512) launch_fwd<1, 1>(grid, st, p, f32, int8);
  else if (p.D <= 1024) launch_fwd<2, 1>(grid, st, p, f32, int8);
  else if (p.D <= 2048) launch_fwd<4, 1>(grid, st, p, f32, int8);
  else if (p.D <= 4096) launch_fwd<2, 4>(grid, st, p, f32, int8);
  else launch_fwd<4, 4>(grid, st, p, f32, int8);
  return check_launch(what);
}

extern "C" size_t aa_adaln_bwd_workspace(int64_t B, int64_t S, int64_t D, int sums) {
  if (B <= 0 || S <= 0 || D <= 0 || !sums) return 0;
  const int64_t rpc = bwd_rows_per_chunk(B, S, D, true, false);
  return (size_t)(B * ((S + rpc - 1) / rpc) * 4 * D) * sizeof(float);
}

extern "C" int aa_adaln_bwd(const aa_adaln_bwd_args* a, void* workspace, size_t workspace_bytes,
                            void* stream) {
  clear_error();
  const char* what = "adaln_bwd";
  if (!a) return fail(AA_EINVAL, "adaln_bwd: null args");
  if (int rc = check_sizes(what, a->B, a->S, a->D, a->dtype, a->mod_dtype)) return rc;
  const bool sums = a->dgate || a->dscale || a->dshift || a->dweight;
  if (a->B * a->S == 0) {
    if (sums) return fail(AA_EINVAL, "adaln_bwd: no tokens to sum over");
    return AA_OK;
  }
  if (!a->x || !a->stats || !a->dx || (a->y && !a->dy)) return fail(AA_EINVAL, "adaln_bwd: null pointer");
  if (a->weight && !a->y) return fail(AA_EINVAL, "adaln_bwd: weight without y");
  if ((a->dgate && !a->y) || (a->dweight && !a->weight))
    return fail(AA_EINVAL, "adaln_bwd: a gradient of an input that is not there");
  if (a->y)
    if (int rc = check_mod(what, a->gate, a->gate_stride, a->D, a->mod_dtype)) return rc;
  if (int rc = check_mod(what, a->scale, a->scale_stride, a->D, a->mod_dtype)) return rc;
  for (const void* t : {a->x, a->y, a->dr, a->dh, (const void*)a->dx, (const void*)a->dy,
                        (const void*)a->weight, (const void*)a->stats, (const void*)workspace})
    if (!aligned16(t)) return fail(AA_EINVAL, "adaln_bwd: pointers must be 16-byte aligned");
  for (const int64_t n : {a->gate_rows, a->scale_rows, a->shift_rows})
    if (sums && n != 1 && n != a->B) return fail(AA_EINVAL, "adaln_bwd: modulation rows must be 1 or B");
  if (sums && a->B > 65535) return fail(AA_EUNSUPPORTED, "adaln_bwd: too many batch items (65535)");
  const size_t need = aa_adaln_bwd_workspace(a->B, a->S, a->D, sums);
  if (need && (!workspace || workspace_bytes < need))
    return fail(AA_EINVAL, "adaln_bwd: workspace too small");
  AdBwd p;
  p.dr = (const bf16*)a->dr;
  p.dh = (const bf16*)a->dh;
  p.x = (const bf16*)a->x;
  p.y = (const bf16*)a->y;
  p.gate = a->gate;
  p.scale = a->scale;
  p.gs = a->gate_stride;
  p.ss = a->scale_stride;
  p.w = a->weight;
  p.stats = a->stats;
  p.dx = (bf16*)a->dx;
  p.dy = (bf16*)a->dy;
  p.part = (float*)workspace;
  p.S = (int)a->S;
  p.D = (int)a->D;
  const bool wave_rows = !sums && !a->weight;
  p.rpc = bwd_rows_per_chunk(a->B, a->S, a->D, sums, wave_rows);
  p.chunks = (p.S + p.rpc - 1) / p.rpc;
  p.c = a->branch_scale;
  const int nc = !sums ? 0 : a->weight ? 4 : 3;
  if (!grid_fits(a->B * p.chunks, kAdBThreads)) return fail(AA_EUNSUPPORTED, "adaln_bwd: too many tokens");
  const dim3 grid((unsigned)(a->B * p.chunks));
  hipStream_t st = (hipStream_t)stream;
  const bool f32 = a->mod_dtype == AA_DTYPE_FP32;
  if (p.D <= 512) launch_bwd<1, 1>(grid, st, p, sums, f32);
  else if (p.D <= 1024) launch_bwd<2, 1>(grid, st, p, sums, f32);
  else if (p.D <= 2048 && wave_rows) launch_bwd_nc<4, 1, 0, false>(grid, st, p, f32);
  else if (p.D <= 2048) launch_bwd<2, 2, false>(grid, st, p, sums, f32);
  else if (p.D <= 4096) launch_bwd<2, 4>(grid, st, p, sums, f32);
  else launch_bwd<2, 8>(grid, st, p, sums, f32);
  if (int rc = check_launch(what)) return rc;
  if (!sums) return AA_OK;
  ColSum c;
  c.part = p.part;
  c.nc = nc;
  c.D = p.D;
  c.chunks = p.chunks;
  c.B = (int)a->B;
  int n = 0, zmax = 1;
  const auto add = [&](void* out, int vec, int64_t rows, bool is_f32) {
    if (!out) return;
    c.out[n++] = {out, vec, (int)rows, is_f32 ? 1 : 0};
    zmax = std::max(zmax, (int)rows);
  };
  add(a->dscale, 0, a->scale_rows, f32);
  add(a->dshift, 1, a->shift_rows, f32);
  add(a->dgate, 2, a->gate_rows, f32);
  add(a->dweight, 3, 1, true);
  colsum_kernel<<<dim3((p.D + 63) / 64, n, zmax), 64 * kCsParts, 0, st>>>(c);
  return check_launch(what);
}
