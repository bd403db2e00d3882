// Rotary positions on their own: tables of cos and sin, and the turn of queries
// and keys by them, for gfx950. Both are bound by HBM.
//
// Tables: angle = position * frequency. A position of 10^6 leaves no digit of
//   its angle in fp32, so the frequency is kept in quarter turns (radians /
//   (pi / 2)) in fp64, the product's whole quarters are dropped in fp64 and only
//   the rest r in [-1/2, 1/2] goes to fp32, for sin and cos of (pi / 2) r.
//
// Turn: a pair (a, b) becomes (a cos - b sin, b cos + a sin), in fp32, rounded
//   once to the type of q and k. A pair is (i, i + part / 2) of a head or
//   (2 i, 2 i + 1); values from `part` on are copied. A lane owns one unit of
//   a head, 16 bytes at most on either side of its pairs, holds that unit's
//   cos and sin in registers and goes through several heads of its token with
//   them, so the tables are read once for those heads and each lane has that
//   many loads in flight. 2 x 9216 tokens of 16 + 16 heads of 128: 58 us, 5.2 TB/s
//   (fp16 and fp32 2 x 4096: 25 and 44 us, 5.4 and 6.1).
#include <algorithm>
#include <cmath>
#include <string>

#include "aa_common.h"

namespace aa {
namespace rotary {

// ---------------------------------------------------------------- tables --

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 256;
constexpr int kThreads = 256;

struct TableParams {
  const void* positions;  // [rows, axes]
  float* cos;             // [rows, pairs]
  float* sin;
  uint32_t total;         // threads: step * pairs / VEC
  uint32_t rows, step;    // a thread's rows: row, row + step, ...
  int axes, pairs;
  float amplitude;
  double quarters[kMaxPairs]; // a position's quarter turns of pair i
  uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ double position(const void* p, uint64_t i, int type) {
  switch (type) {
    case AA_POSITION_INT32: return (double)((const int32_t*)p)[i];
    case AA_POSITION_INT64: return (double)((const int64_t*)p)[i];
    case AA_POSITION_FP32: return (double)((const float*)p)[i];
    default: return ((const double*)p)[i];
  }
}

// sin and cos of q quarter turns. Polynomials of r^2 for |r| <= 1/2, fitted to
// the least largest error and rounded to fp32 (in exact arithmetic then 3.4e-8 of
// the sine, 2.2e-8 at most, and 0.6e-8 off the cosine; with their fp32 sums and
// r's own rounding 1.0e-7 and 0.7e-7, a step of 1 being 1.2e-7),
// in place of a library sine for any argument (11 fp32 instructions; with
// one the kernel was bound by its instructions, 131072 positions x 64 pairs 23 us).
__device__ __forceinline__ void sincos_quarters(double q, float& s, float& c) {
  const double whole = rint(q);
  const float r = (float)(q - whole);
  const float y = r * r;
  const float sn = r * fmaf(y, fmaf(y, fmaf(y, -0.004601658f, 0.07968003f), -0.6459635f), 1.5707964f);
  const float cs = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 0.000903363f, -0.020859936f), 0.25366917f), -1.2337005f), 1.0f);
  // The quarter modulo 4: its two low bits, of a double of up to 2^53.
  const int n = (int)(whole - 4.0 * floor(0.25 * whole));
  s = n & 1 ? cs : sn;
  c = n & 1 ? sn : cs;
  s = n & 2 ? -s : s;
  c = (n + 1) & 2 ? -c : c;
}

// VEC pairs of ROWS rows a thread, whose frequencies stay in registers; the rows
// of a workgroup's threads on one unit are `step` apart.
template <int VEC, int ROWS>
__global__ __launch_bounds__(kThreads) void tables_kernel(const TableParams p, int type) {
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  if (idx >= p.total) return;
  const uint32_t units = (uint32_t)p.pairs / VEC;
  const uint32_t row0 = idx / units;
  const int i0 = (int)(idx - row0 * units) * VEC;
  double quarters[VEC];
  int axis[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    quarters[j] = p.quarters[i0 + j];
    axis[j] = p.axis[i0 + j];
  }
  double pos[ROWS][VEC];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const uint64_t row = row0 + (uint64_t)r * p.step;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      pos[r][j] = row < p.rows ? position(p.positions, row * p.axes + axis[j], type) : 0;
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const uint64_t row = row0 + (uint64_t)r * p.step;
    if (row >= p.rows) return;
    float c[VEC], s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sincos_quarters(pos[r][j] * quarters[j], s[j], c[j]);
      c[j] *= p.amplitude;
      s[j] *= p.amplitude;
    }
    const uint64_t at = row * p.pairs + i0;
    if constexpr (VEC == 4) {
      __builtin_nontemporal_store(f32x4{c[0], c[1], c[2], c[3]}, reinterpret_cast<f32x4*>(p.cos + at));
      __builtin_nontemporal_store(f32x4{s[0], s[1], s[2], s[3]}, reinterpret_cast<f32x4*>(p.sin + at));
    } else {
      p.cos[at] = c[0];
      p.sin[at] = s[0];
    }
  }
}

// ------------------------------------------------------------------ turn --

struct TurnParams {
  const void* q;
  const void* k;
  void* qo;
  void* ko;
  const float* cos;
  const float* sin;
  int64_t qs[3], ks[3], qos[3], kos[3];  // batch, token, head strides
  int64_t table_stride;                  // between the batch items' tables
  uint32_t total;                        // threads: B * S * slices * units
  uint32_t S;
  int H, heads;                          // heads of q; of q and k
  int slices;                            // a thread's heads: slice, slice + slices, ...
  int part, units, turned;               // units of a head, the first `turned` of them pairs
  float sign;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// PER heads a thread; W: values of one side of a unit's pairs, and of a unit
// that is copied (INTERLEAVED: a unit is 2 W neighbouring values).
template <typename T, int W, bool INTERLEAVED, int PER>
__global__ __launch_bounds__(kThreads) void turn_kernel(const TurnParams p) {
  constexpr int C = INTERLEAVED ? 2 * W : W;  // values per access
  using V = Pack<T, C>;
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  if (idx >= p.total) return;
  const uint32_t g = idx / (uint32_t)p.units;
  const int u = (int)(idx - g * (uint32_t)p.units);
  const uint32_t token = g / (uint32_t)p.slices;
  const int slice = (int)(g - token * (uint32_t)p.slices);
  const uint32_t b = token / p.S;
  const uint32_t s = token - b * p.S;

  const bool turned = u < p.turned;
  // First value of the unit and, in the half layout, of its partner.
  const int lo = turned ? u * C : p.part + (u - p.turned) * C;
  const int hi = lo + (p.part >> 1);
  float c[W], sn[W];
  if (turned) {
    const int64_t at = (int64_t)b * p.table_stride + (int64_t)s * (p.part >> 1) + u * W;
    const Pack<float, W < 4 ? W : 4>* cp = reinterpret_cast<const Pack<float, W < 4 ? W : 4>*>(p.cos + at);
    const Pack<float, W < 4 ? W : 4>* sp = reinterpret_cast<const Pack<float, W < 4 ? W : 4>*>(p.sin + at);
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const auto cv = cp[j / 4], sv = sp[j / 4];
#pragma unroll
      for (int e = 0; e < (W < 4 ? W : 4); ++e) {
        c[j + e] = cv.v[e];
        sn[j + e] = sv.v[e] * p.sign;
      }
    }
  }
  V x[PER], y[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int h = slice + i * p.slices;
    if (h < p.heads) {
      const bool key = h >= p.H;
      const T* base = key ? (const T*)p.k + (int64_t)b * p.ks[0] + (int64_t)s * p.ks[1] + (h - p.H) * p.ks[2]
                          : (const T*)p.q + (int64_t)b * p.qs[0] + (int64_t)s * p.qs[1] + h * p.qs[2];
      x[i] = *reinterpret_cast<const V*>(base + lo);
      if (!INTERLEAVED && turned) y[i] = *reinterpret_cast<const V*>(base + hi);
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int h = slice + i * p.slices;
    if (h < p.heads) {
      const bool key = h >= p.H;
      T* base = key ? (T*)p.ko + (int64_t)b * p.kos[0] + (int64_t)s * p.kos[1] + (h - p.H) * p.kos[2]
                    : (T*)p.qo + (int64_t)b * p.qos[0] + (int64_t)s * p.qos[1] + h * p.qos[2];
      if (turned) {
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float a = (float)x[i].v[2 * j], d = (float)x[i].v[2 * j + 1];
            x[i].v[2 * j] = (T)(a * c[j] - d * sn[j]);
            x[i].v[2 * j + 1] = (T)(d * c[j] + a * sn[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const float a = (float)x[i].v[j], d = (float)y[i].v[j];
            x[i].v[j] = (T)(a * c[j] - d * sn[j]);
            y[i].v[j] = (T)(d * c[j] + a * sn[j]);
          }
          *reinterpret_cast<V*>(base + hi) = y[i];
        }
      }
      *reinterpret_cast<V*>(base + lo) = x[i];
    }
  }
}

template <typename T, int W, bool INTERLEAVED>
void launch_turn(TurnParams p, int64_t tokens, hipStream_t stream) {
  const auto run = [&](auto per) {
    constexpr int PER = decltype(per)::value;
    p.slices = (p.heads + PER - 1) / PER;
    p.total = (uint32_t)(tokens * p.slices * p.units);
    turn_kernel<T, W, INTERLEAVED, PER><<<(p.total + kThreads - 1) / kThreads, kThreads, 0, stream>>>(p);
  };
  // One head a thread while that fills no more than half of the chip (256
  // tokens, 32 heads of 128: 5.2 -> 3.7 us; 3003 tokens of 16 x 80: 6.0 -> 7.9).
  if (tokens * p.heads * p.units <= 1024 * (int64_t)device_cu_count()) run(std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, 4>{});
}

template <typename T>
void launch_turn(const TurnParams& p, int64_t tokens, int W, bool interleaved, hipStream_t stream) {
  if (interleaved) {
    switch (W) {
      case 4: if constexpr (sizeof(T) == 2) return launch_turn<T, 4, true>(p, tokens, stream);
      case 2: return launch_turn<T, 2, true>(p, tokens, stream);
      default: return launch_turn<T, 1, true>(p, tokens, stream);
    }
  }
  switch (W) {
    case 8: if constexpr (sizeof(T) == 2) return launch_turn<T, 8, false>(p, tokens, stream);
    case 4: return launch_turn<T, 4, false>(p, tokens, stream);
    case 2: return launch_turn<T, 2, false>(p, tokens, stream);
    default: return launch_turn<T, 1, false>(p, tokens, stream);
  }
}

}  // namespace rotary
}  // namespace aa

using namespace aa;

extern "C" int aa_rotary_tables(const aa_rotary_tables_args* a, void* stream) {
  using namespace rotary;
  clear_error();
  if (!a) return fail(AA_EINVAL, "rotary_tables: null args");
  if (a->axes < 1 || a->axes > kMaxAxes) return fail(AA_EUNSUPPORTED, "rotary_tables: 1 to 4 axes");
  if (a->position_type < AA_POSITION_INT32 || a->position_type > AA_POSITION_FP64)
    return fail(AA_EUNSUPPORTED, "rotary_tables: positions must be int32, int64, float32 or float64");
  if (a->scaling < AA_SCALING_NTK || a->scaling > AA_SCALING_YARN)
    return fail(AA_EINVAL, "rotary_tables: unknown scaling");
  if (a->scaling == AA_SCALING_YARN && !(a->original > 0 && std::isfinite(a->original)))
    return fail(AA_EINVAL, "rotary_tables: yarn needs the trained length (original > 0)");
  if (a->rows < 0) return fail(AA_EINVAL, "rotary_tables: bad rows");
  TableParams p = {};
  double most = 1.0;
  for (int64_t x = 0; x < a->axes; ++x) {
    const int64_t d = a->dims[x];
    const double scale = a->scale[x], base = a->theta[x];
    if (d < 0 || d % 2 || p.pairs + d / 2 > kMaxPairs)
      return fail(AA_EUNSUPPORTED, "rotary_tables: dims must be even, 2 to 512 together");
    if (!(scale >= 1 && std::isfinite(scale)) || !(base > 0 && std::isfinite(base)))
      return fail(AA_EINVAL, "rotary_tables: scale must be at least 1 and theta positive");
    most = std::max(most, scale);
    // The base grows with the length so that the slowest pair is stretched by
    // the scale and the fastest not at all (d = 2 has only the fastest).
    const double theta = a->scaling == AA_SCALING_NTK && d > 2 ? base * std::pow(scale, (double)d / (double)(d - 2)) : base;
    for (int64_t i = 0; i < d / 2; ++i) {
      double f = std::pow(theta, -2.0 * (double)i / (double)d);
      if (a->scaling == AA_SCALING_LINEAR) f /= scale;
      if (a->scaling == AA_SCALING_YARN) {
        // Pairs that turn 32 times or more in the trained length stay, those
        // with one turn or less are stretched, a ramp between (arXiv
        // 2309.00071, section 3.2, with alpha 1 and beta 32).
        const double turns = a->original * f / (2 * M_PI);
        const double keep = std::min(1.0, std::max(0.0, (turns - 1) / 31));
        f *= keep + (1 - keep) / scale;
      }
      p.quarters[p.pairs] = f / M_PI_2;
      p.axis[p.pairs++] = (uint8_t)x;
    }
  }
  if (p.pairs == 0) return fail(AA_EUNSUPPORTED, "rotary_tables: dims must be even, 2 to 512 together");
  p.amplitude = a->scaling == AA_SCALING_YARN ? (float)(0.1 * std::log(most) + 1) : 1.0f;
  if (a->rows == 0) return AA_OK;
  if (!a->positions || !a->cos || !a->sin) return fail(AA_EINVAL, "rotary_tables: null pointer");
  if (!aligned16(a->cos) || !aligned16(a->sin)) return fail(AA_EINVAL, "rotary_tables: outputs must be 16-byte aligned");
  const uintptr_t unit = a->position_type == AA_POSITION_INT32 || a->position_type == AA_POSITION_FP32 ? 4 : 8;
  if ((uintptr_t)a->positions % unit) return fail(AA_EINVAL, "rotary_tables: misaligned positions");
  const int vec = p.pairs % 4 ? 1 : 4;
  if (a->rows > 0xffffffff / p.pairs) return fail(AA_EUNSUPPORTED, "rotary_tables: too many positions");
  p.positions = a->positions;
  p.cos = a->cos;
  p.sin = a->sin;
  p.axes = (int)a->axes;
  p.rows = (uint32_t)a->rows;
  // Four rows a thread where that still fills the chip (131072 positions of 64
  // pairs 21.8 -> 18.5 us, 16384 with one row 5.8, with four 7.1).
  const int rows = a->rows * p.pairs / vec >= 4096 * (int64_t)device_cu_count() ? 4 : 1;
  p.step = (uint32_t)((a->rows + rows - 1) / rows);
  p.total = (uint32_t)(p.step * (uint64_t)p.pairs / vec);
  const uint32_t blocks = (uint32_t)(((uint64_t)p.total + kThreads - 1) / kThreads);
  if (!grid_fits(blocks, kThreads)) return fail(AA_EUNSUPPORTED, "rotary_tables: too many positions");
  const auto run = [&](auto v, auto r) {
    tables_kernel<decltype(v)::value, decltype(r)::value><<<blocks, kThreads, 0, (hipStream_t)stream>>>(p, a->position_type);
  };
  using I1 = std::integral_constant<int, 1>;
  using I4 = std::integral_constant<int, 4>;
  if (vec == 4) rows == 4 ? run(I4{}, I4{}) : run(I4{}, I1{});
  else rows == 4 ? run(I1{}, I4{}) : run(I1{}, I1{});
  return check_launch("rotary_tables");
}

extern "C" int aa_rotary(const aa_rotary_args* a, void* stream) {
  using namespace rotary;
  clear_error();
  if (!a) return fail(AA_EINVAL, "rotary: null args");
  if (a->dtype != AA_DTYPE_BF16 && a->dtype != AA_DTYPE_FP16 && a->dtype != AA_DTYPE_FP32)
    return fail(AA_EUNSUPPORTED, "rotary: dtype must be bf16, fp16 or fp32");
  if (a->B < 0 || a->S < 0 || a->H < 0 || a->Hk < 0) return fail(AA_EINVAL, "rotary: negative size");
  if (a->hd < 8 || a->hd % 8 || a->hd > 512) return fail(AA_EUNSUPPORTED, "rotary: head_dim must be a multiple of 8, 8 to 512");
  if (a->part < 2 || a->part % 2 || a->part > a->hd)
    return fail(AA_EUNSUPPORTED, "rotary: the turned part must be even, 2 to head_dim");
  if (a->B == 0 || a->S == 0 || a->H + a->Hk == 0) return AA_OK;
  if ((a->H && (!a->q || !a->q_out)) || (a->Hk && (!a->k || !a->k_out)) || !a->cos || !a->sin)
    return fail(AA_EINVAL, "rotary: null pointer");
  const int64_t elem = a->dtype == AA_DTYPE_FP32 ? 4 : 2, unit = 16 / elem;
  for (const void* ptr : {a->q, a->k, (const void*)a->q_out, (const void*)a->k_out, (const void*)a->cos, (const void*)a->sin})
    if (!aligned16(ptr)) return fail(AA_EINVAL, "rotary: pointers must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    for (const int64_t st : {a->q_stride[i], a->k_stride[i], a->q_out_stride[i], a->k_out_stride[i]})
      if (st % unit) return fail(AA_EINVAL, "rotary: strides must be multiples of 16 bytes");
  // The widest access that every unit of a head is aligned to.
  const int64_t side = a->interleaved ? a->part : a->part / 2;
  int64_t width = unit;
  while (side % width) width /= 2;
  if (a->table_stride < 0 || a->table_stride % (a->interleaved ? std::max<int64_t>(width / 2, 1) : width))
    return fail(AA_EINVAL, "rotary: bad table stride");
  TurnParams p = {};
  p.turned = (int)(side / width);
  p.units = p.turned + (int)((a->hd - a->part) / width);
  p.q = a->q;
  p.k = a->k;
  p.qo = a->q_out;
  p.ko = a->k_out;
  p.cos = a->cos;
  p.sin = a->sin;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_stride[i];
    p.ks[i] = a->k_stride[i];
    p.qos[i] = a->q_out_stride[i];
    p.kos[i] = a->k_out_stride[i];
  }
  p.table_stride = a->table_stride;
  p.S = (uint32_t)a->S;
  p.H = (int)a->H;
  p.heads = (int)(a->H + a->Hk);
  p.part = (int)a->part;
  p.sign = a->inverse ? -1.0f : 1.0f;
  const int64_t most = int64_t{0xffffffff} - kThreads;
  if (a->H > 65535 || a->Hk > 65535 || a->B > most / a->S || a->B * a->S > most / (p.heads * (int64_t)p.units))
    return fail(AA_EUNSUPPORTED, "rotary: too many values");
  const int64_t tokens = a->B * a->S;
  const int W = (int)(a->interleaved ? width / 2 : width);
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == AA_DTYPE_BF16) launch_turn<bf16>(p, tokens, W, a->interleaved != 0, st);
  else if (a->dtype == AA_DTYPE_FP16) launch_turn<_Float16>(p, tokens, W, a->interleaved != 0, st);
  else launch_turn<float>(p, tokens, W, a->interleaved != 0, st);
  return check_launch("rotary");
}
