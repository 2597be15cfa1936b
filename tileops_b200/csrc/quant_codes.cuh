// Shared by the kernels that quantise to 8 bits (quant_elem.cu, norm_quant.cu): vector packs, scale
// layouts, the output encodings, codes without a division per element, and running |x| maxima.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace tob {
namespace {

inline bool aligned_to(const void* p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0;
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> ld_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void st_pack(T* p, const Pack<T, V>& v) {
  *reinterpret_cast<Pack<T, V>*>(p) = v;
}

struct ScaleLayout {
  int64_t cm_rows;    // > 0: the reference's column_major_scales layout (see scale_offset)
  int64_t cm_groups;  // groups per row
  int64_t tma_ld = 0;  // > 0: TMA-aligned column-major scales, cm_groups groups per row
};

// Position of group g's scale. Natural order is g. With column_major_scales the reference
// returns s_flat.reshape(..., G_, M).transpose(-2, -1).contiguous() (quant_fp8.py:129-136):
// within each batch of M rows x G_ groups, flat scale t lands at row t % M, column t / M of
// a contiguous [M, G_] tensor.
// With tma_ld > 0 (the layout DeepGEMM-style kernels load with TMA): the scale of row r, group
// j of a 2-D input sits at j * tma_ld + r, tma_ld being the row count rounded up to 4 floats
// (16 bytes) so that every column starts 16-byte aligned.
__device__ __forceinline__ int64_t scale_offset(int64_t g, const ScaleLayout& sl) {
  if (sl.tma_ld > 0) {
    const int64_t r = g / sl.cm_groups;
    return (g - r * sl.cm_groups) * sl.tma_ld + r;
  }
  if (sl.cm_rows <= 0) return g;
  const int64_t per_batch = sl.cm_rows * sl.cm_groups;
  const int64_t b = g / per_batch;
  const int64_t t = g - b * per_batch;
  return b * per_batch + (t % sl.cm_rows) * sl.cm_groups + t / sl.cm_rows;
}

// 2^ceil(log2(max(s, 1e-30))) with log2 rounded to fp32 first, as torch evaluates
// torch.exp2(torch.ceil(torch.log2(s))) (quant_fp8.py:48-49).
__device__ __forceinline__ float ue8m0_round(float s) {
  if (isinf(s)) return s;
  s = fmaxf(s, 1e-30f);
  const float l = (float)log2((double)s);
  return ldexpf(1.0f, (int)ceilf(l));
}

// Output codes of the quantisers: int8, OCP float8_e4m3fn, or float8_e4m3fnuz (the encoding
// with exponent bias 8, no infinities, no negative zero and one NaN, 0x80; the reference's
// `dtype` argument accepts it, tileops/quant_fp8.py:19-45).
enum QKind : int { kQI8 = 0, kQE4M3 = 1, kQE4M3Fnuz = 2 };

// fp32 -> e4m3fnuz, round to nearest even, for |v| <= 240 (the quantisers clamp first). The
// fnuz grid is the e4m3fn grid halved (bias 8 against 7, same mantissa), so the code is the
// e4m3fn code of 2v, except: above 232 (the tie between 224 and 240) the nearest fnuz value is
// 240, code 0x7F, which e4m3fn spends on NaN; and e4m3fn's -0 (0x80) is fnuz's NaN, so a
// result of zero is +0.
__device__ __forceinline__ uint8_t f32_to_e4m3fnuz(float v) {
  uint8_t b = f32_to_e4m3(2.0f * v);
  if (fabsf(v) > 232.0f) b = (uint8_t)(((__float_as_uint(v) >> 24) & 0x80u) | 0x7Fu);
  return b == 0x80 ? (uint8_t)0 : b;
}
__device__ __forceinline__ float e4m3fnuz_to_f32(uint8_t b) {
  if (b == 0x80) return __uint_as_float(0x7FC00000u);
  if ((b & 0x7F) == 0x7F) return (b & 0x80) ? -240.0f : 240.0f;
  return 0.5f * e4m3_to_f32(b);
}

// e4m3 code of a NaN quotient x / scale, as the reference's fp32 division and cast produce it
// on the x86 host it is pinned to: with a NaN scale (a NaN in the group) the quotient is the
// NaN operand that comes first -- x itself when x is NaN, else the scale's sign-clear NaN --
// and the cast keeps its sign (0x7F or 0xFF); with a numeric scale the NaN comes from an
// invalid operation (inf / inf, 0 / 0), whose default NaN has the sign set (0xFF).
// `neg_x` is the sign bit of x as stored: the conversion of a 16-bit NaN to fp32 does not
// keep its sign on the GPU.
__device__ __forceinline__ uint8_t nan_code_div(float x, bool neg_x, bool nan_scale) {
  if (!nan_scale) return 0xFF;
  return (isnan(x) && neg_x) ? (uint8_t)0xFF : (uint8_t)0x7F;
}

// Codes of x / scale without a division per element: the bracket test. With r = 1 / scale
// rounded to fp32, lo = r (1 - 2^-21) and hi = r (1 + 2^-21), each rounded, the products x lo
// and x hi enclose both the exact quotient and its fp32 rounding: r, lo, hi and a rounded
// product are each off by at most 2^-24 relatively, 4 x 2^-24 in all, inside the 8 x 2^-24
// margin. Rounding onto the code grid (e4m3fn RNE with saturation, or RNE to an integer) is
// monotone, so when both products give the same code the correctly rounded quotient gives it
// too; a pack where they differ takes the IEEE division for every value. The test holds on the
// e4m3 subnormal grid and at saturation alike. It needs a scale whose reciprocal is a normal
// fp32 number and a group without NaN or infinity (a finite absmax); a scale within
// [1.2e-38, 8e37] implies both.
struct Bracket {
  float lo, hi;
};
__device__ __forceinline__ Bracket make_bracket(float scale) {
  const float r = __frcp_rn(scale);
  return {__fmul_rn(r, 1.0f - 0x1p-21f), __fmul_rn(r, 1.0f + 0x1p-21f)};
}

// RNE integer of the exact product x * m plus 1.5 x 2^23: for |x m| < 2^22 the sum's low bits
// are the integer in two's complement (its low byte is the int8 code).
__device__ __forceinline__ uint32_t rne_int_bits(float x, float m) {
  return __float_as_uint(__fmaf_rn(x, m, 12582912.0f));
}

// The code of the IEEE quotient x / scale (a finite x, a normal scale: no NaN can arise).
template <int Q> __device__ __forceinline__ uint32_t exact_code(float x, float scale) {
  const float y = __fdiv_rn(x, scale);
  if constexpr (Q == kQE4M3) return f32_to_e4m3(fminf(fmaxf(y, -448.f), 448.f));
  else return (uint8_t)rne_clamp_i8(y);
}

// Four codes from the two ends' codes wl, wh (byte j for x[j]): where they differ -- a quotient
// on or next to a rounding boundary, which bf16 inputs hit often since x / scale is then
// frequently an exact e4m3 midpoint -- that value alone divides.
template <int Q>
__device__ __noinline__ uint32_t fix_codes(uint32_t wl, uint32_t wh, float x0, float x1, float x2,
                                           float x3, float scale) {
  const float x[4] = {x0, x1, x2, x3};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (((wl ^ wh) >> (8 * j)) & 0xFFu)
      wl = (wl & ~(0xFFu << (8 * j))) | (exact_code<Q>(x[j], scale) << (8 * j));
  return wl;
}

// Codes of a pack by the bracket test, the products two lanes per instruction (mul.rn.f32x2 /
// fma.rn.f32x2 round each lane like the scalar forms). e4m3fn: a pair converts in one
// cvt.rn.satfinite.e4m3x2. int8: |x / scale| <= 127 (1 + 2^-22) on this path (scale =
// max(absmax, eps) / 127 rounded), so no value reaches the clamp, and the two ends differ by at
// most one, so their low bytes tell whether they differ. One branch per pack leads to the
// per-value fix-ups.
template <int Q, typename T, int V>
__device__ __forceinline__ void bracket_codes(const Pack<T, V>& t, const Bracket& b, float scale,
                                              Pack<uint8_t, V>& o) {
  if constexpr (V == 1) {
    const float x = to_f32(t.v[0]);
    uint32_t l, h;
    if constexpr (Q == kQE4M3) {
      const uint32_t c = f32x2_to_e4m3x2(__fmul_rn(x, b.lo), __fmul_rn(x, b.hi));
      l = c & 0xFFu;
      h = c >> 8;
    } else {
      l = rne_int_bits(x, b.lo) & 0xFFu;
      h = rne_int_bits(x, b.hi) & 0xFFu;
    }
    o.v[0] = (uint8_t)(l == h ? l : exact_code<Q>(x, scale));
  } else {
    static_assert(V % 4 == 0, "bracket_codes packs four codes to a word");
    constexpr int W = V / 4;
    const float2 lo2 = make_float2(b.lo, b.lo), hi2 = make_float2(b.hi, b.hi);
    uint32_t wl[W], wh[W], diff = 0u;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 x01 = make_float2(to_f32(t.v[4 * k]), to_f32(t.v[4 * k + 1]));
      const float2 x23 = make_float2(to_f32(t.v[4 * k + 2]), to_f32(t.v[4 * k + 3]));
      if constexpr (Q == kQE4M3) {
        const float2 l01 = mul2_rn(x01, lo2), h01 = mul2_rn(x01, hi2);
        const float2 l23 = mul2_rn(x23, lo2), h23 = mul2_rn(x23, hi2);
        wl[k] = __byte_perm(f32x2_to_e4m3x2(l01.x, l01.y), f32x2_to_e4m3x2(l23.x, l23.y), 0x5410);
        wh[k] = __byte_perm(f32x2_to_e4m3x2(h01.x, h01.y), f32x2_to_e4m3x2(h23.x, h23.y), 0x5410);
      } else {
        const float2 m2 = make_float2(12582912.0f, 12582912.0f);
        const float2 l01 = fma2_rn(x01, lo2, m2), h01 = fma2_rn(x01, hi2, m2);
        const float2 l23 = fma2_rn(x23, lo2, m2), h23 = fma2_rn(x23, hi2, m2);
        wl[k] = __byte_perm(__byte_perm(__float_as_uint(l01.x), __float_as_uint(l01.y), 0x0040),
                            __byte_perm(__float_as_uint(l23.x), __float_as_uint(l23.y), 0x0040),
                            0x5410);
        wh[k] = __byte_perm(__byte_perm(__float_as_uint(h01.x), __float_as_uint(h01.y), 0x0040),
                            __byte_perm(__float_as_uint(h23.x), __float_as_uint(h23.y), 0x0040),
                            0x5410);
      }
      diff |= wl[k] ^ wh[k];
    }
    if (diff != 0u) {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (wl[k] != wh[k])
          wl[k] = fix_codes<Q>(wl[k], wh[k], to_f32(t.v[4 * k]), to_f32(t.v[4 * k + 1]),
                               to_f32(t.v[4 * k + 2]), to_f32(t.v[4 * k + 3]), scale);
    }
    uint32_t* w = reinterpret_cast<uint32_t*>(o.v);
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = wl[k];
  }
}

// Running maximum of |x| over packs, read out as the abs_key of the largest |x|. 16-bit types
// keep the sign-cleared bit patterns two to a word and take halfword-wise unsigned maxima
// (max.u16x2): patterns of non-negative values order as the values, with NaNs above infinity,
// and the largest converts to the same fp32 key the per-value path finds.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T> struct AbsMax {
  unsigned k = 0u;
  template <int V> __device__ __forceinline__ void add(const Pack<T, V>& p) {
#pragma unroll
    for (int j = 0; j < V; ++j) k = max(k, abs_key(to_f32(p.v[j])));
  }
  __device__ __forceinline__ unsigned key() const { return k; }
};
__device__ __forceinline__ unsigned short bits16(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ unsigned short bits16(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
template <typename T> struct AbsMax16 {
  uint32_t k2 = 0u;
  template <int V> __device__ __forceinline__ void add(const Pack<T, V>& p) {
    if constexpr (V % 2 == 0) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(p.v);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) k2 = max_u16x2(k2, w[i] & 0x7FFF7FFFu);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        k2 = max(k2, (uint32_t)(bits16(p.v[j]) & 0x7FFFu));
    }
  }
  __device__ __forceinline__ unsigned key() const {
    const unsigned short m = (unsigned short)max(k2 & 0xFFFFu, k2 >> 16);
    if constexpr (std::is_same<T, __half>::value) return abs_key(__half2float(__ushort_as_half(m)));
    else return abs_key(__bfloat162float(__ushort_as_bfloat16(m)));
  }
};
template <> struct AbsMax<__half> : AbsMax16<__half> {};
template <> struct AbsMax<__nv_bfloat16> : AbsMax16<__nv_bfloat16> {};

// Sign bit of a stored value.
__device__ __forceinline__ bool sign_of(float v) { return __float_as_uint(v) >> 31; }
__device__ __forceinline__ bool sign_of(__half v) { return __half_as_ushort(v) >> 15; }
__device__ __forceinline__ bool sign_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v) >> 15; }

}  // namespace
}  // namespace tob
