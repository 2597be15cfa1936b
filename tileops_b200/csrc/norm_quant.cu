// Residual add, root-mean-square norm and 8-bit quantisation of a row in one pass:
//   h = x + r;  rstd = (mean(h^2) + eps)^(-1/2);  y = (h w) rstd
//   per group of G columns: s = max(max|y|, quant_eps) / qmax, q = e4m3 or int8 codes of y / s
// and h, rounded to the input type, as the next residual. The sums, the norm and the quotients are
// fp32; nothing is rounded to the input type on the way to the codes.
//
// rstd is one factor of a whole row, so what waits for the row's sum is one number: p = h w stays in
// registers, max|y| = rstd max|p| per group, and a code is the code of p c with c = rstd / s.
//
// Bound by HBM: 2 + 2 B read, 2 + 1 B written per element (16-bit input); x and r are read once by
// rows that a block holds: 16-bit rows of up to 16384 columns where there are as many SMs as rows, of
// 8192 up to two rows an SM, of 12288 beyond. What a longer row has left is read again, once or
// (groups off the packs) twice, mostly from L2. A
// team of threads (whole warps) holds a row, MAXV 16-byte packs per thread; the group maxima are
// shuffles where a group is a power-of-two number of packs within a warp, the team's reduction
// (with the sum's) where it is the row, and shared-memory maxima (order-independent) for any other
// group size. Few rows take one or two packs per thread: their time is the latency of one load.
#include <string.h>

#include <algorithm>

#include "quant_codes.cuh"

namespace tob {
namespace {

enum GroupMode : int { kGroupLanes = 0, kGroupRow = 1, kGroupShared = 2 };

struct NormArgs {
  const void* x;
  const void* r;       // null: no residual
  const void* w;
  void* h;             // residual output, null without r; may be x or r
  uint8_t* q;
  float* scales;
  int64_t rows, cols, ldx, ldr, ldh;
  int G;               // columns per group
  int team;            // threads per row, a multiple of 32
  int rows_per_block, nvec, groups, lanes_log2;
  float eps, quant_eps, qmax, qmax_inv, cols_inv;
  float floor_factor;  // qmax / quant_eps
  int ue8m0;
  ScaleLayout sl;
};

// Data that pass once: x and r are not read again, h and the codes not before another kernel. Marked
// to leave L2 first, they do not push one another out (8192 x 8192 back to back: 88 us unmarked,
// 80.5 with loads and stores marked, 81 with the stores alone; a product that follows reads the codes
// as fast).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> ld_once(const T* p) {
  Pack<T, V> o;
  if constexpr (sizeof(o) == 16) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    memcpy(&o, &u, 16);
  } else if constexpr (sizeof(o) == 8) {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    memcpy(&o, &u, 8);
  } else {
    o = ld_pack<T, V>(p);
  }
  return o;
}
template <typename T, int V>
__device__ __forceinline__ void st_once(T* p, const Pack<T, V>& v) {
  if constexpr (sizeof(v) == 16) {
    uint4 u;
    memcpy(&u, &v, 16);
    __stcs(reinterpret_cast<uint4*>(p), u);
  } else if constexpr (sizeof(v) == 8) {
    uint2 u;
    memcpy(&u, &v, 8);
    __stcs(reinterpret_cast<uint2*>(p), u);
  } else if constexpr (sizeof(v) == 4) {
    unsigned u;
    memcpy(&u, &v, 4);
    __stcs(reinterpret_cast<unsigned*>(p), u);
  } else {
    st_pack<T, V>(p, v);
  }
}

// max(|v|, m), NaN when either is.
__device__ __forceinline__ float max_abs_nan(float v, float m) {
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %1;\n\tmax.NaN.f32 %0, t, %2;\n\t}" : "=f"(m) : "f"(v), "f"(m));
  return m;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
  return a;
}

// x + r of a pack in fp32. 16-bit values go straight into mixed-precision products with one, which
// convert and add in the same instruction.
template <typename T, int V, bool RES>
__device__ __forceinline__ Pack<float, V> sum_packs(const Pack<T, V>& px, const Pack<T, V>& pr) {
  Pack<float, V> o;
  if constexpr (RES && V > 1 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      asm("{\n\t.reg .b16 xl, xh, rl, rh, one;\n\tmov.b32 {xl, xh}, %2;\n\tmov.b32 {rl, rh}, %3;\n\t"
          "mov.b16 one, 0x3F80;\n\t"
          "fma.rn.f32.bf16 %0, rl, one, 0f00000000;\n\tfma.rn.f32.bf16 %1, rh, one, 0f00000000;\n\t"
          "fma.rn.f32.bf16 %0, xl, one, %0;\n\tfma.rn.f32.bf16 %1, xh, one, %1;\n\t}"
          : "=&f"(o.v[j]), "=&f"(o.v[j + 1])
          : "r"(*reinterpret_cast<const uint32_t*>(px.v + j)),
            "r"(*reinterpret_cast<const uint32_t*>(pr.v + j)));
  } else if constexpr (RES && V > 1 && std::is_same<T, __half>::value) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      asm("{\n\t.reg .b16 xl, xh, rl, rh, one;\n\tmov.b32 {xl, xh}, %2;\n\tmov.b32 {rl, rh}, %3;\n\t"
          "mov.b16 one, 0x3C00;\n\t"
          "fma.rn.f32.f16 %0, rl, one, 0f00000000;\n\tfma.rn.f32.f16 %1, rh, one, 0f00000000;\n\t"
          "fma.rn.f32.f16 %0, xl, one, %0;\n\tfma.rn.f32.f16 %1, xh, one, %1;\n\t}"
          : "=&f"(o.v[j]), "=&f"(o.v[j + 1])
          : "r"(*reinterpret_cast<const uint32_t*>(px.v + j)),
            "r"(*reinterpret_cast<const uint32_t*>(pr.v + j)));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      o.v[j] = to_f32(px.v[j]);
      if constexpr (RES) o.v[j] += to_f32(pr.v[j]);
    }
  }
  return o;
}

// scale = clamp(max|y|, min = quant_eps) / qmax; a NaN maximum passes through unchanged.
template <int Q>
__device__ __forceinline__ float scale_of(float maxp, float rstd, const NormArgs& a) {
  const float m = maxp * rstd;
  if (isnan(m)) return __uint_as_float(0x7FC00000u);
  // The IEEE quotient by the constant: qmax_inv is the rounded reciprocal, one correction makes the
  // rounded quotient of it (fp32 subnormal results excepted, where it may be one step off).
  const float n = fmaxf(m, a.quant_eps), t = n * a.qmax_inv;
  float s = isinf(n) ? n : fmaf(fmaf(-t, a.qmax, n), a.qmax_inv, t);
  if (Q == kQE4M3 && a.ue8m0) s = ue8m0_round(s);
  return s;
}

// The factor rstd / s of a group in two terms (c, what rounding c left out): qmax / max|p|, or what
// the floor of the scale leaves. With the second term a quotient that is a tie, half the largest
// value say, comes out as one. (0, 0) stands for the groups whose codes need a division each (a NaN
// or an infinity, or numbers near the ends of fp32's range).
template <int Q>
__device__ __forceinline__ float2 code_factor(float maxp, float rstd, const NormArgs& a) {
  const float m = maxp * rstd;
  const bool free = m > a.quant_eps && !(Q == kQE4M3 && a.ue8m0);
  float c = free ? __fdiv_rn(a.qmax, maxp) : rstd * a.floor_factor;
  if (Q == kQE4M3 && a.ue8m0) c = __fdiv_rn(rstd, scale_of<Q>(maxp, rstd, a));
  const float lo = free ? fmaf(-c, maxp, a.qmax) * (c * a.qmax_inv) : 0.f;
  const bool plain = m <= 1e30f && maxp <= 1e30f && (maxp >= 1e-30f || maxp == 0.f) &&
                     c <= 1e30f;  // false for NaN
  return plain ? make_float2(c, lo) : make_float2(0.f, 0.f);
}

// The codes of V values p c. With a factor every value is finite and |p c| <= qmax (1 + 2^-22),
// which saturates (e4m3) or rounds (int8) to qmax.
template <int Q, int V>
__device__ __forceinline__ Pack<uint8_t, V> codes_of(const Pack<float, V>& f, float2 c) {
  Pack<uint8_t, V> o;
  auto z = [&](int j) { return fmaf(f.v[j], c.x, f.v[j] * c.y); };
  // the low byte of z + 1.5 x 2^23 is rint(z)
  auto i8 = [&](int j) { return __float_as_uint(z(j) + 12582912.0f); };
  if constexpr (V == 1) {
    o.v[0] = Q == kQE4M3 ? f32_to_e4m3(z(0)) : (uint8_t)i8(0);
  } else if constexpr (V == 2) {
    uint16_t w;
    if constexpr (Q == kQE4M3) w = f32x2_to_e4m3x2(z(0), z(1));
    else w = (uint16_t)__byte_perm(i8(0), i8(1), 0x0040);
    *reinterpret_cast<uint16_t*>(o.v) = w;
  } else {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      uint32_t lo, hi;
      if constexpr (Q == kQE4M3) {
        lo = f32x2_to_e4m3x2(z(k), z(k + 1));
        hi = f32x2_to_e4m3x2(z(k + 2), z(k + 3));
      } else {
        lo = __byte_perm(i8(k), i8(k + 1), 0x0040);
        hi = __byte_perm(i8(k + 2), i8(k + 3), 0x0040);
      }
      reinterpret_cast<uint32_t*>(o.v)[k / 4] = __byte_perm(lo, hi, 0x5410);
    }
  }
  return o;
}
// One code by division, for the groups without a factor. Out of line: it is never fetched else.
template <int Q>
__device__ __noinline__ uint8_t divided_code(float p, float rstd, float s) {
  const float z = __fdiv_rn(p * rstd, s);
  if (Q == kQE4M3) return isnan(z) ? (uint8_t)0x7F : f32_to_e4m3(fminf(fmaxf(z, -448.f), 448.f));
  return (uint8_t)rne_clamp_i8(z);
}

// Threads of a block at most, and blocks of an SM the registers are sized for. 32 values a thread
// (four 16-byte packs of 16-bit values) want 80 registers, 16 or fewer fit 64 (16 single values do
// not: that form spills some 100 to 500 bytes). Many rows run on blocks of 512 threads at most, so
// that an SM always holds two and one's loads cover the other's arithmetic (a row of 13248 columns on
// one block of 832 threads per SM took three times as long); what a longer row has left is re-read.
// Two packs of 16-bit values serve few rows alone, see block_threads.
template <int V, int MAXV> constexpr bool kFewRows = V == 8 && MAXV == 2;
template <int V, int MAXV>
constexpr int kBlockMax = V * MAXV > 16 ? 384 : V * MAXV == 16 && !kFewRows<V, MAXV> ? 512 : 1024;
template <int V, int MAXV>
constexpr int kBlocksMin = V * MAXV >= 16 && !kFewRows<V, MAXV> ? 2 : 1;

// One block per rows_per_block rows, a team of threads each. RES: with a residual and its output.
// Loads are not guarded but clamped (rows and packs past the end re-read the last and count as
// zero), so that all of a thread's loads go out together. 8192 x 8192 bf16 -> e4m3 with residual:
// 80.5 us back to back, 5.9 TB/s (floor at the copy rate 73); a persistent form fed by bulk copies into
// shared memory ran no faster.
template <typename T, int Q, int V, int MAXV, int MODE, bool RES>
__global__ void __launch_bounds__(kBlockMax<V, MAXV>, kBlocksMin<V, MAXV>)
    k_norm_quant(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][32];
  extern __shared__ unsigned gmax[];  // kGroupShared: [rows of the CTA][groups]
  // Launched as a programmatic dependent: blocks may start while the previous kernel drains, and
  // wait for its completion before they touch memory or let the next kernel start.
  grid_dependency_wait();
  grid_dependents_launch();
  const int team = a.team;
  int tid = (int)threadIdx.x, local = 0;
  if (team < (int)blockDim.x) {
    local = tid / team;
    tid -= local * team;
  }
  const int64_t row = (int64_t)blockIdx.x * a.rows_per_block + local;
  const bool active = row < a.rows;
  const int nvec = a.nvec, groups = a.groups;
  const int64_t lrow = active ? row : a.rows - 1;
  const T* x = (const T*)a.x + lrow * a.ldx;
  const T* r = RES ? (const T*)a.r + lrow * a.ldr : nullptr;
  const T* w = (const T*)a.w;
  T* h = RES ? (T*)a.h + lrow * a.ldh : nullptr;
  uint8_t* q = a.q + lrow * a.cols;
  using F = Pack<float, V>;

  auto store_h = [&](int v, const F& f) {
    if constexpr (RES) {
      Pack<T, V> o;
      if constexpr (V > 1 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int j = 0; j < V; j += 2)
          *reinterpret_cast<__nv_bfloat162*>(o.v + j) = __floats2bfloat162_rn(f.v[j], f.v[j + 1]);
      } else if constexpr (V > 1 && std::is_same<T, __half>::value) {
#pragma unroll
        for (int j = 0; j < V; j += 2)
          *reinterpret_cast<__half2*>(o.v + j) = __floats2half2_rn(f.v[j], f.v[j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = from_f32<T>(f.v[j]);
      }
      st_once<T, V>(h + (int64_t)v * V, o);
    }
  };
  auto load_h = [&](int v) {
    Pack<T, V> pr;
    if constexpr (RES) pr = ld_pack<T, V>(r + (int64_t)v * V);
    return sum_packs<T, V, RES>(ld_pack<T, V>(x + (int64_t)v * V), pr);
  };
  auto weigh = [&](F& f, const Pack<T, V>& pw) {
#pragma unroll
    for (int j = 0; j < V; ++j) f.v[j] *= to_f32(pw.v[j]);
  };
  float ss = 0.f, rowmax = 0.f;
  auto square = [&](const F& f) {
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fmaf(f.v[j], f.v[j], ss);
  };
  auto max_of = [&](const F& f, float m) {
#pragma unroll
    for (int j = 0; j < V; ++j) m = max_abs_nan(f.v[j], m);
    return m;
  };

  // Packs past MAXV are re-read in each pass; their h is stored in the last one, since it may
  // overwrite x or r.
  F y[MAXV];
  {
    Pack<T, V> px[MAXV], pr[MAXV];
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int v = min(tid + i * team, nvec - 1);
      px[i] = ld_once<T, V>(x + (int64_t)v * V);
      if constexpr (RES) pr[i] = ld_once<T, V>(r + (int64_t)v * V);
    }
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int v = tid + i * team;
      const Pack<T, V> pw = ld_pack<T, V>(w + (int64_t)min(v, nvec - 1) * V);
      y[i] = sum_packs<T, V, RES>(px[i], pr[i]);
      if (v < nvec) {
        if (active) store_h(v, y[i]);
        square(y[i]);
        weigh(y[i], pw);
        if constexpr (MODE == kGroupRow) rowmax = max_of(y[i], rowmax);
      } else if constexpr (MODE == kGroupLanes) {  // counts as zero in the shuffled maxima
#pragma unroll
        for (int j = 0; j < V; ++j) y[i].v[j] = 0.f;
      }
    }
  }
  for (int v = tid + MAXV * team; v < nvec; v += team) {
    F f = load_h(v);
    square(f);
    if constexpr (MODE == kGroupRow) {
      weigh(f, ld_pack<T, V>(w + (int64_t)v * V));
      rowmax = max_of(f, rowmax);
    }
  }
  // The team's sum, and with one scale per row its maximum.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (MODE == kGroupRow) rowmax = max_nan(rowmax, __shfl_xor_sync(0xffffffffu, rowmax, o));
  }
  if (team > 32) {
    const int warp = threadIdx.x >> 5, warps = team >> 5, w0 = local * warps;
    if ((threadIdx.x & 31) == 0) {
      red[0][warp] = ss;
      if constexpr (MODE == kGroupRow) red[1][warp] = rowmax;
    }
    __syncthreads();
    // Lane l takes warp l's number; every warp adds them up alike.
    const int l = threadIdx.x & 31;
    ss = l < warps ? red[0][w0 + l] : 0.f;
    if constexpr (MODE == kGroupRow) rowmax = l < warps ? red[1][w0 + l] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if constexpr (MODE == kGroupRow)
        rowmax = max_nan(rowmax, __shfl_xor_sync(0xffffffffu, rowmax, o));
    }
  }
  const float rstd = rsqrtf(fmaf(ss, a.cols_inv, a.eps));

  float* scales = a.scales + lrow * groups;
  auto put_scale = [&](int g, float s) {
    if (a.sl.cm_rows > 0) a.scales[scale_offset(row * groups + g, a.sl)] = s;
    else scales[g] = s;
  };
  // Codes of a pack whose group has the maximum maxp.
  auto emit = [&](int v, const F& f, float maxp, float2 c) {
    Pack<uint8_t, V> o;
    if (c.x != 0.f) {
      o = codes_of<Q, V>(f, c);
    } else {
      const float s = scale_of<Q>(maxp, rstd, a);
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = divided_code<Q>(f.v[j], rstd, s);
    }
    st_once<uint8_t, V>(q + (int64_t)v * V, o);
  };

  if constexpr (MODE == kGroupLanes) {
    // A group is `lanes` consecutive packs: packs of one i are consecutive over the team's
    // threads and the team is whole warps, so a group never leaves its warp.
    const int shift = a.lanes_log2;
    auto group_max = [&](float m) {
#pragma unroll
      for (int b = 0; b < 5; ++b)
        if (b < shift) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1 << b));
      return m;
    };
    auto finish = [&](int v, const F& f, float m) {
      if (!active || v >= nvec) return;
      if ((v & ((1 << shift) - 1)) == 0) put_scale(v >> shift, scale_of<Q>(m, rstd, a));
      emit(v, f, m, code_factor<Q>(m, rstd, a));
    };
    if (MAXV > 1 && shift >= 2) {
      // Lane i of a group works out the scale and the factor of the thread's i-th pack, once per
      // row instead of once per pack.
      static_assert(MAXV <= 4, "lane i of a group of four or more");
      float m[MAXV];
#pragma unroll
      for (int i = 0; i < MAXV; ++i) m[i] = group_max(max_of(y[i], 0.f));
      const int lane = threadIdx.x & 31, i_mine = lane & ((1 << shift) - 1);
      float mine = m[0];
#pragma unroll
      for (int i = 1; i < MAXV; ++i) mine = i == i_mine ? m[i] : mine;
      const int v_mine = tid + i_mine * team;
      if (active && i_mine < MAXV && v_mine < nvec)
        put_scale(v_mine >> shift, scale_of<Q>(mine, rstd, a));
      const float2 c = code_factor<Q>(mine, rstd, a);
#pragma unroll
      for (int i = 0; i < MAXV; ++i) {
        const float2 ci = make_float2(__shfl_sync(0xffffffffu, c.x, lane - i_mine + i),
                                      __shfl_sync(0xffffffffu, c.y, lane - i_mine + i));
        if (active && tid + i * team < nvec) emit(tid + i * team, y[i], m[i], ci);
      }
    } else {
#pragma unroll
      for (int i = 0; i < MAXV; ++i)
        finish(tid + i * team, y[i], group_max(max_of(y[i], 0.f)));
    }
    // uniform trip count: the shuffles need all lanes
    for (int v = tid + MAXV * team; v - tid < nvec; v += team) {
      F f;
#pragma unroll
      for (int j = 0; j < V; ++j) f.v[j] = 0.f;
      if (v < nvec) {
        f = load_h(v);
        if (active) store_h(v, f);
        weigh(f, ld_pack<T, V>(w + (int64_t)v * V));
      }
      finish(v, f, group_max(max_of(f, 0.f)));
    }
  } else {
    unsigned* gm = gmax + local * groups;
    if constexpr (MODE == kGroupRow) {
      if (active && tid == 0) put_scale(0, scale_of<Q>(rowmax, rstd, a));
    } else {
      for (int g = tid; g < groups; g += team) gm[g] = 0u;
      __syncthreads();
      // Bit patterns of non-negative floats order as the floats, NaN above all.
      auto note = [&](int v, const F& f) {
        atomicMax(gm + (v * V) / a.G, __float_as_uint(max_of(f, 0.f)));
      };
#pragma unroll
      for (int i = 0; i < MAXV; ++i)
        if (tid + i * team < nvec) note(tid + i * team, y[i]);
      for (int v = tid + MAXV * team; v < nvec; v += team) {
        F f = load_h(v);
        weigh(f, ld_pack<T, V>(w + (int64_t)v * V));
        note(v, f);
      }
      __syncthreads();
      for (int g = tid; active && g < groups; g += team)
        put_scale(g, scale_of<Q>(__uint_as_float(gm[g]), rstd, a));
    }
    const float2 c_row =
        MODE == kGroupRow ? code_factor<Q>(rowmax, rstd, a) : make_float2(0.f, 0.f);
    auto finish = [&](int v, const F& f) {
      if constexpr (MODE == kGroupRow) {
        emit(v, f, rowmax, c_row);
      } else {
        const float m = __uint_as_float(gm[(v * V) / a.G]);
        emit(v, f, m, code_factor<Q>(m, rstd, a));
      }
    };
#pragma unroll
    for (int i = 0; i < MAXV; ++i)
      if (active && tid + i * team < nvec) finish(tid + i * team, y[i]);
    for (int v = tid + MAXV * team; active && v < nvec; v += team) {
      F f = load_h(v);
      store_h(v, f);
      weigh(f, ld_pack<T, V>(w + (int64_t)v * V));
      finish(v, f);
    }
  }
}

// Threads a block has at most. Two packs a thread: 1024 threads hold a row of 2048 packs where every
// row has an SM to itself; with more rows two blocks of 512 on an SM are faster although they read
// the rest of a row again. fp16, G = row, 16384 columns: 64 rows 3.83 us on 512 threads, 3.44 on 1024;
// 256 rows 6.65 and 8.19 (11008 columns: 3.22, 2.92; 5.02, 6.45). Four packs on 384 threads: 4.27 and
// 6.75 (3.26, 4.91).
template <int V, int MAXV>
int block_threads(int64_t rows) {
  return kFewRows<V, MAXV> && rows > sm_count() ? 512 : kBlockMax<V, MAXV>;
}

template <typename T, int Q, int V, int MAXV, int MODE>
int launch_norm(NormArgs a, cudaStream_t st) {
  auto kern = a.h != nullptr ? k_norm_quant<T, Q, V, MAXV, MODE, true>
                             : k_norm_quant<T, Q, V, MAXV, MODE, false>;
  const int64_t nvec = a.cols / V;
  int64_t team = ceil_div(ceil_div(nvec, MAXV), 32) * 32;
  team = std::min<int64_t>(team, block_threads<V, MAXV>(a.rows));
  a.team = (int)team;
  // Small rows share a CTA of up to 256 threads.
  int64_t per_cta = std::max<int64_t>(1, 256 / team);
  const int64_t groups = a.cols / a.G;
  size_t smem = 0;
  if (MODE == kGroupShared) {
    while (per_cta > 1 && per_cta * groups * 4 > 48 * 1024) per_cta /= 2;
    smem = (size_t)(per_cta * groups * 4);
    if (smem > 200 * 1024)
      return fail(TO_EUNSUPPORTED, "add_rms_norm_group_quant: %lld groups in a row (at most 51200)",
                  (long long)groups);
    const cudaError_t e = ensure_smem_attr((const void*)kern, 200 * 1024);
    if (e != cudaSuccess) return cuda_fail(e, "add_rms_norm_group_quant: shared memory attribute");
  }
  a.rows_per_block = (int)per_cta;
  a.nvec = (int)nvec;
  a.groups = (int)groups;
  a.lanes_log2 = 0;
  while (MODE == kGroupLanes && (V << a.lanes_log2) < a.G) ++a.lanes_log2;
  const int64_t blocks = ceil_div(a.rows, per_cta);
  if (blocks > INT32_MAX) return fail(TO_EUNSUPPORTED, "add_rms_norm_group_quant: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3((unsigned)(team * per_cta), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return cuda_fail(e, "add_rms_norm_group_quant launch");
  return check_launch("add_rms_norm_group_quant");
}

// Whether packs of v values can be used: the row length, the group, every row start.
template <typename T>
bool packs_of(const NormArgs& a, int v) {
  const size_t b = v * sizeof(T);
  return a.cols % v == 0 && a.G % v == 0 && aligned_to(a.x, b) && aligned_to(a.w, b) &&
         a.ldx % v == 0 && aligned_to(a.q, v) &&
         (!a.r || (aligned_to(a.r, b) && a.ldr % v == 0 && aligned_to(a.h, b) && a.ldh % v == 0));
}

template <typename T, int Q>
int launch_norm_any(const NormArgs& a, cudaStream_t st) {
  constexpr int VV = 16 / sizeof(T);
  auto narrow = [&](auto v) {  // sixteen values a thread
    constexpr int V = decltype(v)::value;
    return a.G == a.cols ? launch_norm<T, Q, V, 16 / V, kGroupRow>(a, st)
                         : launch_norm<T, Q, V, 16 / V, kGroupShared>(a, st);
  };
  if (!packs_of<T>(a, VV)) {
    if (VV > 4 && packs_of<T>(a, 4)) return narrow(std::integral_constant<int, 4>{});
    if (packs_of<T>(a, 2)) return narrow(std::integral_constant<int, 2>{});
    return narrow(std::integral_constant<int, 1>{});
  }
  const int lanes = a.G / VV;
  const int mode = lanes <= 32 && (lanes & (lanes - 1)) == 0 ? kGroupLanes
                   : a.G == a.cols                          ? kGroupRow
                                                            : kGroupShared;
  if (mode == kGroupShared) return launch_norm<T, Q, VV, 4, kGroupShared>(a, st);
  // Packs per thread: few rows (two per SM) take one where a block holds the row so and two up to
  // 2048 packs, for latency; many, and longer rows, take four, for bytes in flight at few threads.
  const int64_t nvec = a.cols / VV;
  const int maxv = a.rows > 2 * sm_count() || nvec > 2048 ? 4 : nvec <= 1024 ? 1 : 2;
  auto run = [&](auto m) {
    constexpr int MODE = decltype(m)::value;
    if (maxv == 1) return launch_norm<T, Q, VV, 1, MODE>(a, st);
    if (maxv == 2) return launch_norm<T, Q, VV, 2, MODE>(a, st);
    return launch_norm<T, Q, VV, 4, MODE>(a, st);
  };
  return mode == kGroupLanes ? run(std::integral_constant<int, kGroupLanes>{})
                             : run(std::integral_constant<int, kGroupRow>{});
}

}  // namespace
}  // namespace tob

extern "C" int to_add_rms_norm_group_quant(
    const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int dtype,
    int64_t rows, int64_t cols, int64_t group_size, float eps, float quant_eps, int ue8m0,
    int column_major, int q_dtype, void* q, float* scales, void* residual_out, int64_t ldh,
    void* stream) {
  using namespace tob;
  const char* op = "add_rms_norm_group_quant";
  if (rows < 0 || cols < 0 || cols > kDimMax || group_size <= 0 || cols % group_size != 0 ||
      (rows > 1 && (ldx < cols || (residual && ldr < cols) || (residual_out && ldh < cols))))
    return fail(TO_EINVAL, "%s: invalid shape rows=%lld cols=%lld group=%lld strides=(%lld, %lld, "
                "%lld)", op, (long long)rows, (long long)cols, (long long)group_size,
                (long long)ldx, (long long)ldr, (long long)ldh);
  if (!(quant_eps >= 1e-35f && quant_eps < 3e38f) || !(eps >= 0.0f && eps < 3e38f))
    return fail(TO_EINVAL, "%s: eps=%g must be at least 0, quant_eps=%g at least 1e-35", op,
                (double)eps, (double)quant_eps);
  if (q_dtype != TO_E4M3 && q_dtype != TO_I8)
    return fail(TO_EUNSUPPORTED, "%s: codes %s (float8_e4m3fn or int8)", op, dtype_name(q_dtype));
  if (q_dtype == TO_I8 && (ue8m0 || column_major))
    return fail(TO_EINVAL, "%s: ue8m0 / column-major scales are FP8 options", op);
  if (rows == 0 || cols == 0) return TO_OK;
  if (!x || !weight || !q || !scales) return fail(TO_EINVAL, "%s: null pointer", op);
  if ((residual == nullptr) != (residual_out == nullptr))
    return fail(TO_EINVAL, "%s: a residual and its output go together", op);
  NormArgs a;
  a.x = x;
  a.r = residual;
  a.w = weight;
  a.h = residual_out;
  a.q = (uint8_t*)q;
  a.scales = scales;
  a.rows = rows;
  a.cols = cols;
  a.ldx = ldx;
  a.ldr = ldr;
  a.ldh = ldh;
  a.G = (int)group_size;
  a.team = 0;
  a.eps = eps;
  a.quant_eps = quant_eps;
  a.qmax = q_dtype == TO_E4M3 ? 448.0f : 127.0f;
  a.qmax_inv = 1.0f / a.qmax;
  a.cols_inv = 1.0f / (float)cols;
  a.floor_factor = a.qmax / quant_eps;
  a.ue8m0 = ue8m0;
  a.sl = ScaleLayout{column_major ? rows : 0, column_major ? cols / group_size : 1};
  cudaStream_t st = (cudaStream_t)stream;
  TOB_DISPATCH_FLOAT(dtype, T, {
    return q_dtype == TO_E4M3 ? launch_norm_any<T, kQE4M3>(a, st)
                              : launch_norm_any<T, kQI8>(a, st);
  });
  return TO_OK;
}
