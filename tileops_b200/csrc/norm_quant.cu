// Residual add, root-mean-square norm and 8-bit quantisation of a row in one pass:
//   h = x + r;  rstd = (mean(h^2) + eps)^(-1/2);  y = (h rstd) w
//   per group of G columns: s = max(max|y|, quant_eps) / qmax, q = e4m3 or int8 codes of y / s
// and h, rounded to the input type, as the next residual. The sums, the norm and the quotients are
// fp32; nothing is rounded to the input type on the way to the codes.
//
// Bound by HBM: 2 + 2 B read, 2 + 1 B written per element (16-bit input), so the row stays in
// registers between its reduction and its codes and x, r are read once. A team of threads (whole
// warps) holds a row, MAXV 16-byte packs per thread; the group maxima are shuffles where a group
// is a power-of-two number of packs within a warp, the team's reduction where it is the row, and
// shared-memory maxima (order-independent) for any other group size.
#include <algorithm>

#include "quant_codes.cuh"

namespace tob {
namespace {

enum GroupMode : int { kGroupLanes = 0, kGroupRow = 1, kGroupShared = 2 };

struct NormArgs {
  const void* x;
  const void* r;       // null: no residual
  const void* w;
  void* h;             // null: no residual output; may be x or r
  uint8_t* q;
  float* scales;
  int64_t rows, cols, ldx, ldr, ldh;
  int G;               // columns per group
  int team;            // threads per row, a multiple of 32
  float eps, quant_eps, qmax;
  int ue8m0;
  ScaleLayout sl;
};

// Maximum key / sum over the team. `red`: one word per warp of the CTA. Every thread of the CTA
// calls it; the barrier in front separates uses of `red`.
template <typename R, typename F>
__device__ __forceinline__ R team_reduce(R v, int team, R* red, F op) {
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (team == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  const int warps = team >> 5, w0 = warp / warps * warps;
  R t = red[w0];
  for (int i = 1; i < warps; ++i) t = op(t, red[w0 + i]);
  return t;
}

template <typename T, int Q, int V, int MAXV, int MODE>
__global__ void __launch_bounds__(1024) k_norm_quant(const NormArgs a) {
  __shared__ float red_sum[32];
  __shared__ unsigned red_max[32];
  extern __shared__ unsigned gmax[];  // kGroupShared: [rows of the CTA][groups]
  // Launched as a programmatic dependent: blocks may start while the previous kernel drains, and
  // wait for its completion before they touch memory.
  grid_dependents_launch();
  grid_dependency_wait();
  const int team = a.team;
  const int tid = (int)threadIdx.x % team, local = (int)threadIdx.x / team;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / team) + local;
  const bool active = row < a.rows;
  const int nvec = (int)(a.cols / V);
  const int groups = (int)(a.cols / a.G);
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const T* w = (const T*)a.w;
  T* h = a.h ? (T*)a.h + row * a.ldh : nullptr;
  using F = Pack<float, V>;

  auto load_h = [&](int v) {
    F o;
    const Pack<T, V> px = ld_pack<T, V>(x + (int64_t)v * V);
    if (r != nullptr) {
      const Pack<T, V> pr = ld_pack<T, V>(r + (int64_t)v * V);
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = to_f32(px.v[j]) + to_f32(pr.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = to_f32(px.v[j]);
    }
    return o;
  };
  auto store_h = [&](int v, const F& f) {
    if (h == nullptr) return;
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = from_f32<T>(f.v[j]);
    st_pack<T, V>(h + (int64_t)v * V, o);
  };

  // h of this thread's packs, and the row's sum of squares. Packs past MAXV are re-read in each
  // pass; their h is stored in the last one, since it may overwrite x or r.
  F y[MAXV];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int v = tid + i * team;
    if (active && v < nvec) y[i] = load_h(v);
  }
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int v = tid + i * team;
    if (active && v < nvec) {
      store_h(v, y[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) ss = fmaf(y[i].v[j], y[i].v[j], ss);
    }
  }
  for (int v = tid + MAXV * team; active && v < nvec; v += team) {
    const F f = load_h(v);
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fmaf(f.v[j], f.v[j], ss);
  }
  ss = team_reduce(ss, team, red_sum, [](float p, float q) { return p + q; });
  const float rstd = __frsqrt_rn(ss / (float)a.cols + a.eps);

  auto norm = [&](int v, F f) {
    const Pack<T, V> pw = ld_pack<T, V>(w + (int64_t)v * V);
#pragma unroll
    for (int j = 0; j < V; ++j) f.v[j] = f.v[j] * rstd * to_f32(pw.v[j]);
    return f;
  };
  auto key_of = [&](const F& f) {
    unsigned k = 0u;
#pragma unroll
    for (int j = 0; j < V; ++j) k = max(k, abs_key(f.v[j]));
    return k;
  };
  // scale = clamp(absmax, min = quant_eps) / qmax; a NaN absmax passes through unchanged.
  auto scale_of = [&](unsigned key) {
    const float m = __uint_as_float(key);
    if (isnan(m)) return m;
    float s = __fdiv_rn(fmaxf(m, a.quant_eps), a.qmax);
    if (Q == kQE4M3 && a.ue8m0) s = ue8m0_round(s);
    return s;
  };
  auto put_scale = [&](int g, float s) { a.scales[scale_offset(row * groups + g, a.sl)] = s; };
  auto emit = [&](int v, const F& f, float s) {
    Pack<uint8_t, V> o;
    if (s >= 1.2e-38f && s <= 8.0e37f) {
      bracket_codes<Q>(f, make_bracket(s), s, o);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float z = __fdiv_rn(f.v[j], s);
        if (Q == kQE4M3)
          o.v[j] = isnan(z) ? (uint8_t)0x7F : f32_to_e4m3(fminf(fmaxf(z, -448.f), 448.f));
        else
          o.v[j] = (uint8_t)rne_clamp_i8(z);
      }
    }
    st_pack<uint8_t, V>(a.q + row * a.cols + (int64_t)v * V, o);
  };

#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int v = tid + i * team;
    if (active && v < nvec) y[i] = norm(v, y[i]);
  }

  if constexpr (MODE == kGroupLanes) {
    // A group is `lanes` consecutive packs: packs of one i are consecutive over the team's
    // threads and the team is whole warps, so a group never leaves its warp.
    const int lanes = a.G / V;
    const int shift = 31 - __clz(lanes);
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int v = tid + i * team;
      const bool have = active && v < nvec;
      const unsigned k = warp_max_key(have ? key_of(y[i]) : 0u, lanes);
      if (have) {
        const float s = scale_of(k);
        if ((v & (lanes - 1)) == 0) put_scale(v >> shift, s);
        emit(v, y[i], s);
      }
    }
    const int rounds = (nvec + team - 1) / team;  // uniform trip count: the shuffles need all lanes
    for (int i = MAXV; i < rounds; ++i) {
      const int v = tid + i * team;
      const bool have = active && v < nvec;
      F f;
      if (have) {
        f = load_h(v);
        store_h(v, f);
        f = norm(v, f);
      }
      const unsigned k = warp_max_key(have ? key_of(f) : 0u, lanes);
      if (have) {
        const float s = scale_of(k);
        if ((v & (lanes - 1)) == 0) put_scale(v >> shift, s);
        emit(v, f, s);
      }
    }
  } else {
    unsigned* gm = gmax + local * groups;
    if constexpr (MODE == kGroupShared) {
      for (int g = tid; g < groups; g += team) gm[g] = 0u;
      __syncthreads();
    }
    unsigned k = 0u;
    auto note = [&](int v, const F& f) {
      if constexpr (MODE == kGroupRow) k = max(k, key_of(f));
      else atomicMax(gm + (int)(((int64_t)v * V) / a.G), key_of(f));  // V divides G
    };
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int v = tid + i * team;
      if (active && v < nvec) note(v, y[i]);
    }
    for (int v = tid + MAXV * team; active && v < nvec; v += team) note(v, norm(v, load_h(v)));
    float s = 0.f;
    if constexpr (MODE == kGroupRow) {
      k = team_reduce(k, team, red_max, [](unsigned p, unsigned q) { return max(p, q); });
      s = scale_of(k);
      if (active && tid == 0) put_scale(0, s);
    } else {
      __syncthreads();
      for (int g = tid; active && g < groups; g += team) {
        const float t = scale_of(gm[g]);
        put_scale(g, t);
        gm[g] = __float_as_uint(t);
      }
      __syncthreads();
    }
    auto scale_at = [&](int v) {
      if constexpr (MODE == kGroupRow) return s;
      else return __uint_as_float(gm[(int)(((int64_t)v * V) / a.G)]);
    };
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int v = tid + i * team;
      if (active && v < nvec) emit(v, y[i], scale_at(v));
    }
    for (int v = tid + MAXV * team; active && v < nvec; v += team) {
      const F f = load_h(v);
      const float sv = scale_at(v);
      const F z = norm(v, f);
      store_h(v, f);
      emit(v, z, sv);
    }
  }
}

template <typename T, int Q, int V, int MAXV, int MODE>
int launch_norm(NormArgs a, cudaStream_t st) {
  const int64_t nvec = a.cols / V;
  int64_t team = ceil_div(ceil_div(nvec, MAXV), 32) * 32;
  if (team > 1024) team = 1024;
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
    const cudaError_t e =
        ensure_smem_attr((const void*)k_norm_quant<T, Q, V, MAXV, MODE>, 200 * 1024);
    if (e != cudaSuccess) return cuda_fail(e, "add_rms_norm_group_quant: shared memory attribute");
  }
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_norm_quant<T, Q, V, MAXV, MODE>, a);
  if (e != cudaSuccess) return cuda_fail(e, "add_rms_norm_group_quant launch");
  return check_launch("add_rms_norm_group_quant");
}

template <typename T, int Q>
int launch_norm_any(const NormArgs& a, cudaStream_t st) {
  constexpr int VV = 16 / sizeof(T);
  const bool vec = a.cols % VV == 0 && a.G % VV == 0 && aligned16(a.x) && aligned16(a.w) &&
                   a.ldx % VV == 0 && aligned_to(a.q, VV) &&
                   (!a.r || (aligned16(a.r) && a.ldr % VV == 0)) &&
                   (!a.h || (aligned16(a.h) && a.ldh % VV == 0));
  if (!vec) {
    if (a.G == a.cols) return launch_norm<T, Q, 1, 8, kGroupRow>(a, st);
    return launch_norm<T, Q, 1, 8, kGroupShared>(a, st);
  }
  const int lanes = a.G / VV;
  if (a.G == a.cols && lanes > 32) return launch_norm<T, Q, VV, 4, kGroupRow>(a, st);
  if (lanes <= 32 && (lanes & (lanes - 1)) == 0)
    return launch_norm<T, Q, VV, 4, kGroupLanes>(a, st);
  if (a.G == a.cols) return launch_norm<T, Q, VV, 4, kGroupRow>(a, st);
  return launch_norm<T, Q, VV, 4, kGroupShared>(a, st);
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
  if (rows < 0 || cols < 0 || cols > INT32_MAX || group_size <= 0 || cols % group_size != 0 ||
      (rows > 1 && (ldx < cols || (residual && ldr < cols) || (residual_out && ldh < cols))))
    return fail(TO_EINVAL, "%s: invalid shape rows=%lld cols=%lld group=%lld strides=(%lld, %lld, "
                "%lld)", op, (long long)rows, (long long)cols, (long long)group_size,
                (long long)ldx, (long long)ldr, (long long)ldh);
  if (q_dtype != TO_E4M3 && q_dtype != TO_I8)
    return fail(TO_EUNSUPPORTED, "%s: codes %s (float8_e4m3fn or int8)", op, dtype_name(q_dtype));
  if (q_dtype == TO_I8 && (ue8m0 || column_major))
    return fail(TO_EINVAL, "%s: ue8m0 / column-major scales are FP8 options", op);
  if (rows == 0 || cols == 0) return TO_OK;
  if (!x || !weight || !q || !scales) return fail(TO_EINVAL, "%s: null pointer", op);
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
  a.ue8m0 = ue8m0;
  a.sl = ScaleLayout{column_major ? rows : 0, column_major ? cols / group_size : 1};
  cudaStream_t st = (cudaStream_t)stream;
  TOB_DISPATCH_FLOAT(dtype, T, {
    return q_dtype == TO_E4M3 ? launch_norm_any<T, kQE4M3>(a, st)
                              : launch_norm_any<T, kQI8>(a, st);
  });
  return TO_OK;
}
