// Epilogue of the products with bias, activation and residual:
//   C[m, n] = T( act( acc[m, n] + bias[n] ) + residual[m, n] )
// acc is the scaled fp32 sum; everything up to the one rounding to T is fp32.
#pragma once

#include "common.cuh"

namespace tob {

// 0 none, 1 relu, 2 silu, 3 gelu (tanh form): the `act` argument of the C entries.
enum EpiAct : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// Both gated forms are x * sigmoid(z): silu with z = x, gelu_tanh with z = 2 sqrt(2/pi)
// (x + 0.044715 x^3), since (1 + tanh(u)) / 2 = sigmoid(2u). In this form nothing cancels for
// negative x.
__device__ __forceinline__ float epi_act_exact(float x, int act) {
  if (act == kActNone) return x;
  if (act == kActRelu) return x < 0.0f ? 0.0f : x;  // NaN stays NaN
  const float z = act == kActSilu ? x : 1.5957691216057308f * fmaf(0.044715f * x * x, x, x);
  return x / (1.0f + expf(-z));
}

// The same for the tensor-core kernels, whose epilogues run once per tile: their time is the
// fetching of their instructions (unrolled over 32 columns with a four-way choice each they took
// 8000 cycles a chunk), so the four activations share two short forms chosen by numbers:
//   plain  x < lo ? lo : x                           (none: lo = -inf, relu: 0)
//   gated  x / (1 + 2^(x (c1 + c2 min(x^2, 1e30))))  (the exponent is -z log2(e))
// with the hardware's exponential and division: a relative error of about 1e-6 where the result is
// not negligible, far below half a step of a 16-bit result. The minimum keeps 0 * inf out of silu.
struct ActForm {
  int gated;
  float lo, c1, c2;
};
inline ActForm act_form(int act) {
  constexpr float kLog2e = 1.4426950408889634f, kGelu = 1.5957691216057308f;
  if (act == kActSilu) return {1, 0.f, -kLog2e, 0.f};
  if (act == kActGelu) return {1, 0.f, -kLog2e * kGelu, -kLog2e * kGelu * 0.044715f};
  return {0, act == kActRelu ? 0.f : -__builtin_inff(), 0.f, 0.f};
}
__device__ __forceinline__ float act_plain(float x, const ActForm& f) {
  return x < f.lo ? f.lo : x;  // NaN stays NaN
}
__device__ __forceinline__ float act_gated(float x, const ActForm& f) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * fmaf(f.c2, fminf(x * x, 1e30f), f.c1)));
  return __fdividef(x, 1.0f + e);
}

// The gated forms for fp32 results, of which that error would be many steps: the accurate
// exponential, and the quotient by Markstein's correction (q + (x - q d) / d from an approximate
// reciprocal of d), which has no branches as the division operator has: with that, the epilogue of
// 8192 x 1024 -> 8192 made 180 us 490. Where the correction is no number (x or d infinite) the
// first quotient stands: inf, 0 or NaN as x / d.
__device__ __forceinline__ float act_gated_f32(float x, int act) {
  const float z = act == kActSilu ? x : 1.5957691216057308f * fmaf(0.044715f * x * x, x, x);
  const float d = 1.0f + expf(-z);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  const float q = x * r, t = fmaf(-q, d, x);
  return t == t ? fmaf(t, r, q) : q;
}

// Launches of these kernels carry the programmatic-dependency attribute always: a kernel's blocks may
// start (barriers, tensor memory, tensor maps) while the previous kernel of the stream drains, and
// every thread that touches global memory first waits for that kernel's completion
// (griddepcontrol.wait), so the order of the stream holds as with plain launches, whatever the
// launch-overlap switch says: the weights' copies wait too, since a B that the caller hands over
// in another layout has just been copied. (Weights read ahead with overlap on saved 0.4 to 0.7 us
// a call: 4096 x 4096, one token, 8.0 against 8.5.) Each block waits before it ends, so completion
// stays transitive along a chain. A block lets the next kernel
// start (griddepcontrol.launch_dependents) only after its own wait: at most two kernels of a stream
// are in flight, so a later kernel that reads its weights early (launch overlap) can meet its
// immediate predecessor alone, never a writer further back. (The later start costs 0.1 to 0.2 us a
// launch: the norm of one token 2.1 us before, 2.2 so.)

// What a product's epilogue reads and writes besides the accumulators. Row strides in elements.
struct LinEpi {
  const float* a_s = nullptr;  // scale of token m in K block kb: a_s[m * a_s_ld + kb]; null: 1
  const float* b_s = nullptr;  // scale of column n: b_s[(n / bn) * b_s_ld + kb]; null: 1
  int64_t a_s_ld = 0, b_s_ld = 0;
  int64_t bn = 1;
  int kb_per_scale = 1;        // 128-byte K slices per scale block (block-scaled products)
  const void* bias = nullptr;  // [N] of `dtype`, or null
  const void* res = nullptr;   // [M, N] of `dtype`, rows ldr apart, or null
  void* c = nullptr;           // [M, N] of `dtype`, rows ldc apart
  int64_t ldr = 0, ldc = 0;
  int dtype = TO_F32;
  int act = kActNone;
  ActForm form = {};           // act_form(act)
};

// The operands of a product: A [M, K] rows lda elements apart, B [N, K] (8-bit) or [K, N] (16-bit)
// rows ldb apart. a_k >= K: columns of A that exist, zero past K (a padded copy); b_in likewise for
// the inner dimension of B.
struct LinOps {
  const void* a;
  const void* b;
  int64_t lda, ldb, a_k, b_in;
  int64_t M, N, K;
};

// Element i of an array of `dtype` (TO_F32 / TO_F16 / TO_BF16) as fp32, and its store. The
// residual may be the output itself (in-place add), so its loads stay ordinary loads.
__device__ __forceinline__ float ld_dtype(const void* p, int64_t i, int dtype) {
  if (dtype == TO_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == TO_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
// The same in two steps, load and conversion, without a branch between loads: a choice of type
// around each load makes the next one wait for it.
__device__ __forceinline__ uint32_t ld_raw(const void* p, int64_t i, bool wide) {
  return wide ? reinterpret_cast<const uint32_t*>(p)[i]
              : (uint32_t)reinterpret_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float raw_to_f32(uint32_t v, int dtype) {
  const float h = __half2float(__ushort_as_half((unsigned short)v));
  return dtype == TO_F16 ? h : __uint_as_float(dtype == TO_BF16 ? v << 16 : v);
}
__device__ __forceinline__ void st_dtype(void* p, int64_t i, int dtype, float v) {
  if (dtype == TO_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == TO_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

}  // namespace tob
