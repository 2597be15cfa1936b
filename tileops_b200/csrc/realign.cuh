// Sixteen bytes from any address: two aligned 16-byte loads, shifted together in registers.
#pragma once

#include "common.cuh"

namespace tob {

// Bytes [p, p + valid) of an operand whose memory is [lo, hi), valid <= 16; the rest reads as zero.
// issue() starts the loads, finish() shifts: several can be in flight. Nothing outside [lo, hi) is
// touched: an aligned word that reaches outside it (the operand's first and last bytes only) is
// read byte by byte.
struct Unaligned16 {
  uint4 a, b;
  const uint8_t* p;
  int valid;
  bool ragged;

  __device__ __forceinline__ void issue(const uint8_t* at, int n, const uint8_t* lo,
                                        const uint8_t* hi) {
    p = at;
    valid = n;
    const int o = (int)(reinterpret_cast<uintptr_t>(at) & 15u);
    const uint8_t* base = at - o;
    const bool need0 = n > 0, need1 = n > 0 && o + n > 16;
    const bool in0 = base >= lo && base + 16 <= hi, in1 = base + 32 <= hi;
    a = make_uint4(0u, 0u, 0u, 0u);
    b = make_uint4(0u, 0u, 0u, 0u);
    if (need0 && in0) a = __ldg(reinterpret_cast<const uint4*>(base));
    if (need1 && in1) b = __ldg(reinterpret_cast<const uint4*>(base) + 1);
    ragged = (need0 && !in0) || (need1 && !in1);
  }
  __device__ __forceinline__ uint4 finish() const {
    uint32_t w[4];
    if (ragged) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = 0u;
#pragma unroll 1
      for (int i = 0; i < valid; ++i) {
        const uint32_t v = (uint32_t)__ldg(p + i) << (8 * (i & 3));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] |= i / 4 == j ? v : 0u;
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const int o = (int)(reinterpret_cast<uintptr_t>(p) & 15u);
    uint32_t s[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
    uint32_t last = b.w;
    if (o & 8) {
#pragma unroll
      for (int i = 0; i < 5; ++i) s[i] = s[i + 2];
      s[5] = last;
    }
    if (o & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) s[i] = s[i + 1];
    }
    const int sh = 8 * (o & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(s[j], s[j + 1], sh);
    if (valid < 16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int nb = valid - 4 * j;
        w[j] = nb >= 4 ? w[j] : nb <= 0 ? 0u : w[j] & ((1u << (8 * nb)) - 1u);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

}  // namespace tob
