// Shared by the many-token kernels of the products with an epilogue (linear_pair_sm100.cu,
// linear_bs_sm100.cu): tile order, the chunk that leaves through shared memory, tensor maps.
#pragma once

#include <cudaTypedefs.h>

#include <type_traits>

#include "linear_epi.cuh"
#include "sm100.cuh"

namespace tob {
namespace sm100 {

PFN_cuTensorMapEncodeTiled_v12000 get_encode();

namespace {

constexpr int kEpiWarpsT = 8;       // epilogue warps of a CTA, two per TMEM lane quarter
constexpr int kSlab = 32 * 32 * 2;  // one 32 x 32 chunk of 16-bit results

// Bands of M tiles, M fastest: the tiles in flight share a band's A rows and a few B columns.
__device__ __forceinline__ void band_tile(int t, int m_tiles, int n_tiles, int band, int& mt,
                                          int& nt) {
  const int per = band * n_tiles;
  const int b = t / per;
  const int rows = min(band, m_tiles - b * band);
  const int local = t - b * per;
  mt = b * band + local % rows;
  nt = local / rows;
}

__device__ __forceinline__ void epi_barrier() {  // the epilogue warps of this CTA
  asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarpsT * 32) : "memory");
}

// Bias, activation, residual and store of one warp's 32 x 32 chunks. Two slabs of shared memory
// alternate; a chunk's residual is copied into its slab up to two chunks ahead and overwritten there
// by the result, which leaves by a TMA store. One mbarrier per slab, each used once per visit.
// Order per tile: fetch(0), fetch(1); then per chunk acquire, put and, after it, fetch(1) for the
// chunk after next. want() brings the residual of later chunks near (into L2) at the tile's start.
struct ChunkWriter {
  uint8_t* slab0;        // two slabs
  uint64_t* rbar;        // two barriers
  const CUtensorMap* tmC;
  const CUtensorMap* tmR;
  volatile int* abort_flag;
  int* err;
  ActForm form;
  int dtype, lane;
  bool res;
  int cnt = 0;  // chunks visited: slab cnt & 1, residual phase (cnt >> 1) & 1

  __device__ __forceinline__ void want(int col0, int row0) {
    if (!res || lane != 0) return;
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                     reinterpret_cast<uint64_t>(tmR)),
                 "r"(col0), "r"(row0)
                 : "memory");
  }
  // The residual of the ahead-th chunk from now (0 or 1), at (col0, row0).
  __device__ __forceinline__ void fetch(int ahead, int col0, int row0) {
    if (!res || lane != 0) return;
    bulk_wait_read<0>();  // no store still reads the slab
    uint64_t* bar = rbar + ((cnt + ahead) & 1);
    mbar_arrive_expect_tx(bar, kSlab);
    tma_load_2d(slab0 + ((cnt + ahead) & 1) * kSlab, tmR, col0, row0, bar, policy_evict_first());
  }
  // Waits until the current chunk's slab may be written (with the residual in it).
  __device__ __forceinline__ bool acquire() {
    if (res) return mbar_wait_polled(rbar + (cnt & 1), (uint32_t)(cnt >> 1) & 1u, abort_flag, err);
    if (lane == 0) bulk_wait_read<1>();  // the store before last has read this slab
    __syncwarp();
    return true;
  }
  // v: this lane's row of the chunk, scaled; bias: of its 32 columns, in shared memory. Straight
  // code per step, one uniform choice around each (see ActForm). F32: the result is fp32.
  template <bool F32 = false>
  __device__ __forceinline__ void finish_acts(float* v, const float* bias, int act = kActNone) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 b = *reinterpret_cast<const float4*>(bias + i);
      v[i] += b.x;
      v[i + 1] += b.y;
      v[i + 2] += b.z;
      v[i + 3] += b.w;
    }
    if (F32 && act == kActSilu) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_gated_f32(v[i], kActSilu);
    } else if (F32 && act == kActGelu) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_gated_f32(v[i], kActGelu);
    } else if (!F32 && form.gated) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_gated(v[i], form);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_plain(v[i], form);
    }
  }
  // The chunk where the output or the residual is no TMA tensor (16-byte rows, 16-bit values): it
  // turns in both slabs, so that a lane is a column and rows are read and written whole.
  template <typename T>
  __device__ __forceinline__ void put_rows(float* v, const float* bias, int col0, int row0,
                                           const LinEpi& ep, int M, int N, bool store) {
    const int n = col0 + lane, rows = min(32, M - row0);
    const bool mine = n < N && store, whole = rows == 32;
    // The residual's column first: its latency passes under the activation.
    T f[16];
    const T* rp = reinterpret_cast<const T*>(ep.res) + (int64_t)row0 * ep.ldr + n;
    auto fetch_rows = [&]() {
#pragma unroll
      for (int r = 0; r < 16; ++r, rp += ep.ldr) f[r] = *rp;
    };
    if (ep.res != nullptr && mine && whole) fetch_rows();
    finish_acts<std::is_same<T, float>::value>(v, bias, ep.act);
    float* turn = reinterpret_cast<float*>(slab0);
    __syncwarp();  // the previous chunk has been read
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<float4*>(turn + lane * 32 + ((c ^ (lane & 7)) << 2)) =
          make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    __syncwarp();
    if (!mine) return;
    auto at = [&](int r) { return turn[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)]; };
    T* cp = reinterpret_cast<T*>(ep.c) + (int64_t)row0 * ep.ldc + n;
    if (!whole) {  // the last rows
#pragma unroll 1
      for (int r = 0; r < rows; ++r, cp += ep.ldc, rp += ep.ldr)
        *cp = from_f32<T>(at(r) + (ep.res != nullptr ? to_f32<T>(*rp) : 0.f));
    } else if (ep.res != nullptr) {
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += 16) {
        if (r0 > 0) fetch_rows();
#pragma unroll
        for (int r = 0; r < 16; ++r, cp += ep.ldc) *cp = from_f32<T>(at(r0 + r) + to_f32<T>(f[r]));
      }
    } else {
#pragma unroll 16
      for (int r = 0; r < 32; ++r, cp += ep.ldc) *cp = from_f32<T>(at(r));
    }
  }
  __device__ __forceinline__ void put_plain(float* v, const float* bias, int col0, int row0,
                                            const LinEpi& ep, int M, int N, bool store) {
    if (dtype == TO_BF16) put_rows<__nv_bfloat16>(v, bias, col0, row0, ep, M, N, store);
    else if (dtype == TO_F16) put_rows<__half>(v, bias, col0, row0, ep, M, N, store);
    else put_rows<float>(v, bias, col0, row0, ep, M, N, store);
  }
  __device__ __forceinline__ void put(float* v, const float* bias, int col0, int row0, bool store) {
    finish_acts(v, bias);
    uint8_t* slab = slab0 + (cnt & 1) * kSlab;
    // 16-byte pieces of 8 columns, swizzled as the TMA box is
    auto at = [&](int c) {
      return reinterpret_cast<uint4*>(slab + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
    };
    if (dtype == TO_BF16) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (res) w = *at(c);
        uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const __nv_bfloat162 o =
              __floats2bfloat162_rn(v[c * 8 + 2 * p] + __uint_as_float(wp[p] << 16),
                                    v[c * 8 + 2 * p + 1] + __uint_as_float(wp[p] & 0xFFFF0000u));
          wp[p] = *reinterpret_cast<const uint32_t*>(&o);
        }
        *at(c) = w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (res) w = *at(c);
        uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&wp[p]));
          const __half2 o = __floats2half2_rn(v[c * 8 + 2 * p] + f.x, v[c * 8 + 2 * p + 1] + f.y);
          wp[p] = *reinterpret_cast<const uint32_t*>(&o);
        }
        *at(c) = w;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && store) {
      tma_store_2d(tmC, col0, row0, slab);
      bulk_commit();
    }
    ++cnt;
  }
};

// Tensor map with the given box and swizzle; strides in bytes.
inline int tiled_map(CUtensorMap* out, CUtensorMapDataType dt, const void* p, int rank,
              const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
              CUtensorMapSwizzle sw) {
  auto encode = get_encode();
  if (!encode) return fail(TO_ECUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(out, dt, (cuuint32_t)rank, const_cast<void*>(p), dims, strides, box,
                            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TO_OK
                           : fail(TO_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

// K-major operand: boxes of box_rows rows x `slices` 128-byte slices (3-D view, K whole slices), or
// of one slice (2-D, slices = 1).
inline int kmajor_map(CUtensorMap* out, const void* p, int64_t rows, int64_t K, int64_t pitch,
                      int elem, int box_rows, int slices) {
  const auto dt = elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  const cuuint32_t bk = (cuuint32_t)(128 / elem);
  if (slices > 1) {
    const cuuint64_t dims[3] = {bk, (cuuint64_t)rows, (cuuint64_t)(K / bk)};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch, 128};
    const cuuint32_t box[3] = {bk, (cuuint32_t)box_rows, (cuuint32_t)slices};
    return tiled_map(out, dt, p, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {bk, (cuuint32_t)box_rows};
  return tiled_map(out, dt, p, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The map of a 16-bit [rows, cols] output or residual: 32 x 32 boxes, 64-byte swizzle.
inline int chunk_map(CUtensorMap* out, const void* p, int64_t rows, int64_t cols, int64_t ld) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * 2)};
  const cuuint32_t box[2] = {32, 32};
  return tiled_map(out, CU_TENSOR_MAP_DATA_TYPE_UINT16, p, 2, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_64B);
}

// Whether output or residual need the plain path: fp32, rows that TMA cannot address, or rows of C
// that end inside 16 bytes: a TMA store writes those 16 bytes whole, the next columns of a wider
// row with them.
inline bool aligned_rows(const void* p, int64_t pitch);
inline bool plain_output(const LinEpi& ep, int64_t N) {
  return ep.dtype == TO_F32 || N % 8 != 0 || !aligned_rows(ep.c, ep.ldc * 2) ||
         (ep.res != nullptr && !aligned_rows(ep.res, ep.ldr * 2));
}
inline bool aligned_rows(const void* p, int64_t pitch) {
  return ((reinterpret_cast<uint64_t>(p) | (uint64_t)pitch) & 15u) == 0;
}

}  // namespace
}  // namespace sm100
}  // namespace tob
