// Products with bias, activation and residual in their epilogue, many tokens: 256 x BN output tiles
// on CTA pairs (tcgen05 cta_group::2), persistent over the tiles.
//
//   A tokens [M, K] (K-major); B weights int8 / e4m3 [N, K] (K-major) or fp16 / bf16 [K, N]
//   (MN-major, 64-column strips)
//
// A pair's MMA is 256 x BN: each CTA streams its 128 rows of A and BN / 2 columns of B, two 128-byte
// K slices per stage and copy, and holds 128 x BN sums in its own tensor memory, in two buffers, so
// one tile's epilogue runs under the next one's main loop. With BN = 256 an SM reads 32 KB per
// 128 x 256 x 128-byte step, which L2 delivers at the tensor cores' rate (a 128 x 128 tile per CTA
// needs twice that and was bound by it).
//
// The residual arrives by TMA in the slab of shared memory its chunk's result leaves from, two
// chunks ahead of its use; results leave by TMA stores. (Turned by generic stores and written in
// 16-byte pieces instead, 4096 x 512 -> 4096 FP8 with residual took 36 us instead of 28.)
//
// Bound by the tensor cores under the power cap: 2048 x 8192 x 28672 bf16 with bias and gelu 635 to
// 820 us on different boxes and in longer or shorter runs, 1.17 to 1.51 PFLOP/s (a plain library
// product: 1.40 sustained); FP8 8192^3 with bias, gelu and residual 370 to 476 us, 2.3 to 3.0. Between 65 and some 1000 tokens, by the operands through L2: 512 tokens of FP8
// 7168 -> 2048 15 us, 128 tokens of bf16 1024 -> 28672 18 us.
//
// Roles: warp 0 copies of A, warp 1 MMA issue (leader CTA) and TMEM, warps 2..9 epilogue (two per
// TMEM lane quarter), warp 10 copies of B. Every wait is bounded (kWaitLimitNs).
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "linear_tile.cuh"

namespace tob {
namespace sm100 {
namespace {

constexpr int kKC = 2;          // 128-byte K slices per stage
constexpr int kBWarpP = 2 + kEpiWarpsT;
constexpr int kThreadsP = 32 * (kBWarpP + 1);

template <Kind KD, int BN>
struct PairCfg2 {
  static constexpr int kElem = KindTraits<KD>::kElemBytes;
  static constexpr bool kMn = kElem == 2;
  static constexpr int kBK = 128 / kElem;
  static constexpr int kACh = 128 * 128;          // one slice of this CTA's A rows
  static constexpr int kBCh = (BN / 2) * 128;     // one slice of this CTA's B columns
  static constexpr int kABytes = kKC * kACh, kBBytes = kKC * kBCh;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kFixed = kEpiWarpsT * 2 * kSlab + BN * 8 + 512;  // slabs, columns, barriers
  static constexpr int kStages = std::min(8, (232448 - kFixed) / kStageBytes);
  static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kFixed;
  static constexpr int kTmemCols = 2 * BN <= 128 ? 128 : 2 * BN <= 256 ? 256 : 512;
  static_assert(BN % 32 == 0 && BN >= 64 && BN <= 256, "tile width");
  static_assert(!kMn || BN % 128 == 0, "MN-major: whole 64-column strips per CTA");
  static_assert(kStages >= 3, "ring");
  static_assert((2 * kStages + 5 + 2 * kEpiWarpsT) * 8 + 16 <= 512, "barrier area");
};

struct PairArgs {
  int M, N, K;
  int a3d, b3d;    // operand through a 3-D map: {128 B, rows, slices} of whole slices, or (MN-major
                   // B) {64 columns, K rows, strips} of whole strips
  int plain_out;   // output or residual is no TMA tensor
  int band;        // M tiles per band of the tile order
  int small_m;     // one row of tiles: A stays in L2, B streams
  LinEpi ep;
};

template <Kind KD, int BN>
__global__ void __launch_bounds__(kThreadsP, 1)
    k_linear_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                  const __grid_constant__ PairArgs g, int* err) {
  using C = PairCfg2<KD, BN>;
  using Tr = KindTraits<KD>;
  constexpr int ST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sA = smem_raw;
  uint8_t* sB = smem_raw + (size_t)ST * C::kABytes;
  uint8_t* slabs = smem_raw + (size_t)ST * C::kStageBytes;
  float* scale = reinterpret_cast<float*>(slabs + kEpiWarpsT * 2 * kSlab);  // of the tile's columns
  float* bias = scale + BN;
  uint64_t* full = reinterpret_cast<uint64_t*>(bias + BN);
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;   // [2] sums of a tile complete
  uint64_t* tempty = tfull + 2;   // [2] read by the epilogues of both CTAs (leader's barrier)
  uint64_t* drain = tempty + 2;
  uint64_t* rbar = drain + 1;     // [8][2] a chunk's residual has landed
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(rbar + 2 * kEpiWarpsT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x & 1);
  const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
  const int m_tiles = (g.M + 255) / 256, n_tiles = (g.N + BN - 1) / BN;
  const int tiles = m_tiles * n_tiles;
  const int slices = (g.K + C::kBK - 1) / C::kBK;
  const int steps = (slices + kKC - 1) / kKC;
  const bool misaligned = (smem_u32(smem_raw) & 1023u) != 0;
  const LinEpi& ep = g.ep;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full + s, 1);   // the leader's expectation; both CTAs' bytes complete it
      mbar_init(empty + s, 1);  // the leader's commit, to both CTAs
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull + b, 1);
      mbar_init(tempty + b, 2 * kEpiWarpsT);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 2 * kEpiWarpsT; ++i) mbar_init(rbar + i, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmC);
    if (ep.res != nullptr && !g.plain_out) prefetch_tmap(&tmR);
    if (misaligned && err) atomicExch(err, (int)kErrSmemAlign);
  }
  cluster_arrive_relaxed();
  if (warp == 1) tmem_alloc_pair<C::kTmemCols>(tmem_holder);
  cluster_wait_acquire();  // both CTAs' barriers exist
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (misaligned) {
    // nothing to do; fall through to the teardown
  } else if (warp == 0 || warp == kBWarpP) {
    // ------------------------------------------------------------ copies of A / of B
    if (lane == 0) {
      const bool is_a = warp == 0;
      const uint64_t pol = !g.small_m ? policy_evict_normal()
                           : is_a     ? policy_evict_last()
                                      : policy_evict_first();
      const uint32_t lead_full = mapa_shared(smem_u32(full), 0);
      grid_dependency_wait();
      if (is_a) grid_dependents_launch();  // the next kernel may set itself up
      uint32_t issued_mask = 0, issued_phase = 0;
      bool ok = true;
      int it = 0;  // stages issued
      for (int t = pair; ok && t < tiles; t += pairs) {
        int mt, nt;
        band_tile(t, m_tiles, n_tiles, g.band, mt, nt);
        const int arow = mt * 256 + rank * 128;
        const int bcol = nt * BN + rank * (BN / 2);
        for (int st = 0; st < steps; ++st, ++it) {
          const int s = it % ST;
          const uint32_t ph = (uint32_t)(it / ST) & 1u;
          if (it >= ST && !mbar_wait_polled(empty + s, ph ^ 1, abort_flag, err)) { ok = false; break; }
          const uint32_t bar = lead_full + (uint32_t)s * 8u;
          const int sl = st * kKC, k = sl * C::kBK;
          if (is_a) {
            if (rank == 0) {
              mbar_arrive_expect_tx(full + s, 2 * C::kStageBytes);
              issued_mask |= 1u << s;
              issued_phase = (issued_phase & ~(1u << s)) | (ph << s);
            }
            uint8_t* dst = sA + (size_t)s * C::kABytes;
            if (g.a3d) {
              tma_load_3d_pair(dst, &tmA, 0, arow, sl, bar, pol);
            } else {
#pragma unroll
              for (int c = 0; c < kKC; ++c)
                tma_load_2d_pair(dst + c * C::kACh, &tmA, k + c * C::kBK, arow, bar, pol);
            }
          } else {
            uint8_t* dst = sB + (size_t)s * C::kBBytes;
            if constexpr (C::kMn) {
              // strips of 128 K rows x 64 columns, 16 KB each
              if (g.b3d) {
                tma_load_3d_pair(dst, &tmB, 0, k, bcol / 64, bar, pol);
              } else {
#pragma unroll
                for (int c = 0; c < BN / 128; ++c)
                  tma_load_2d_pair(dst + c * 16384, &tmB, bcol + 64 * c, k, bar, pol);
              }
            } else if (g.b3d) {
              tma_load_3d_pair(dst, &tmB, 0, bcol, sl, bar, pol);
            } else {
#pragma unroll
              for (int c = 0; c < kKC; ++c)
                tma_load_2d_pair(dst + c * C::kBCh, &tmB, k + c * C::kBK, bcol, bar, pol);
            }
          }
        }
      }
      if (!ok && rank == 0 && is_a) {
        // Unwinding: the leader's full barriers count both CTAs' bytes; let them land. One
        // deadline for all stages: a stage whose other copies were never issued cannot complete.
        const uint64_t tw = globaltimer_ns();
        for (int i = 0; i < ST; ++i)
          if (issued_mask & (1u << i))
            while (!mbar_try_wait(full + i, (issued_phase >> i) & 1u) &&
                   globaltimer_ns() - tw < kWaitLimitNs) {
            }
      } else if (!ok) {
        // Unwinding: these copies cannot be observed here; they land within microseconds.
        const uint64_t tw = globaltimer_ns();
        while (globaltimer_ns() - tw < 50000ull) {
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    // The whole warp walks the loop and one lane issues: addresses and descriptors then stay in
    // uniform registers.
    if (rank == 0) {
      constexpr uint32_t idesc =
          make_idesc_major(Tr::kDFmt, Tr::kAFmt, Tr::kBFmt, 256, BN, 0, C::kMn ? 1 : 0);
      const uint64_t adesc = smem_desc_kmajor_sw128(smem_u32(sA));
      const uint64_t bdesc = C::kMn ? smem_desc_mnmajor_sw128(smem_u32(sB), 16384, 1024)
                                    : smem_desc_kmajor_sw128(smem_u32(sB));
      const bool issue = elect_one();
      grid_dependency_wait();  // the waits below count this kernel's time, not the previous one's
      bool ok = true;
      int fill = 0, s = 0;  // accumulator fills started; stage
      uint32_t ph = 0;
      for (int t = pair; ok && t < tiles; t += pairs) {
        if (fill >= 2)
          ok = mbar_wait_warp(tempty + (fill & 1), ((uint32_t)(fill >> 1) & 1u) ^ 1, abort_flag,
                              err);
        if (!ok) break;
        const uint32_t d = tmem + (uint32_t)((fill & 1) * BN);
        for (int st = 0; st < steps; ++st) {
          ok = mbar_wait_warp(full + s, ph, abort_flag, err);
          if (!ok) break;
          tc_fence_after();
          if (issue) {
            const uint64_t ad = adesc + (uint64_t)(s * (C::kABytes >> 4));
            const uint64_t bd = bdesc + (uint64_t)(s * (C::kBBytes >> 4));
#pragma unroll
            for (int i = 0; i < 4 * kKC; ++i) {
              // 32 bytes of K: within a slice 32 B on, MN-major 16 K rows (2 KB) on
              const int ao = (i / 4) * C::kACh + 32 * (i % 4);
              const int bo = C::kMn ? (i / 4) * 8192 + 2048 * (i % 4)
                                    : (i / 4) * C::kBCh + 32 * (i % 4);
              umma_pair<KD>(d, ad + (ao >> 4), bd + (bo >> 4), idesc, (st | i) != 0);
            }
            umma_commit_pair_mc(empty + s, 0x3);
            if (st == steps - 1) umma_commit_pair_mc(tfull + (fill & 1), 0x3);
          }
          __syncwarp();
          if (++s == ST) { s = 0; ph ^= 1; }
        }
        ++fill;
      }
      if (!ok && issue) {
        // Unwinding: wait (bounded) until the MMAs already issued have finished.
        umma_commit_pair(drain);
        const uint64_t tw = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - tw < kWaitLimitNs) {
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;            // TMEM lane quarter
    const int eg = (warp - 2) >> 2;    // which half of the tile's chunks
    const int ew = warp - 2;
    constexpr int kChunks = BN / 32;
    constexpr int kMine = (kChunks + 1) / 2;
    const uint32_t lead_tempty = mapa_shared(smem_u32(tempty), 0);
    ChunkWriter wr{slabs + ew * 2 * kSlab, rbar + 2 * ew, &tmC, &tmR, abort_flag, err,
                   ep.form, ep.dtype, lane, ep.res != nullptr && !g.plain_out};
    grid_dependency_wait();
    int fill = 0;  // accumulator fills read
    bool ok = true;
    auto chunk_col = [&](int j) { return (2 * j + eg) * 32; };  // this warp's j-th chunk
    // Scale and bias of this thread's column of a tile, read one tile ahead.
    static_assert(BN <= 32 * kEpiWarpsT, "a thread per column");
    const int col = (int)threadIdx.x - 64;
    float scale_next = 1.f, bias_next = 0.f;
    auto read_cols = [&](int t) {
      if (t >= tiles || col >= BN) return;
      int mt, nt;
      band_tile(t, m_tiles, n_tiles, g.band, mt, nt);
      const int n = min(nt * BN + col, g.N - 1);
      if (ep.b_s != nullptr) scale_next = __ldg(ep.b_s + (int64_t)(n / ep.bn) * ep.b_s_ld);
      if (ep.bias != nullptr) bias_next = ld_dtype(ep.bias, n, ep.dtype);
    };
    read_cols(pair);
    for (int t = pair; t < tiles; t += pairs) {
      int mt, nt;
      band_tile(t, m_tiles, n_tiles, g.band, mt, nt);
      const int n0 = nt * BN;
      const int row0 = mt * 256 + rank * 128 + q * 32;
      const int row = min(row0 + lane, g.M - 1);
      const bool rows_in = row0 < g.M;
      // Chunks of this tile that hold output columns.
      int mine = 0;
      while (mine < kMine && chunk_col(mine) < BN && n0 + chunk_col(mine) < g.N) ++mine;
      if (!rows_in) mine = 0;
      // Scale and bias of the tile's columns.
      epi_barrier();  // every warp is done with the previous tile's
      if (col < BN) {
        scale[col] = scale_next;
        bias[col] = bias_next;
      }
      epi_barrier();
      read_cols(t + pairs);
      // After a failed wait a warp still walks the tiles: the others count on it at the barriers.
      if (!ok) continue;
      if (mine > 0) wr.fetch(0, n0 + chunk_col(0), row0);
      if (mine > 1) wr.fetch(1, n0 + chunk_col(1), row0);
      for (int j = 2; j < mine; ++j) wr.want(n0 + chunk_col(j), row0);
      const float sa = ep.a_s != nullptr ? __ldg(ep.a_s + (int64_t)row * ep.a_s_ld) : 1.f;
      const int b = fill & 1;
      if (!mbar_wait_polled(tfull + b, (uint32_t)(fill >> 1) & 1u, abort_flag, err)) {
        ok = false;
        continue;
      }
      tc_fence_after();
#pragma unroll 1
      for (int j = 0; j < mine; ++j) {
        const int c0 = chunk_col(j);
        uint32_t r[32];
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN + c0);
        tmem_ld16(taddr, r);
        tmem_ld16(taddr + 16, r + 16);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4 sb = make_float4(1.f, 1.f, 1.f, 1.f);
          if (!C::kMn) sb = *reinterpret_cast<const float4*>(scale + c0 + i);
          const float sbv[4] = {sb.x, sb.y, sb.z, sb.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float a = KD == Kind::I8 ? (float)(int32_t)r[i + u] : __uint_as_float(r[i + u]);
            v[i + u] = C::kMn ? a : a * (sa * sbv[u]);
          }
        }
        if (g.plain_out) {
          wr.put_plain(v, bias + c0, n0 + c0, row0, ep, g.M, g.N, ok);
          continue;
        }
        if (!wr.acquire()) ok = false;
        wr.put(v, bias + c0, n0 + c0, row0, ok);
        if (j + 2 < mine) wr.fetch(1, n0 + chunk_col(j + 2), row0);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(lead_tempty + (uint32_t)b * 8u);
      ++fill;
    }
    if (lane == 0) bulk_wait_read<0>();  // stores have read their slabs
    if (!ok && lane == 0) {
      // Unwinding: a residual copy in flight lands within microseconds.
      const uint64_t tw = globaltimer_ns();
      while (globaltimer_ns() - tw < 50000ull) {
      }
    }
  }

  grid_dependency_wait();
  tc_fence_before();
  cluster_sync_all();  // both epilogues are done with TMEM; no signal to a peer is pending
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair<C::kTmemCols>(tmem);
  }
}

template <Kind KD, int BN>
int launch_pair(const LinOps& o, bool plain_out, const LinEpi& ep, cudaStream_t st) {
  using C = PairCfg2<KD, BN>;
  auto kern = k_linear_pair<KD, BN>;
  const cudaError_t ae = ensure_smem_attr((const void*)kern, (int)C::kSmem);
  if (ae != cudaSuccess) return cuda_fail(ae, "linear epilogue (pairs): shared memory attribute");
  const int64_t M = o.M, N = o.N, K = o.K;
  PairArgs g;
  memset((void*)&g, 0, sizeof(g));
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.a3d = (o.a_k * C::kElem) % 128 == 0;
  g.b3d = (o.b_in * C::kElem) % 128 == 0;
  g.plain_out = plain_out;
  // Bands whose A rows stay within 32 MB of L2.
  g.band = (int64_t)16 * 256 * K * C::kElem <= ((int64_t)32 << 20) ? 16 : 8;
  g.small_m = M <= 256;
  g.ep = ep;
  CUtensorMap ta, tb, tc, tr;
  memset(&tc, 0, sizeof(tc));
  memset(&tr, 0, sizeof(tr));
  int rc = kmajor_map(&ta, o.a, M, o.a_k, o.lda * C::kElem, C::kElem, 128, g.a3d ? kKC : 1);
  if (rc) return rc;
  if (!C::kMn) {
    rc = kmajor_map(&tb, o.b, N, o.b_in, o.ldb, C::kElem, BN / 2, g.b3d ? kKC : 1);
  } else if (g.b3d) {
    const cuuint64_t dims[3] = {64, (cuuint64_t)K, (cuuint64_t)(o.b_in / 64)};
    const cuuint64_t strides[2] = {(cuuint64_t)(o.ldb * 2), 128};
    const cuuint32_t box[3] = {64, 64 * kKC, BN / 128};
    rc = tiled_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT16, o.b, 3, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    const cuuint64_t dims[2] = {(cuuint64_t)o.b_in, (cuuint64_t)K};
    const cuuint64_t strides[1] = {(cuuint64_t)(o.ldb * 2)};
    const cuuint32_t box[2] = {64, 64 * kKC};
    rc = tiled_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT16, o.b, 2, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (!rc && !plain_out) rc = chunk_map(&tc, ep.c, M, N, ep.ldc);
  if (!rc && !plain_out && ep.res != nullptr) rc = chunk_map(&tr, ep.res, M, N, ep.ldr);
  if (rc) return rc;
  const int64_t tiles = ceil_div(M, 256) * ceil_div(N, BN);
  if (tiles > INT32_MAX) return fail(TO_EUNSUPPORTED, "linear epilogue: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, sm_count() / 2)), 1, 1);
  cfg.blockDim = dim3(kThreadsP, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, tr, g, device_error_ptr());
  if (e != cudaSuccess) return cuda_fail(e, "linear epilogue (pairs) launch");
  return check_launch("linear epilogue (pairs)");
}

}  // namespace

// The tile width for a product, 0 where pairs do not pay (few tokens, or too few tiles to fill the
// SMs without splitting K). Operands have to be of 16-byte aligned rows.
static int pair_width(int kind, int64_t M, int64_t N) {
  const int e = kind == TO_F16 || kind == TO_BF16 ? 2 : 1;
  // Up to 64 tokens the weights-as-rows tiles waste less (64 tokens, 8192 -> 28672 bf16: 78.7 us
  // there, 94.4 here); above, the pairs win although half their rows may be empty (80 tokens: 119 and
  // 96; 1024 -> 28672: 39.2 and 18.1; FP8, 8192 -> 14336: 39.1 and 30.4).
  if (M <= 64) return 0;
  const int64_t pairs = sm_count() / 2;
  // Tile width: the one whose rounds of tiles cost least; a tile's time is its width plus a fixed
  // part worth about 32 columns.
  const int64_t mt = ceil_div(M, 256);
  int best = 0;
  int64_t best_cost = 0;
  const int widths[5] = {256, 192, 160, 128, 64};
  for (int w : widths) {
    if (e == 2 && w % 128 != 0) continue;
    const int64_t cost = ceil_div(mt * ceil_div(N, w), pairs) * (w + 32);
    if (best == 0 || cost < best_cost) {
      best = w;
      best_cost = cost;
    }
  }
  return mt * ceil_div(N, best) * 2 < pairs ? 0 : best;
}

// Runs the product on CTA pairs, or returns TO_EUNSUPPORTED (nothing launched, nothing recorded)
// where the tiles do not apply.
int linear_pair_launch(int kind, const LinOps& o, const LinEpi& ep, cudaStream_t st) {
  const int e = kind == TO_F16 || kind == TO_BF16 ? 2 : 1;
  const int best = pair_width(kind, o.M, o.N);
  if (best == 0 || !aligned_rows(o.a, o.lda * e) || !aligned_rows(o.b, o.ldb * e))
    return TO_EUNSUPPORTED;
  const bool plain = plain_output(ep, o.N);
  if (kind == TO_F16)
    return best == 256 ? launch_pair<Kind::F16, 256>(o, plain, ep, st)
                       : launch_pair<Kind::F16, 128>(o, plain, ep, st);
  if (kind == TO_BF16)
    return best == 256 ? launch_pair<Kind::BF16, 256>(o, plain, ep, st)
                       : launch_pair<Kind::BF16, 128>(o, plain, ep, st);
  auto run = [&](auto kd) {
    constexpr Kind KD = decltype(kd)::value;
    switch (best) {
      case 256: return launch_pair<KD, 256>(o, plain, ep, st);
      case 192: return launch_pair<KD, 192>(o, plain, ep, st);
      case 160: return launch_pair<KD, 160>(o, plain, ep, st);
      case 128: return launch_pair<KD, 128>(o, plain, ep, st);
      default: return launch_pair<KD, 64>(o, plain, ep, st);
    }
  };
  return kind == TO_I8 ? run(std::integral_constant<Kind, Kind::I8>{})
                       : run(std::integral_constant<Kind, Kind::E4M3>{});
}

}  // namespace sm100
}  // namespace tob
