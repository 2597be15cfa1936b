// Products with bias, activation and residual in their epilogue, many tokens: 256 x BN output tiles
// on CTA pairs (tcgen05 cta_group::2), persistent over the tiles, 16-bit output.
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
// Block scales (BS): the products of one 128-byte K slice are one scale block. The MMA alternates
// the two buffers per slice and the epilogue threads fold each into 128 fp32 running sums in
// registers, run = fma(P, a_s b_s, run), while the tensor core fills the other.
//
// The residual arrives by TMA in the slab of shared memory its chunk's result leaves from, one
// chunk ahead of its use; results leave by TMA stores.
//
// Roles: warp 0 copies of A, warp 1 MMA issue (leader CTA) and TMEM, warps 2..9 epilogue (two per
// TMEM lane quarter), warp 10 copies of B. Every wait is bounded (kWaitLimitNs).
#include <cudaTypedefs.h>

#include <string.h>

#include <algorithm>

#include "linear_epi.cuh"
#include "sm100.cuh"

namespace tob {
namespace sm100 {

PFN_cuTensorMapEncodeTiled_v12000 get_encode();

namespace {

constexpr int kKC = 2;          // 128-byte K slices per stage
constexpr int kEpiWarpsP = 8;
constexpr int kBWarpP = 2 + kEpiWarpsP;
constexpr int kThreadsP = 32 * (kBWarpP + 1);
constexpr int kSlab = 32 * 32 * 2;  // one 32 x 32 chunk of 16-bit results

template <Kind KD, int BN, bool BS>
struct PairCfg2 {
  static constexpr int kElem = KindTraits<KD>::kElemBytes;
  static constexpr bool kMn = kElem == 2;
  static constexpr int kBK = 128 / kElem;
  static constexpr int kACh = 128 * 128;          // one slice of this CTA's A rows
  static constexpr int kBCh = (BN / 2) * 128;     // one slice of this CTA's B columns
  static constexpr int kABytes = kKC * kACh, kBBytes = kKC * kBCh;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kFixed = kEpiWarpsP * 2 * kSlab + BN * 8 + 512;  // slabs, columns, barriers
  static constexpr int kStages = std::min(8, (232448 - kFixed) / kStageBytes);
  static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kFixed;
  static constexpr int kTmemCols = 2 * BN <= 128 ? 128 : 2 * BN <= 256 ? 256 : 512;
  static_assert(BN % 32 == 0 && BN >= 64 && BN <= 256, "tile width");
  static_assert(!kMn || BN % 128 == 0, "MN-major: whole 64-column strips per CTA");
  static_assert(!BS || BN == 256, "block scales: 64 KB of sums per CTA");
  static_assert(kStages >= 3, "ring");
  static_assert((2 * kStages + 5 + 2 * kEpiWarpsP) * 8 + 16 <= 512, "barrier area");
};

struct PairArgs {
  int M, N, K;
  int slices3d;    // K-major operands through {128 B, rows, slices} maps (K is whole slices)
  int strips3d;    // MN-major B through the strip map (N % 64 == 0)
  int band;        // M tiles per band of the tile order
  int small_m;     // one row of tiles: A stays in L2, B streams
  LinEpi ep;
};

__device__ __forceinline__ void pair_tile(int t, int m_tiles, int n_tiles, int band, int& mt,
                                          int& nt) {
  // Bands of M tiles, M fastest: the tiles in flight share a band's A rows and a few B columns.
  const int per = band * n_tiles;
  const int b = t / per;
  const int rows = min(band, m_tiles - b * band);
  const int local = t - b * per;
  mt = b * band + local % rows;
  nt = local / rows;
}

__device__ __forceinline__ void epi_barrier() {  // the epilogue warps of this CTA
  asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarpsP * 32) : "memory");
}

template <Kind KD, int BN, bool BS>
__global__ void __launch_bounds__(kThreadsP, 1)
    k_linear_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                  const __grid_constant__ PairArgs g, int* err) {
  using C = PairCfg2<KD, BN, BS>;
  using Tr = KindTraits<KD>;
  constexpr int ST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sA = smem_raw;
  uint8_t* sB = smem_raw + (size_t)ST * C::kABytes;
  uint8_t* slabs = smem_raw + (size_t)ST * C::kStageBytes;
  float2* cols = reinterpret_cast<float2*>(slabs + kEpiWarpsP * 2 * kSlab);  // {scale, bias}
  uint64_t* full = reinterpret_cast<uint64_t*>(cols + BN);
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;   // [2] sums of a tile (BS: of a slice) complete
  uint64_t* tempty = tfull + 2;   // [2] read by the epilogues of both CTAs (leader's barrier)
  uint64_t* drain = tempty + 2;
  uint64_t* rbar = drain + 1;     // [8][2] a chunk's residual has landed
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(rbar + 2 * kEpiWarpsP);
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
      mbar_init(tempty + b, 2 * kEpiWarpsP);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 2 * kEpiWarpsP; ++i) mbar_init(rbar + i, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmC);
    if (ep.res != nullptr) prefetch_tmap(&tmR);
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
      if (is_a) grid_dependency_wait();  // A may be the previous kernel's output
      uint32_t issued_mask = 0, issued_phase = 0;
      bool ok = true;
      int it = 0;  // stages issued
      for (int t = pair; ok && t < tiles; t += pairs) {
        int mt, nt;
        pair_tile(t, m_tiles, n_tiles, g.band, mt, nt);
        const int arow = mt * 256 + rank * 128;
        const int bcol = nt * BN + rank * (BN / 2);
        for (int st = 0; st < steps; ++st, ++it) {
          const int s = it % ST;
          const uint32_t ph = (uint32_t)(it / ST) & 1u;
          if (it >= ST && !mbar_wait(empty + s, ph ^ 1, abort_flag, err)) { ok = false; break; }
          const uint32_t bar = lead_full + (uint32_t)s * 8u;
          const int sl = st * kKC, k = sl * C::kBK;
          if (is_a) {
            if (rank == 0) {
              mbar_arrive_expect_tx(full + s, 2 * C::kStageBytes);
              issued_mask |= 1u << s;
              issued_phase = (issued_phase & ~(1u << s)) | (ph << s);
            }
            uint8_t* dst = sA + (size_t)s * C::kABytes;
            if (g.slices3d) {
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
              if (g.strips3d) {
                tma_load_3d_pair(dst, &tmB, 0, k, bcol / 64, bar, pol);
              } else {
#pragma unroll
                for (int c = 0; c < BN / 128; ++c)
                  tma_load_2d_pair(dst + c * 16384, &tmB, bcol + 64 * c, k, bar, pol);
              }
            } else if (g.slices3d) {
              tma_load_3d_pair(dst, &tmB, 0, bcol, sl, bar, pol);
            } else {
#pragma unroll
              for (int c = 0; c < kKC; ++c)
                tma_load_2d_pair(dst + c * C::kBCh, &tmB, k + c * C::kBK, bcol, bar, pol);
            }
          }
        }
      }
      if (ok && is_a) grid_dependents_launch();
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
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc =
          make_idesc_major(Tr::kDFmt, Tr::kAFmt, Tr::kBFmt, 256, BN, 0, C::kMn ? 1 : 0);
      bool ok = true, any = false;
      int it = 0, fill = 0;  // stages consumed; accumulator fills started
      for (int t = pair; ok && t < tiles; t += pairs) {
        if (!BS) {
          if (fill >= 2 &&
              !mbar_wait(tempty + (fill & 1), ((uint32_t)(fill >> 1) & 1u) ^ 1, abort_flag, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        for (int st = 0; st < steps; ++st, ++it) {
          const int s = it % ST;
          if (!mbar_wait(full + s, (uint32_t)(it / ST) & 1u, abort_flag, err)) { ok = false; break; }
          const uint32_t a0 = smem_u32(sA + (size_t)s * C::kABytes);
          const uint32_t b0 = smem_u32(sB + (size_t)s * C::kBBytes);
#pragma unroll
          for (int c = 0; c < kKC; ++c) {
            if (BS) {
              if (st * kKC + c >= slices) break;  // the last stage may hold one slice
              if (fill >= 2 && !mbar_wait(tempty + (fill & 1), ((uint32_t)(fill >> 1) & 1u) ^ 1,
                                          abort_flag, err)) {
                ok = false;
                break;
              }
            }
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)((fill & 1) * BN);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t bd =
                  C::kMn ? smem_desc_mnmajor_sw128(b0 + c * 8192 + 2048 * k, 16384, 1024)
                         : smem_desc_kmajor_sw128(b0 + c * C::kBCh + 32 * k);
              umma_pair<KD>(d, smem_desc_kmajor_sw128(a0 + c * C::kACh + 32 * k), bd, idesc,
                            BS ? k != 0 : (st | c | k) != 0);
            }
            any = true;
            if (BS) {
              umma_commit_pair_mc(tfull + (fill & 1), 0x3);
              ++fill;
            }
          }
          if (!ok) break;
          umma_commit_pair_mc(empty + s, 0x3);
        }
        if (!ok) break;
        if (!BS) {
          umma_commit_pair_mc(tfull + (fill & 1), 0x3);
          ++fill;
        }
      }
      if (!ok && any) {
        // Unwinding: wait (bounded) until the MMAs already issued have finished.
        umma_commit_pair(drain);
        const uint64_t tw = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - tw < kWaitLimitNs) {
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;            // TMEM lane quarter
    const int eg = (warp - 2) >> 2;    // which half of the tile's chunks
    const int ew = warp - 2;
    constexpr int kChunks = BN / 32;
    constexpr int kMine = (kChunks + 1) / 2;
    uint8_t* slab0 = slabs + ew * 2 * kSlab;
    const uint32_t lead_tempty = mapa_shared(smem_u32(tempty), 0);
    const bool res = ep.res != nullptr;
    grid_dependency_wait();
    int fill = 0;  // accumulator fills read
    int cnt = 0;   // chunks stored: slab cnt & 1, residual phase (cnt >> 1) & 1
    bool ok = true;
    // The j-th chunk of this warp: BS halves the tile's columns, the other form alternates chunks.
    auto chunk_col = [&](int j) { return BS ? (eg * kMine + j) * 32 : (2 * j + eg) * 32; };
    auto fetch_res = [&](int c, int col0, int row0) {  // lane 0: residual of chunk c into its slab
      bulk_wait_read<0>();  // no store still reads the slab
      uint64_t* bar = rbar + 2 * ew + (c & 1);
      mbar_arrive_expect_tx(bar, kSlab);
      tma_load_2d(slab0 + (c & 1) * kSlab, &tmR, col0, row0, bar, policy_evict_first());
    };
    for (int t = pair; t < tiles; t += pairs) {
      int mt, nt;
      pair_tile(t, m_tiles, n_tiles, g.band, mt, nt);
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
      for (int i = threadIdx.x - 64; i < BN; i += kEpiWarpsP * 32) {
        const int n = min(n0 + i, g.N - 1);
        float2 cb = make_float2(1.f, 0.f);
        if (!BS && ep.b_s != nullptr) cb.x = __ldg(ep.b_s + (int64_t)(n / ep.bn) * ep.b_s_ld);
        if (ep.bias != nullptr) cb.y = ld_dtype(ep.bias, n, ep.dtype);
        cols[i] = cb;
      }
      epi_barrier();
      // After a failed wait a warp still walks the tiles: the others count on it at the barriers.
      if (!ok) continue;
      if (res && mine > 0 && lane == 0) fetch_res(cnt, n0 + chunk_col(0), row0);

      // One 32 x 32 chunk: v holds this lane's row, scaled; slab, TMA store.
      auto put_chunk = [&](int j, float* v) {
        const int col0 = chunk_col(j);
        uint8_t* slab = slab0 + (cnt & 1) * kSlab;
        const float4* cb4 = reinterpret_cast<const float4*>(cols + col0);
        if (res) {
          if (j + 1 < mine && lane == 0) fetch_res(cnt + 1, n0 + chunk_col(j + 1), row0);
          if (!mbar_wait(rbar + 2 * ew + (cnt & 1), (uint32_t)(cnt >> 1) & 1u, abort_flag, err))
            ok = false;
        } else {
          if (lane == 0) bulk_wait_read<1>();  // the store before last has read this slab
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // 16-byte pieces of 8 columns, swizzled as the TMA box is
          uint4* at = reinterpret_cast<uint4*>(slab + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
          uint4 rv = make_uint4(0u, 0u, 0u, 0u);
          if (res) rv = *at;
          const uint32_t rw[4] = {rv.x, rv.y, rv.z, rv.w};
          uint32_t ow[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const float4 cb = cb4[c * 4 + p];
            float x0 = epi_act<true>(v[c * 8 + 2 * p] + cb.y, ep.act);
            float x1 = epi_act<true>(v[c * 8 + 2 * p + 1] + cb.w, ep.act);
            if (ep.dtype == TO_BF16) {
              if (res) {
                x0 += __uint_as_float(rw[p] << 16);
                x1 += __uint_as_float(rw[p] & 0xFFFF0000u);
              }
              const __nv_bfloat162 o = __floats2bfloat162_rn(x0, x1);
              ow[p] = *reinterpret_cast<const uint32_t*>(&o);
            } else {
              if (res) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&rw[p]));
                x0 += f.x;
                x1 += f.y;
              }
              const __half2 o = __floats2half2_rn(x0, x1);
              ow[p] = *reinterpret_cast<const uint32_t*>(&o);
            }
          }
          *at = make_uint4(ow[0], ow[1], ow[2], ow[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && ok) {
          tma_store_2d(&tmC, n0 + col0, row0, slab);
          bulk_commit();
        }
        ++cnt;
      };

      if constexpr (BS) {
        const float* arow = ep.a_s + (int64_t)row * ep.a_s_ld;
        const int half0 = min(n0 + eg * 128, g.N - 1);
        const float* bcol = ep.b_s + (int64_t)(half0 / ep.bn) * ep.b_s_ld;
        float run[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) run[j] = 0.f;
        float sc_next = __ldg(arow) * __ldg(bcol);
        for (int sl = 0; sl < slices; ++sl, ++fill) {
          const float sc = sc_next;
          if (sl + 1 < slices) {
            const int kb = (sl + 1) / ep.kb_per_scale;
            sc_next = __ldg(arow + kb) * __ldg(bcol + kb);
          }
          const int b = fill & 1;
          if (!mbar_wait(tfull + b, (uint32_t)(fill >> 1) & 1u, abort_flag, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN + eg * 128);
          const float2 sc2 = make_float2(sc, sc);
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            uint32_t r[32];
            tmem_ld16(taddr + c, r);
            tmem_ld16(taddr + c + 16, r + 16);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float2 p;
              if constexpr (KD == Kind::I8) {
                // exact: |P| <= 128^3 < 2^22, (bits(1.5 2^23) + P) - 1.5 2^23
                p = sub2_rn(make_float2(__int_as_float(0x4B400000 + (int32_t)r[j]),
                                        __int_as_float(0x4B400000 + (int32_t)r[j + 1])),
                            make_float2(12582912.0f, 12582912.0f));
              } else {
                p = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
              }
              const float2 a = fma2_rn(p, sc2, make_float2(run[c + j], run[c + j + 1]));
              run[c + j] = a.x;
              run[c + j + 1] = a.y;
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(lead_tempty + (uint32_t)b * 8u);
        }
        if (!ok) continue;
#pragma unroll
        for (int j = 0; j < kMine; ++j)
          if (j < mine) put_chunk(j, run + 32 * j);
      } else {
        const float sa = ep.a_s != nullptr ? __ldg(ep.a_s + (int64_t)row * ep.a_s_ld) : 1.f;
        const int b = fill & 1;
        if (!mbar_wait(tfull + b, (uint32_t)(fill >> 1) & 1u, abort_flag, err)) {
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
          for (int i = 0; i < 32; ++i) {
            const float a = KD == Kind::I8 ? (float)(int32_t)r[i] : __uint_as_float(r[i]);
            v[i] = C::kMn ? a : a * (sa * cols[c0 + i].x);
          }
          put_chunk(j, v);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(lead_tempty + (uint32_t)b * 8u);
        ++fill;
      }
    }
    if (lane == 0) bulk_wait_read<0>();  // stores have read their slabs
    if (!ok && lane == 0) {
      // Unwinding: a residual copy in flight lands within microseconds.
      const uint64_t tw = globaltimer_ns();
      while (globaltimer_ns() - tw < 50000ull) {
      }
    }
  }

  tc_fence_before();
  cluster_sync_all();  // both epilogues are done with TMEM; no signal to a peer is pending
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair<C::kTmemCols>(tmem);
  }
}

// Tensor map with the given box and swizzle; strides in bytes.
int tiled_map(CUtensorMap* out, CUtensorMapDataType dt, const void* p, int rank,
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

// K-major operand: box_rows rows of kKC slices (3-D) or of one slice (2-D).
int kmajor_map(CUtensorMap* out, const void* p, int64_t rows, int64_t K, int64_t pitch, int elem,
               int box_rows, bool slices3d) {
  const auto dt = elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  const cuuint32_t bk = (cuuint32_t)(128 / elem);
  if (slices3d) {
    const cuuint64_t dims[3] = {bk, (cuuint64_t)rows, (cuuint64_t)(K / bk)};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch, 128};
    const cuuint32_t box[3] = {bk, (cuuint32_t)box_rows, (cuuint32_t)kKC};
    return tiled_map(out, dt, p, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {bk, (cuuint32_t)box_rows};
  return tiled_map(out, dt, p, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <Kind KD, int BN, bool BS>
int launch_pair(const void* a, int64_t lda, const void* b, int64_t M, int64_t N, int64_t K,
                const LinEpi& ep, cudaStream_t st) {
  using C = PairCfg2<KD, BN, BS>;
  auto kern = k_linear_pair<KD, BN, BS>;
  const cudaError_t ae = ensure_smem_attr((const void*)kern, (int)C::kSmem);
  if (ae != cudaSuccess) return cuda_fail(ae, "linear epilogue (pairs): shared memory attribute");
  PairArgs g;
  memset((void*)&g, 0, sizeof(g));
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.slices3d = (K * C::kElem) % 128 == 0;
  g.strips3d = C::kMn && N % 64 == 0;
  // Bands whose A rows stay within 32 MB of L2.
  g.band = (int64_t)16 * 256 * K * C::kElem <= ((int64_t)32 << 20) ? 16 : 8;
  g.small_m = M <= 256;
  g.ep = ep;
  CUtensorMap ta, tb, tc, tr;
  memset(&tr, 0, sizeof(tr));
  int rc = kmajor_map(&ta, a, M, K, lda * C::kElem, C::kElem, 128, g.slices3d);
  if (rc) return rc;
  if (!C::kMn) {
    rc = kmajor_map(&tb, b, N, K, K * C::kElem, C::kElem, BN / 2, g.slices3d);
  } else if (g.strips3d) {
    const cuuint64_t dims[3] = {64, (cuuint64_t)K, (cuuint64_t)(N / 64)};
    const cuuint64_t strides[2] = {(cuuint64_t)(N * 2), 128};
    const cuuint32_t box[3] = {64, 64 * kKC, BN / 128};
    rc = tiled_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT16, b, 3, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)K};
    const cuuint64_t strides[1] = {(cuuint64_t)(N * 2)};
    const cuuint32_t box[2] = {64, 64 * kKC};
    rc = tiled_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT16, b, 2, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (rc) return rc;
  const cuuint64_t odims[2] = {(cuuint64_t)N, (cuuint64_t)M};
  const cuuint32_t obox[2] = {32, 32};
  const cuuint64_t cstr[1] = {(cuuint64_t)(ep.ldc * 2)}, rstr[1] = {(cuuint64_t)(ep.ldr * 2)};
  rc = tiled_map(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT16, ep.c, 2, odims, cstr, obox,
                 CU_TENSOR_MAP_SWIZZLE_64B);
  if (!rc && ep.res != nullptr)
    rc = tiled_map(&tr, CU_TENSOR_MAP_DATA_TYPE_UINT16, ep.res, 2, odims, rstr, obox,
                   CU_TENSOR_MAP_SWIZZLE_64B);
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
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (launch_overlap()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, tr, g, device_error_ptr());
  if (e != cudaSuccess) return cuda_fail(e, "linear epilogue (pairs) launch");
  return check_launch("linear epilogue (pairs)");
}

bool aligned_rows(const void* p, int64_t pitch) {
  return ((reinterpret_cast<uint64_t>(p) | (uint64_t)pitch) & 15u) == 0;
}

}  // namespace

// Runs the product on CTA pairs, or returns TO_EUNSUPPORTED (nothing launched, nothing recorded)
// where the tiles do not apply: 16-bit output, rows of every operand 16-byte aligned, block scales
// constant over 128 columns, and enough tiles to fill the SMs.
int linear_pair_launch(int kind, bool block_scaled, const void* a, int64_t lda, const void* b,
                       int64_t M, int64_t N, int64_t K, const LinEpi& ep, cudaStream_t st) {
  const int e = kind == TO_F16 || kind == TO_BF16 ? 2 : 1;
  if (M <= 128 || (ep.dtype != TO_F16 && ep.dtype != TO_BF16)) return TO_EUNSUPPORTED;
  if (!aligned_rows(a, lda * e) || !aligned_rows(b, (e == 2 ? N : K) * e) ||
      !aligned_rows(ep.c, ep.ldc * 2) || (ep.res && !aligned_rows(ep.res, ep.ldr * 2)))
    return TO_EUNSUPPORTED;
  if (block_scaled && ep.bn % 128 != 0 && ep.bn < N) return TO_EUNSUPPORTED;
  const int64_t pairs = sm_count() / 2;
  // Tile width: the one whose rounds of tiles cost least; a tile's time is its width plus a fixed
  // part worth about 32 columns.
  const int64_t mt = ceil_div(M, 256);
  int best = 0;
  int64_t best_cost = 0;
  const int widths[5] = {256, 192, 160, 128, 64};
  for (int w : widths) {
    if (block_scaled && w != 256) continue;
    if (e == 2 && w % 128 != 0) continue;
    const int64_t cost = ceil_div(mt * ceil_div(N, w), pairs) * (w + 32);
    if (best == 0 || cost < best_cost) {
      best = w;
      best_cost = cost;
    }
  }
  if (mt * ceil_div(N, best) * 2 < pairs) return TO_EUNSUPPORTED;  // split K instead
  if (kind == TO_F16)
    return best == 256 ? launch_pair<Kind::F16, 256, false>(a, lda, b, M, N, K, ep, st)
                       : launch_pair<Kind::F16, 128, false>(a, lda, b, M, N, K, ep, st);
  if (kind == TO_BF16)
    return best == 256 ? launch_pair<Kind::BF16, 256, false>(a, lda, b, M, N, K, ep, st)
                       : launch_pair<Kind::BF16, 128, false>(a, lda, b, M, N, K, ep, st);
  if (block_scaled)
    return kind == TO_I8 ? launch_pair<Kind::I8, 256, true>(a, lda, b, M, N, K, ep, st)
                         : launch_pair<Kind::E4M3, 256, true>(a, lda, b, M, N, K, ep, st);
  auto run = [&](auto kd) {
    constexpr Kind KD = decltype(kd)::value;
    switch (best) {
      case 256: return launch_pair<KD, 256, false>(a, lda, b, M, N, K, ep, st);
      case 192: return launch_pair<KD, 192, false>(a, lda, b, M, N, K, ep, st);
      case 160: return launch_pair<KD, 160, false>(a, lda, b, M, N, K, ep, st);
      case 128: return launch_pair<KD, 128, false>(a, lda, b, M, N, K, ep, st);
      default: return launch_pair<KD, 64, false>(a, lda, b, M, N, K, ep, st);
    }
  };
  return kind == TO_I8 ? run(std::integral_constant<Kind, Kind::I8>{})
                       : run(std::integral_constant<Kind, Kind::E4M3>{});
}

}  // namespace sm100
}  // namespace tob
