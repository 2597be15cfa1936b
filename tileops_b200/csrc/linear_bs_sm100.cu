// W8A8 products with block scales and with bias, activation and residual in their epilogue, many
// tokens: persistent 128 x BN tiles, one CTA per SM.
//   C = act( sum_kb (A_kb B_kb^T)[m, n] a_s[m, kb] b_s[n / bn, kb] + bias ) + residual
//
// The products of one 128-byte K slice land in one of two TMEM buffers of BN columns; eight
// epilogue warps fold each finished buffer into fp32 running sums in registers (32 rows x up to
// four 32-column chunks a warp, 128 values a thread), run = fma(P, a_s b_s, run), while the tensor
// core fills the other. The column scale is constant over a 32-column chunk, so any block width
// that is a multiple of 32 serves, at any tile width.
//
// One CTA per tile, not a pair: a fold releases its buffer to the MMA thread every half
// microsecond, and signals that cross SMs cost more than that. Wide tiles nearly halve the
// operand bytes per product against 128 x 128 (44 KB per slice and 128 x 224 results).
//
// 4096 x 7168 x 7168 FP8 with a residual: 237 to 246 us in a lone launch, 1.7 to 1.8 PFLOP/s, and 282
// to 287 us back to back (power cap); on CTA pairs it was 442 us. That is some 1170 clocks a slice,
// of which the MMAs need 450 and shared memory 700 (44 KB written by the copies, 44 KB read by the
// MMAs, at 128 B a clock); where the other 470 go has not been measured.
//
// Every wait is bounded (kWaitLimitNs).
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "linear_tile.cuh"

namespace tob {
namespace sm100 {
namespace {

// Warps 0..3 (one warpgroup): copies of A, MMA issue and TMEM, copies of B, scales; then the
// epilogue warps. The first warpgroup gives registers to the other two: 128 sums a thread and what
// goes with them spill at the 168 that 384 threads have each. 64 + 2 x 216 <= 3 x 168.
constexpr int kBWarpB = 2, kSWarpB = 3, kEpi0B = 4;
constexpr int kThreadsB = 32 * (kEpi0B + kEpiWarpsT);
// Scales: two blocks of eight slices in shared memory, [slice][128 rows, padded | 8 chunks].
constexpr int kSB = 8;
constexpr int kSRow = 132;
constexpr int kSBlock = kSB * (kSRow + 8);

template <int BN>
struct BsTile {
  static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // slabs, scales, bias, barriers
  static constexpr int kFixed = kEpiWarpsT * 2 * kSlab + 2 * kSBlock * 4 + BN * 4 + 512;
  static constexpr int kStages = std::min(8, (232448 - kFixed) / kStageBytes);
  static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kFixed;
  static constexpr int kBufCols = 256;  // TMEM buffer stride
  static_assert(BN % 32 == 0 && BN >= 128 && BN <= 224, "tile width");
  static_assert(kStages >= 4, "ring");
  static_assert((2 * kStages + 9 + 2 * kEpiWarpsT) * 8 + 16 <= 512, "barrier area");
};

struct BsArgs {
  int M, N, K, band;
  LinEpi ep;
};

// Four bytes from global to shared memory, asynchronously; the thread's arrival on a barrier once
// all its earlier copies have landed.
__device__ __forceinline__ void cp_async4(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// tcgen05.wait::ld that the loaded registers depend on, so that no use of them moves above it.
__device__ __forceinline__ void tmem_ld_wait16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// OUT_ROWS: output or residual is no TMA tensor; a form of its own, since the other's registers are
// all taken (with both in one, 7168 x 7168 at 4096 tokens took 358 us instead of 281). At 224 columns
// it spills some 110 bytes a thread.
template <Kind KD, int BN, bool OUT_ROWS>
__global__ void __launch_bounds__(kThreadsB, 1)
    k_linear_bs(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                const __grid_constant__ BsArgs g, int* err) {
  using C = BsTile<BN>;
  using Tr = KindTraits<KD>;
  constexpr int ST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sA = smem_raw;
  uint8_t* sB = smem_raw + (size_t)ST * C::kABytes;
  uint8_t* slabs = smem_raw + (size_t)ST * C::kStageBytes;
  float* scales = reinterpret_cast<float*>(slabs + kEpiWarpsT * 2 * kSlab);
  float* bias = scales + 2 * kSBlock;
  uint64_t* full = reinterpret_cast<uint64_t*>(bias + BN);
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;   // [2] a slice's products are in buffer b
  uint64_t* tempty = tfull + 2;   // [2] the epilogue warps have read buffer b
  uint64_t* drain = tempty + 2;
  uint64_t* rbar = drain + 1;     // [8][2] a chunk's residual has landed
  uint64_t* sfull = rbar + 2 * kEpiWarpsT;  // [2] a block of scales has landed
  uint64_t* sempty = sfull + 2;             // [2] the epilogue warps are done with it
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m_tiles = (g.M + 127) / 128, n_tiles = (g.N + BN - 1) / BN;
  const int tiles = m_tiles * n_tiles;
  const int slices = (g.K + 127) / 128;
  const bool misaligned = (smem_u32(smem_raw) & 1023u) != 0;
  const LinEpi& ep = g.ep;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full + s, 2);  // the copies of A and of B
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull + b, 1);
      mbar_init(tempty + b, kEpiWarpsT);
      mbar_init(sfull + b, 32);
      mbar_init(sempty + b, kEpiWarpsT);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 2 * kEpiWarpsT; ++i) mbar_init(rbar + i, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmC);
    if (ep.res != nullptr && !OUT_ROWS) prefetch_tmap(&tmR);
    if (misaligned && err) atomicExch(err, (int)kErrSmemAlign);
  }
  if (warp == 1) tmem_alloc<512>(tmem_holder);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < kEpi0B) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (misaligned) {
      // nothing to do; fall through to the teardown
    } else if (warp == 0 || warp == kBWarpB) {
      // ------------------------------------------------------------ copies of A / of B
      if (lane == 0) {
        const bool is_a = warp == 0;
        const uint64_t pol = policy_evict_normal();
        grid_dependency_wait();
        if (is_a) grid_dependents_launch();  // the next kernel may set itself up
        uint32_t issued_mask = 0, issued_phase = 0;
        bool ok = true;
        int it = 0;
        for (int t = (int)blockIdx.x; ok && t < tiles; t += (int)gridDim.x) {
          int mt, nt;
          band_tile(t, m_tiles, n_tiles, g.band, mt, nt);
          for (int sl = 0; sl < slices; ++sl, ++it) {
            const int s = it % ST;
            const uint32_t ph = (uint32_t)(it / ST) & 1u;
            if (it >= ST && !mbar_wait_polled(empty + s, ph ^ 1, abort_flag, err)) { ok = false; break; }
            mbar_arrive_expect_tx(full + s, is_a ? C::kABytes : C::kBBytes);
            if (is_a)
              tma_load_2d(sA + (size_t)s * C::kABytes, &tmA, sl * 128, mt * 128, full + s, pol);
            else
              tma_load_2d(sB + (size_t)s * C::kBBytes, &tmB, sl * 128, nt * BN, full + s, pol);
            issued_mask |= 1u << s;
            issued_phase = (issued_phase & ~(1u << s)) | (ph << s);
          }
        }
        if (!ok) {
          // Unwinding: let the copies in flight land (one deadline for all stages).
          const uint64_t tw = globaltimer_ns();
          for (int i = 0; i < ST; ++i)
            if (issued_mask & (1u << i))
              while (!mbar_try_wait(full + i, (issued_phase >> i) & 1u) &&
                     globaltimer_ns() - tw < kWaitLimitNs) {
              }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      // The whole warp walks the loop and one lane issues: addresses and descriptors then stay in
      // uniform registers. A slice's four MMAs take 450 cycles, and computed per lane the issue of
      // them took nearly as long again.
      constexpr uint32_t idesc = make_idesc(Tr::kDFmt, Tr::kAFmt, Tr::kBFmt, 128, BN);
      const uint64_t adesc = smem_desc_kmajor_sw128(smem_u32(sA));
      const uint64_t bdesc = smem_desc_kmajor_sw128(smem_u32(sB));
      const bool issue = elect_one();
      grid_dependency_wait();  // the waits below count this kernel's time, not the previous one's
      bool ok = true;
      int it = 0, s = 0;
      uint32_t ph = 0;
      for (int t = (int)blockIdx.x; ok && t < tiles; t += (int)gridDim.x) {
        for (int sl = 0; sl < slices; ++sl, ++it) {
          const int b = it & 1;
          ok = mbar_wait_warp(full + s, ph, abort_flag, err);
          if (ok && it >= 2)
            ok = mbar_wait_warp(tempty + b, ((uint32_t)(it >> 1) & 1u) ^ 1, abort_flag, err);
          if (!ok) break;
          tc_fence_after();
          if (issue) {
            const uint64_t ad = adesc + (uint64_t)(s * (C::kABytes >> 4));
            const uint64_t bd = bdesc + (uint64_t)(s * (C::kBBytes >> 4));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma<KD>(tmem + (uint32_t)(b * C::kBufCols), ad + 2 * k, bd + 2 * k, idesc, k != 0);
            umma_commit(tfull + b);
            umma_commit(empty + s);
          }
          __syncwarp();
          if (++s == ST) { s = 0; ph ^= 1; }
        }
      }
      if (!ok && it > 0 && issue) {
        // Unwinding: wait (bounded) until the MMAs already issued have finished with TMEM.
        umma_commit(drain);
        const uint64_t tw = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - tw < kWaitLimitNs) {
        }
      }
      __syncwarp();
    } else if (warp == kSWarpB) {
      // ------------------------------------------------------------ scales, two blocks ahead
      // A lane takes one slice of the block and every fourth row: eight consecutive scales of a row
      // are one 32-byte read, and the epilogue warps' own loads (32 rows, 32 lines each) are spared.
      grid_dependency_wait();
      int blk = 0;
      bool ok = true;
      for (int t = (int)blockIdx.x; ok && t < tiles; t += (int)gridDim.x) {
        int mt, nt;
        band_tile(t, m_tiles, n_tiles, g.band, mt, nt);
        for (int s0 = 0; s0 < slices; s0 += kSB, ++blk) {
          const int sb = blk & 1;
          if (blk >= 2 && !mbar_wait_polled(sempty + sb, ((uint32_t)(blk >> 1) & 1u) ^ 1, abort_flag,
                                            err)) {
            ok = false;
            break;
          }
          const int i = lane & 7;
          const int kb = min(s0 + i, slices - 1) / ep.kb_per_scale;
          float* dst = scales + sb * kSBlock + i * (kSRow + 8);
          const float* a = ep.a_s + kb;
          for (int r = lane >> 3; r < 128; r += 4)
            cp_async4(dst + r, a + (int64_t)min(mt * 128 + r, g.M - 1) * ep.a_s_ld);
          for (int c = lane >> 3; c < BN / 32; c += 4)
            cp_async4(dst + kSRow + c,
                      ep.b_s + min(nt * BN + 32 * c, g.N - 1) / ep.bn * ep.b_s_ld + kb);
          cp_async_arrive(sfull + sb);
        }
      }
      cp_async_wait_all();
    }
  } else {
    // ------------------------------------------------------------ fold and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3;          // TMEM lane quarter
    const int eg = (warp - kEpi0B) >> 2;  // first or second half of the tile's chunks
    const int ew = warp - kEpi0B;
    constexpr int kChunks = BN / 32;
    constexpr int kMax = (kChunks + 1) / 2;                        // chunks of a first-half warp
    const int c_first = eg * kMax;                                 // this warp's first chunk
    const int c_count = eg == 0 ? kMax : kChunks - kMax;
    ChunkWriter wr{slabs + ew * 2 * kSlab, rbar + 2 * ew, &tmC, &tmR, abort_flag, err,
                   ep.form, ep.dtype, lane, ep.res != nullptr && !OUT_ROWS};
    grid_dependency_wait();
    int fill = 0, blk = 0;  // buffers folded, blocks of scales used
    bool ok = true;
    for (int t = (int)blockIdx.x; t < (misaligned ? 0 : tiles); t += (int)gridDim.x) {
      int mt, nt;
      band_tile(t, m_tiles, n_tiles, g.band, mt, nt);
      const int n0 = nt * BN;
      const int row0 = mt * 128 + q * 32;
      epi_barrier();  // every warp is done with the previous tile's bias
      for (int i = threadIdx.x - 32 * kEpi0B; i < BN; i += kEpiWarpsT * 32)
        bias[i] = ep.bias != nullptr ? ld_dtype(ep.bias, min(n0 + i, g.N - 1), ep.dtype) : 0.f;
      epi_barrier();
      // After a failed wait a warp still walks the tiles: the others count on it at the barriers.
      if (!ok) continue;
      int mine = 0;  // chunks that hold output columns
      while (mine < c_count && n0 + (c_first + mine) * 32 < g.N) ++mine;
      if (row0 >= g.M) mine = 0;
      if (mine > 0) wr.fetch(0, n0 + c_first * 32, row0);
      if (mine > 1) wr.fetch(1, n0 + c_first * 32 + 32, row0);
      for (int j = 2; j < mine; ++j) wr.want(n0 + (c_first + j) * 32, row0);

      float run[kMax * 32];
#pragma unroll
      for (int j = 0; j < kMax * 32; ++j) run[j] = 0.f;
      for (int sl = 0; sl < slices; ++sl, ++fill) {
        const int sb_i = sl % kSB;
        if (sb_i == 0 &&
            !mbar_wait_polled(sfull + (blk & 1), (uint32_t)(blk >> 1) & 1u, abort_flag, err)) {
          ok = false;
          break;
        }
        const float* slot = scales + (blk & 1) * kSBlock + sb_i * (kSRow + 8);
        const float sa = slot[q * 32 + lane];
        float4 sb;
        if (BN == 192 && eg == 1) {  // the second half starts at chunk 3: no 16-byte boundary
          sb = make_float4(slot[kSRow + 3], slot[kSRow + 4], slot[kSRow + 5], 0.f);
        } else {
          sb = *reinterpret_cast<const float4*>(slot + kSRow + (kMax == 2 ? 0 : c_first));
          if (kMax == 2 && eg == 1) sb = make_float4(sb.z, sb.w, 0.f, 0.f);
        }
        const float sc[4] = {sa * sb.x, sa * sb.y, sa * sb.z, sa * sb.w};
        const int b = fill & 1;
        if (!mbar_wait_polled(tfull + b, (uint32_t)(fill >> 1) & 1u, abort_flag, err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) +
                               (uint32_t)(b * C::kBufCols + c_first * 32);
        // Sixteen columns at a time; the two warps of a scheduler cover each other's loads. Scalar
        // sums: the packed form has the same rate here and wants its operands in aligned pairs
        // (128 columns of eight warps: 343 cycles against 463 and up). A second-half warp with fewer
        // chunks reads and folds columns past the tile into sums it never stores.
#pragma unroll
        for (int i = 0; i < 2 * kMax; ++i) {
          uint32_t r[16];
          tmem_ld16(taddr + 16 * i, r);
          tmem_ld_wait16(r);
          if (i + 1 == 2 * kMax) {  // everything is in registers: the buffer may be refilled
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty + b);
            if (sb_i == kSB - 1 || sl == slices - 1) {  // the block's scales are in registers too
              if (lane == 0) mbar_arrive(sempty + (blk & 1));
              ++blk;
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float v = KD == Kind::I8 ? (float)(int32_t)r[j] : __uint_as_float(r[j]);
            run[16 * i + j] = fmaf(v, sc[i / 2], run[16 * i + j]);
          }
        }
      }
      if (!ok) continue;
      // The chunk in front is put, the others move up: one copy of the code, fetched once.
#pragma unroll 1
      for (int j = 0; j < mine; ++j) {
        const int c0 = (c_first + j) * 32;
        if constexpr (OUT_ROWS) {
          wr.put_plain(run, bias + c0, n0 + c0, row0, ep, g.M, g.N, ok);
        } else {
          if (!wr.acquire()) ok = false;
          wr.put(run, bias + c0, n0 + c0, row0, ok);
          if (j + 2 < mine) wr.fetch(1, n0 + c0 + 64, row0);
        }
#pragma unroll
        for (int i = 0; i < (kMax - 1) * 32; ++i) run[i] = run[i + 32];
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

  grid_dependency_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

template <Kind KD, int BN>
int launch_bs(const LinOps& o, bool plain_out, const LinEpi& ep, cudaStream_t st) {
  using C = BsTile<BN>;
  auto kern = plain_out ? k_linear_bs<KD, BN, true> : k_linear_bs<KD, BN, false>;
  const cudaError_t ae = ensure_smem_attr((const void*)kern, (int)C::kSmem);
  if (ae != cudaSuccess) return cuda_fail(ae, "linear epilogue (block scales): shared memory");
  const int64_t M = o.M, N = o.N, K = o.K;
  BsArgs g;
  memset((void*)&g, 0, sizeof(g));
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  // Bands whose A rows stay within 32 MB of L2.
  g.band = (int64_t)32 * 128 * K <= ((int64_t)32 << 20) ? 32 : 16;
  g.ep = ep;
  CUtensorMap ta, tb, tc, tr;
  memset(&tc, 0, sizeof(tc));
  memset(&tr, 0, sizeof(tr));
  int rc = kmajor_map(&ta, o.a, M, o.a_k, o.lda, 1, 128, 1);
  if (!rc) rc = kmajor_map(&tb, o.b, N, o.b_in, o.ldb, 1, BN, 1);
  if (!rc && !plain_out) rc = chunk_map(&tc, ep.c, M, N, ep.ldc);
  if (!rc && !plain_out && ep.res != nullptr) rc = chunk_map(&tr, ep.res, M, N, ep.ldr);
  if (rc) return rc;
  const int64_t tiles = ceil_div(M, 128) * ceil_div(N, BN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles, sm_count()), 1, 1);
  cfg.blockDim = dim3(kThreadsB, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, tr, g, device_error_ptr());
  if (e != cudaSuccess) return cuda_fail(e, "linear epilogue (block scales) launch");
  return check_launch("linear epilogue (block scales)");
}

}  // namespace

// The tile width for a block-scaled product, 0 where these tiles do not pay or apply: column blocks
// have to be whole 32-column chunks, and the tiles to fill the SMs.
static int bs_width(int64_t M, int64_t N, int64_t bn) {
  if (M <= 64 || (bn % 32 != 0 && bn < N)) return 0;
  // The width whose rounds of tiles cost least; a tile's time is its width plus a fixed part worth
  // about 32 columns.
  const int64_t mt = ceil_div(M, 128), sms = sm_count();
  int best = 0;
  int64_t best_cost = 0;
  const int widths[3] = {224, 192, 128};
  for (int w : widths) {
    const int64_t cost = ceil_div(mt * ceil_div(N, w), sms) * (w + 32);
    if (best == 0 || cost < best_cost) {
      best = w;
      best_cost = cost;
    }
  }
  const int64_t tiles = mt * ceil_div(N, best);
  return tiles > INT32_MAX || tiles * 2 < sms ? 0 : best;  // few tiles: split K instead
}

// Runs it, or returns TO_EUNSUPPORTED (nothing launched, nothing recorded). Rows of A and B have to
// be 16-byte aligned.
int linear_bs_launch(int kind, const LinOps& o, const LinEpi& ep, cudaStream_t st) {
  const int best = bs_width(o.M, o.N, ep.bn);
  if (best == 0 || !aligned_rows(o.a, o.lda) || !aligned_rows(o.b, o.ldb)) return TO_EUNSUPPORTED;
  const bool plain = plain_output(ep, o.N);
  auto run = [&](auto kd) {
    constexpr Kind KD = decltype(kd)::value;
    switch (best) {
      case 224: return launch_bs<KD, 224>(o, plain, ep, st);
      case 192: return launch_bs<KD, 192>(o, plain, ep, st);
      default: return launch_bs<KD, 128>(o, plain, ep, st);
    }
  };
  return kind == TO_I8 ? run(std::integral_constant<Kind, Kind::I8>{})
                       : run(std::integral_constant<Kind, Kind::E4M3>{});
}

}  // namespace sm100
}  // namespace tob
