// Products with bias, activation and residual in their epilogue, in the orientation "weights as
// rows": C^T = W X^T, a tile being 128 weight columns of the output x NT tokens. The weights are
// the 128-row operand of tcgen05.mma and the tokens its N operand, so a single token costs a
// 16-column tile and not a 128-row one, and the epilogue's lanes run along consecutive output
// columns: bias and column scale are one register per lane, rows of C and of the residual are
// read and written coalesced at any alignment.
//
//   weights  int8 / e4m3 [N, K] (K-major), or fp16 / bf16 [K, N] (MN-major, 64-column strips)
//   tokens   [M, K], rows lda apart
//
// One token: bound by the weights' HBM stream. The K blocks of a column tile are split over the S
// CTAs of a cluster so that every SM streams. Rank r finishes tokens r, r + S, ...: every rank stores
// its partial sums (int32 or fp32) of a token into that rank's shared memory, one cluster barrier
// later the owner adds them in rank order (deterministic, no workspace) and nobody reads a peer.
//
// Operands come by TMA: their rows are 16-byte aligned, by themselves or as padded copies.
//
// Graph-timed on inputs beyond L2 (floor: the bytes at the copy rate of 6.45 TB/s): bf16 4096 x 4096,
// one token 8.5 us (5.2); bf16 14336 -> 4096, 16 tokens 21.7 us (18.3), 5.4 TB/s; FP8 8192 -> 28672, one
// token 39.9 us (36.4), 5.9 TB/s; FP8 block-scaled 7168 x 7168, one token 12.3 us (8.0). What is left of
// the short ones is a launch, the first copy's latency and the cluster's barrier, 3 to 4 us.
//
// Roles: warp 0 weight copies, warp 1 MMA issue and TMEM, warp 2 token copies, warp 3 idle, then
// kEpiWarps epilogue warps (lane quarter = warp % 4).
// Every wait is bounded (kWaitLimitNs); on expiry all roles unwind through the same barriers.
#include <cudaTypedefs.h>

#include <string.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "linear_epi.cuh"
#include "sm100.cuh"

namespace tob {
namespace sm100 {

PFN_cuTensorMapEncodeTiled_v12000 get_encode();

namespace {

template <Kind KD, int NT, bool BS>
struct NtCfg {
  static_assert(NT == 16 || NT == 32 || NT == 64 || NT == 128, "token tile");
  static constexpr int kElem = KindTraits<KD>::kElemBytes;
  static constexpr bool kMn = kElem == 2;   // weights [K, N]
  static constexpr int kBK = 128 / kElem;   // K elements per stage
  static constexpr int kWBytes = 128 * 128;
  static constexpr int kXBytes = NT * 128;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kEpiWarps = NT >= 64 ? 8 : 4;
  static constexpr int kTpt = NT / (kEpiWarps / 4);  // tokens per epilogue thread
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  // Two CTAs per SM where they fit: one CTA's prologue and reduction run under the other's stream.
  // The sums of 128 tokens do not fit twice.
  static constexpr int kMinBlocks = NT == 128 ? 1 : 2;
  static constexpr int kSumBytes = (NT + 7) * 512;  // partial sums [token of this rank][rank][128]
  static constexpr int kStages =
      std::min(8, ((kMinBlocks == 2 ? 110 : 220) * 1024 - kSumBytes) / kStageBytes);
  static constexpr int kTmemCols = (BS ? 2 : 1) * NT < 32 ? 32 : (BS ? 2 : 1) * NT;
  static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kSumBytes + 512;
  static_assert((2 * kStages + 6) * 8 + 16 <= 512, "barrier area");
  static_assert(kStages >= 3, "ring");
  static_assert(kSmem <= 232448, "shared memory");
};

struct NtArgs {
  int M, N, K, splits;
  int strips3d;       // MN-major weights through the 3-D strip map (N % 64 == 0)
  LinEpi ep;
};

template <Kind KD, int NT, bool BS>
__global__ void __launch_bounds__(NtCfg<KD, NT, BS>::kThreads,
                                  NtCfg<KD, NT, BS>::kMinBlocks)
    k_linear_nt(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                const __grid_constant__ NtArgs g, int* err) {
  using C = NtCfg<KD, NT, BS>;
  using Tr = KindTraits<KD>;
  constexpr int ST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sW = smem_raw;
  uint8_t* sX = smem_raw + (size_t)ST * C::kWBytes;
  uint8_t* sums = smem_raw + (size_t)ST * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sums + C::kSumBytes);
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;   // [2]; unscaled products use tfull[0]
  uint64_t* tempty = tfull + 2;   // [2]
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = g.splits;
  const int rank = (int)blockIdx.x % S;
  const int n0 = ((int)blockIdx.x / S) * 128;
  const int t0 = (int)blockIdx.y * NT;
  const int tokens = min(NT, g.M - t0);
  const int kblocks = (g.K + C::kBK - 1) / C::kBK;
  const int kb_lo = (int)((int64_t)kblocks * rank / S);
  const int kb_n = (int)((int64_t)kblocks * (rank + 1) / S) - kb_lo;
  const bool misaligned = (smem_u32(smem_raw) & 1023u) != 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full + s, 2);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull + b, 1);
      mbar_init(tempty + b, C::kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
    if (misaligned && err) atomicExch(err, (int)kErrSmemAlign);
  }
  if (warp == 1) tmem_alloc<C::kTmemCols>(tmem_holder);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  bool ok = !misaligned;
  if (S > 1) cluster_arrive_relaxed();  // this CTA runs: its shared memory may be stored to

  if (!ok) {
    // nothing to do; fall through to the barriers and the teardown
  } else if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------ TMA: weights / tokens
    if (lane == 0) {
      const bool wts = warp == 0;
      // The weights stream once past L2's other contents; every column tile re-reads the tokens.
      const uint64_t pol = wts ? policy_evict_first() : policy_evict_last();
      grid_dependency_wait();
      if (!wts) grid_dependents_launch();  // the next kernel may set itself up
      uint32_t issued_mask = 0, issued_phase = 0;
      for (int it = 0; it < kb_n; ++it) {
        const int s = it % ST;
        const uint32_t ph = (uint32_t)(it / ST) & 1u;
        const int k = (kb_lo + it) * C::kBK;
        if (it >= ST && !mbar_wait_polled(empty + s, ph ^ 1, abort_flag, err)) { ok = false; break; }
        mbar_arrive_expect_tx(full + s, wts ? C::kWBytes : C::kXBytes);
        if (!wts) {
          tma_load_2d(sX + (size_t)s * C::kXBytes, &tmX, k, t0, full + s, pol);
        } else if (!C::kMn) {
          tma_load_2d(sW + (size_t)s * C::kWBytes, &tmW, k, n0, full + s, pol);
        } else if (g.strips3d) {
          tma_load_3d(sW + (size_t)s * C::kWBytes, &tmW, 0, k, n0 / 64, full + s, pol);
        } else {
          tma_load_2d(sW + (size_t)s * C::kWBytes, &tmW, n0, k, full + s, pol);
          tma_load_2d(sW + (size_t)s * C::kWBytes + 8192, &tmW, n0 + 64, k, full + s, pol);
        }
        issued_mask |= 1u << s;
        issued_phase = (issued_phase & ~(1u << s)) | (ph << s);
      }
      if (!ok) {
        // Unwinding: let the copies in flight land before the CTA exits (one deadline).
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
    // The whole warp walks the loop and one lane issues, so that addresses and descriptors stay in
    // uniform registers: per lane, their arithmetic bounds the slices of a split product.
    constexpr uint32_t idesc =
        make_idesc_major(Tr::kDFmt, Tr::kAFmt, Tr::kBFmt, 128, NT, C::kMn ? 1 : 0, 0);
    // MN-major: 64-column strips of 64 K rows (8 KB apart); 16 K rows are 2 KB
    constexpr uint32_t kWStep = (C::kMn ? 2048 : 32) >> 4;
    const uint64_t wdesc = C::kMn ? smem_desc_mnmajor_sw128(smem_u32(sW), 8192, 1024)
                                  : smem_desc_kmajor_sw128(smem_u32(sW));
    const uint64_t xdesc = smem_desc_kmajor_sw128(smem_u32(sX));
    const bool issue = elect_one();
    grid_dependency_wait();  // the waits below count this kernel's time, not the previous one's
    bool any = false;
    int s = 0;
    uint32_t ph = 0;
    for (int it = 0; it < kb_n; ++it) {
      const int b = BS ? it & 1 : 0;
      ok = mbar_wait_warp(full + s, ph, abort_flag, err);
      if (BS && ok && it >= 2)
        ok = mbar_wait_warp(tempty + b, ((uint32_t)(it >> 1) & 1u) ^ 1, abort_flag, err);
      if (!ok) break;
      tc_fence_after();
      if (issue) {
        const uint64_t wd = wdesc + (uint64_t)(s * (C::kWBytes >> 4));
        const uint64_t xd = xdesc + (uint64_t)(s * (C::kXBytes >> 4));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma<KD>(tmem + (uint32_t)(b * NT), wd + kWStep * k, xd + 2 * k, idesc,
                   BS ? k != 0 : (it | k) != 0);
        umma_commit(empty + s);
        if (BS) umma_commit(tfull + b);
      }
      __syncwarp();
      any = true;
      if (++s == ST) { s = 0; ph ^= 1; }
    }
    if (issue) {
      if (ok && !BS) umma_commit(tfull);
      if (!ok && any) {
        // Unwinding: wait (bounded) until the MMAs already issued have finished with TMEM.
        umma_commit(drain);
        const uint64_t tw = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - tw < kWaitLimitNs) {
        }
      }
    }
    __syncwarp();
  }

  // -------------------------------------------------------------- epilogue
  const bool epi = warp >= 4;
  const int q = warp & 3;                     // TMEM lane quarter
  const int half = (warp - 4) >> 2;           // which kTpt tokens of the tile
  const int n = n0 + q * 32 + lane;
  const bool n_ok = n < g.N;
  const LinEpi& ep = g.ep;
  float bias = 0.f, sb = 1.f;
  // This thread's place in the sums, and the store of its partial sum of token tok = own * S + rank
  // of the token's owner.
  const uint32_t sum0 = smem_u32(sums + (q * 32 + lane) * 4);
  auto give = [&](int own, int owner, uint32_t v) {
    const uint32_t at = sum0 + (uint32_t)(own * S + rank) * 512u;
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(at, (uint32_t)owner)), "r"(v)
                 : "memory");
  };
  int owner = epi ? half * C::kTpt % S : 0, own = epi ? half * C::kTpt / S : 0;
  auto next_token = [&]() {
    if (++owner == S) { owner = 0; ++own; }
  };
  // One output of token tok: acc is its scaled sum.
  auto finish = [&](float acc, int tok, float res) {
    const float v = acc + bias;
    const float y = !ep.form.gated       ? act_plain(v, ep.form)
                    : ep.dtype == TO_F32 ? act_gated_f32(v, ep.act)
                                         : act_gated(v, ep.form);
    st_dtype(ep.c, (int64_t)(t0 + tok) * ep.ldc + n, ep.dtype, y + res);
  };
  if (S > 1) cluster_wait_acquire();  // so do the peers
  if (epi && ok) {
    grid_dependency_wait();
    if (n_ok && ep.bias != nullptr) bias = ld_dtype(ep.bias, n, ep.dtype);
    const int64_t brow = (n_ok ? (int64_t)n / ep.bn : 0) * ep.b_s_ld;
    if (!BS && ep.b_s != nullptr && n_ok) sb = __ldg(ep.b_s + brow);
    const uint32_t lane_addr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * C::kTpt);
    if constexpr (BS) {
      // A slice's scales are loaded while the one before is folded: their latency is as long as a
      // slice of few tokens.
      constexpr int kSa = (C::kTpt + 31) / 32;
      float run[C::kTpt], sa_n[kSa], s_col_n = 0.f;
#pragma unroll
      for (int j = 0; j < C::kTpt; ++j) run[j] = 0.f;
      auto load_scales = [&](int it) {
        const int kb = (kb_lo + it) / ep.kb_per_scale;
        s_col_n = n_ok ? __ldg(ep.b_s + brow + kb) : 0.f;
#pragma unroll
        for (int i = 0; i < kSa; ++i) {
          const int t = half * C::kTpt + i * 32 + lane;
          sa_n[i] = t < tokens ? __ldg(ep.a_s + (int64_t)(t0 + t) * ep.a_s_ld + kb) : 0.f;
        }
      };
      if (kb_n > 0) load_scales(0);
      for (int it = 0; it < kb_n; ++it) {
        const float s_col = s_col_n;
        float sa_l[kSa];
#pragma unroll
        for (int i = 0; i < kSa; ++i) sa_l[i] = sa_n[i];
        if (it + 1 < kb_n) load_scales(it + 1);
        const int b = it & 1;
        if (!mbar_wait_polled(tfull + b, (uint32_t)(it >> 1) & 1u, abort_flag, err)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::kTpt; c += 16) {
          uint32_t r[16];
          tmem_ld16(lane_addr + (uint32_t)(b * NT + c), r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float p = KD == Kind::I8 ? (float)(int32_t)r[j] : __uint_as_float(r[j]);
            const float sa = __shfl_sync(0xffffffffu, sa_l[(c + j) / 32], (c + j) & 31);
            run[c + j] = fmaf(p * sa, s_col, run[c + j]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty + b);
      }
      if (ok) {
#pragma unroll
        for (int j = 0; j < C::kTpt; ++j) {
          if (half * C::kTpt + j < tokens) give(own, owner, __float_as_uint(run[j]));
          next_token();
        }
      }
    } else {
      ok = mbar_wait_polled(tfull, 0, abort_flag, err);
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < C::kTpt; c += 16) {
        const int tok0 = half * C::kTpt + c;
        if (!ok || tok0 >= tokens) break;
        uint32_t r[16];
        tmem_ld16(lane_addr + (uint32_t)c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (tok0 + j < tokens) give(own, owner, r[j]);
          next_token();
        }
      }
    }
  }
  // A short loop over this rank's tokens finishes them: this code runs once, so what it costs is the
  // fetching of its instructions and the latency of its loads. Without a split every thread reads
  // back what it stored, so no barrier is needed.
  if (S > 1) cluster_arrive_release();
  const int mine = (tokens - rank + S - 1) / S;  // tokens of this rank
  const int i_step = S > 1 ? C::kEpiWarps / 4 : 1;
  const int i_first = S > 1 ? half : half * C::kTpt;
  const int i_last = S > 1 ? mine : min(mine, (half + 1) * C::kTpt);
  constexpr int U = 4;  // tokens whose loads are in flight together
  uint32_t res[U];
  float sc[U];
  auto operands = [&](int i0) {  // residual and scale of the next U tokens
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + rank + (int64_t)min(i0 + u * i_step, i_last - 1) * S;
      res[u] = ep.res == nullptr ? 0u : ld_raw(ep.res, t * ep.ldr + n, ep.dtype == TO_F32);
      sc[u] = !BS && ep.a_s != nullptr ? __ldg(ep.a_s + t * ep.a_s_ld) * sb : 1.f;
    }
  };
  const bool work = epi && ok && n_ok && i_first < i_last;
  if (work) operands(i_first);
  if (S > 1) cluster_wait_acquire();
  if (work) {
#pragma unroll 1
    for (int i0 = i_first; i0 < i_last; i0 += U * i_step) {
      float acc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * i_step, i_last - 1);
        const uint32_t* at = reinterpret_cast<const uint32_t*>(sums + (q * 32 + lane) * 4) +
                             (size_t)i * S * 128;
        uint32_t sum = at[0];
        for (int s = 1; s < S; ++s) {
          const uint32_t v = at[s * 128];
          if (KD == Kind::I8 && !BS) sum += v;
          else sum = __float_as_uint(__uint_as_float(sum) + __uint_as_float(v));
        }
        acc[u] = (KD == Kind::I8 && !BS ? (float)(int32_t)sum : __uint_as_float(sum)) * sc[u];
      }
      float r_now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r_now[u] = raw_to_f32(res[u], ep.dtype);
      if (i0 + U * i_step < i_last) operands(i0 + U * i_step);  // in flight under the stores
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * i_step < i_last) finish(acc[u], rank + (i0 + u * i_step) * S, r_now[u]);
    }
  }
  grid_dependency_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<C::kTmemCols>(tmem);
  }
}

// 2-D map of `rows` x `cols` elements, rows `pitch` bytes apart, boxes of 128 bytes x box_rows in
// the 128-byte swizzle. Built per call: it costs well under a microsecond.
int rows_map(CUtensorMap* out, const void* p, int64_t rows, int64_t cols, int64_t pitch, int elem,
             int box_rows) {
  auto encode = get_encode();
  if (!encode) return fail(TO_ECUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = encode(
      out, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
      const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TO_ECUDA, "cuTensorMapEncodeTiled failed (%d) for [%lld, %lld]", (int)r,
                (long long)rows, (long long)cols);
  return TO_OK;
}

// Weights [K, N], N % 64 == 0, as {64 columns, K rows, N / 64 strips}: one box of two strips.
int strips_map(CUtensorMap* out, const void* p, int64_t K, int64_t N, int64_t pitch) {
  auto encode = get_encode();
  if (!encode) return fail(TO_ECUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  cuuint64_t dims[3] = {64, (cuuint64_t)K, (cuuint64_t)(N / 64)};
  cuuint64_t strides[2] = {(cuuint64_t)pitch, 128};
  cuuint32_t box[3] = {64, 64, 2};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(p), dims,
                            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TO_ECUDA, "cuTensorMapEncodeTiled (strips) failed (%d) for [%lld, %lld]", (int)r,
                (long long)K, (long long)N);
  return TO_OK;
}

// Clusters of S (at most 8) CTAs that the current device holds at once: the driver's count, asked once
// per device and kernel. Threads that ask at the same time store the same number.
template <Kind KD, int NT, bool BS>
int clusters_at_once(int S) {
  using C = NtCfg<KD, NT, BS>;
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][9];  // count + 1, 0 unknown
  const void* kern = (const void*)k_linear_nt<KD, NT, BS>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
  auto ask = [&](int s) {
    int n = known[dev][s].load(std::memory_order_relaxed);
    if (n > 0) return n - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(s * 1024), 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();  // the launch itself says what is wrong
      return 0;
    }
    known[dev][s].store(n + 1, std::memory_order_relaxed);
    return n;
  };
  // The driver counts one block per SM; the kernels sized for two run two (their blocks were seen to
  // start together, and the split that this count allows is the fastest).
  const int times = ask(1) <= sm_count() ? C::kMinBlocks : 1;
  return ask(S) * times;
}

// K split: the most CTAs that the SMs hold at once, at least two K blocks each, at most a portable
// cluster of eight. Clusters have to fit into the GPU's processor clusters whole, so the count comes
// from the driver. One token, 7168 x 7168 FP8 block-scaled, 56 tiles: two ways 21.6 us, three 16.3,
// four 14.1, and five, 280 CTAs for 296 places but two rounds, 20.0. 0: not even unsplit.
template <Kind KD, int NT, bool BS>
int split_of(const LinOps& o) {
  const int64_t tiles = ceil_div(o.N, 128) * ceil_div(o.M, NT);
  int S = (int)std::min<int64_t>(8, std::max<int64_t>(1, ceil_div(o.K, NtCfg<KD, NT, BS>::kBK) / 2));
  while (S > 0 && tiles > clusters_at_once<KD, NT, BS>(S)) --S;
  return S;
}

template <Kind KD, int NT, bool BS>
cudaError_t set_smem() {
  return ensure_smem_attr((const void*)k_linear_nt<KD, NT, BS>, (int)NtCfg<KD, NT, BS>::kSmem);
}

template <Kind KD, int NT, bool BS>
int launch_nt(const LinOps& o, const LinEpi& ep, cudaStream_t st) {
  using C = NtCfg<KD, NT, BS>;
  auto kern = k_linear_nt<KD, NT, BS>;
  const cudaError_t ae = set_smem<KD, NT, BS>();
  if (ae != cudaSuccess) return cuda_fail(ae, "linear epilogue: shared memory attribute");
  const int64_t M = o.M, N = o.N, K = o.K;
  const int64_t n_tiles = ceil_div(N, 128), m_tiles = ceil_div(M, NT);
  const int64_t S = std::max(1, split_of<KD, NT, BS>(o));
  if (n_tiles * S > INT32_MAX || m_tiles > 65535)
    return fail(TO_EUNSUPPORTED, "linear epilogue: too many tiles (M=%lld N=%lld)", (long long)M,
                (long long)N);
  NtArgs g;
  memset((void*)&g, 0, sizeof(g));
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.splits = (int)S;
  g.strips3d = C::kMn && o.b_in % 64 == 0;
  g.ep = ep;
  CUtensorMap tw, tx;
  const int64_t w_pitch = o.ldb * C::kElem;
  int rc = !C::kMn      ? rows_map(&tw, o.b, N, o.b_in, w_pitch, C::kElem, 128)
           : g.strips3d ? strips_map(&tw, o.b, K, o.b_in, w_pitch)
                        : rows_map(&tw, o.b, K, o.b_in, w_pitch, C::kElem, 64);
  if (!rc) rc = rows_map(&tx, o.a, M, o.a_k, o.lda * C::kElem, C::kElem, NT);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * S), (unsigned)m_tiles, 1);
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw, tx, g, device_error_ptr());
  if (e != cudaSuccess) return cuda_fail(e, "linear epilogue launch");
  return check_launch("linear epilogue");
}

template <Kind KD, bool BS>
int launch_nt_any(const LinOps& o, const LinEpi& ep, cudaStream_t st) {
  const int64_t M = o.M, N = o.N, K = o.K;
  // The token tile: what covers the tokens in one column of tiles, or less where the blocks, K split
  // as far as it goes, would leave SMs idle (each finishes its tokens one group after the other).
  const int64_t n_tiles = ceil_div(N, 128);
  const int64_t split = std::max<int64_t>(
      1, std::min<int64_t>(8, ceil_div(K * KindTraits<KD>::kElemBytes, 128) / 2));
  int nt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  while (nt > 16 && n_tiles * ceil_div(M, nt) * split < sm_count()) nt /= 2;
  // 64 tokens wide, an SM holds two CTAs: better where that lets K split further (145 tokens, 12544
  // -> 2240 bf16: 33.4 us three ways at 128, 25.9 four ways at 64), or where a CTA's K is short and
  // one's start and end pass under the other's loads (128 tokens, 1024 -> 4096: 10.2 and 8.7 us;
  // 200 tokens, 4096 -> 4096: 23.0 and 20.7). On long K the weights read twice cost more (80 tokens,
  // 8192 -> 4096, at the limit of 32: 18.8 and 20.0).
  if (nt == 128 && set_smem<KD, 128, BS>() == cudaSuccess && set_smem<KD, 64, BS>() == cudaSuccess) {
    const int s128 = std::max(1, split_of<KD, 128, BS>(o)), s64 = split_of<KD, 64, BS>(o);
    const int64_t blocks = ceil_div(K * KindTraits<KD>::kElemBytes, 128);
    if (s64 > s128 || (s64 == s128 && blocks <= 32 * s64)) nt = 64;
  }
  if (nt == 16) return launch_nt<KD, 16, BS>(o, ep, st);
  if (nt == 32) return launch_nt<KD, 32, BS>(o, ep, st);
  if (nt == 64) return launch_nt<KD, 64, BS>(o, ep, st);
  return launch_nt<KD, 128, BS>(o, ep, st);
}

}  // namespace

// Entry of this file: `kind` one of TO_I8, TO_E4M3 (weights [N, K]), TO_F16, TO_BF16 (weights
// [K, N]); block_scaled: ep's scales change every ep.kb_per_scale 128-byte K slices.
int linear_nt_launch(int kind, bool block_scaled, const LinOps& o, const LinEpi& ep,
                     cudaStream_t st) {
  switch (kind) {
    case TO_F16: return launch_nt_any<Kind::F16, false>(o, ep, st);
    case TO_BF16: return launch_nt_any<Kind::BF16, false>(o, ep, st);
    case TO_I8:
      return block_scaled ? launch_nt_any<Kind::I8, true>(o, ep, st)
                          : launch_nt_any<Kind::I8, false>(o, ep, st);
    case TO_E4M3:
      return block_scaled ? launch_nt_any<Kind::E4M3, true>(o, ep, st)
                          : launch_nt_any<Kind::E4M3, false>(o, ep, st);
  }
  return fail(TO_EUNSUPPORTED, "linear epilogue: operand dtype %s", dtype_name(kind));
}

}  // namespace sm100
}  // namespace tob
