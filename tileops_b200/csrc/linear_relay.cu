// Copies of a product's operands with 16-byte aligned, zero-padded rows, for the tiles that read
// them by TMA: what a K or N that is no multiple of 16 bytes (or a pointer off alignment) costs a
// product is one pass over the operand. Bound by HBM: each operand read and written once. Both
// operands in one launch. One token 4097 x 4099 bf16 takes 23 us with its copies, 100 tokens 8191 x
// 8191 93; realigned in registers inside the product they took 32 and 166.
#include <algorithm>

#include "linear_epi.cuh"
#include "realign.cuh"

namespace tob {
namespace {

struct RelayJob {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows, row_bytes, src_pitch, dst_pitch;  // dst_pitch: a multiple of 16
};

constexpr int kRelayThreads = 256, kRelayBatch = 4;

__global__ void __launch_bounds__(kRelayThreads)
    k_linear_relay(const RelayJob j0, const RelayJob j1, int blocks0) {
  grid_dependency_wait();  // a programmatic dependent, as the products are
  grid_dependents_launch();
  const bool first = (int)blockIdx.x < blocks0;
  const RelayJob j = first ? j0 : j1;
  const int64_t blocks = first ? blocks0 : (int64_t)gridDim.x - blocks0;
  const int64_t block = first ? blockIdx.x : (int64_t)blockIdx.x - blocks0;
  const int64_t per_row = j.dst_pitch / 16, total = j.rows * per_row;
  const uint8_t* hi = j.src + (j.rows - 1) * j.src_pitch + j.row_bytes;
  const int64_t stride = blocks * kRelayThreads;
  for (int64_t i0 = block * kRelayThreads + threadIdx.x; i0 < total; i0 += stride * kRelayBatch) {
    Unaligned16 v[kRelayBatch];
#pragma unroll
    for (int u = 0; u < kRelayBatch; ++u) {
      const int64_t i = min(i0 + u * stride, total - 1);
      const int64_t r = total <= 0x7FFFFFFF ? (int64_t)((uint32_t)i / (uint32_t)per_row)
                                            : i / per_row;
      const int64_t off = (i - r * per_row) * 16;
      v[u].issue(j.src + r * j.src_pitch + off,
                 (int)max((int64_t)0, min((int64_t)16, j.row_bytes - off)), j.src, hi);
    }
#pragma unroll
    for (int u = 0; u < kRelayBatch; ++u) {
      const int64_t i = i0 + u * stride;
      if (i < total) *reinterpret_cast<uint4*>(j.dst + i * 16) = v[u].finish();
    }
  }
}

bool aligned_rows(const void* p, int64_t pitch) {
  return ((reinterpret_cast<uint64_t>(p) | (uint64_t)pitch) & 15u) == 0;
}
int64_t round128(int64_t bytes) { return (bytes + 127) / 128 * 128; }

}  // namespace

// Bytes of the padded copies of the operands whose rows TMA cannot address (0: none).
int64_t linear_relay_bytes(int kind, const LinOps& o) {
  const int e = kind == TO_F16 || kind == TO_BF16 ? 2 : 1;
  int64_t bytes = 0;
  if (!aligned_rows(o.a, o.lda * e)) bytes += o.M * round128(o.K * e);
  if (!aligned_rows(o.b, o.ldb * e)) bytes += e == 2 ? o.K * round128(o.N * 2) : o.N * round128(o.K);
  return bytes;
}

// Makes the copies in ws and points o at them.
int linear_relay(int kind, LinOps* o, void* ws, cudaStream_t st) {
  const int e = kind == TO_F16 || kind == TO_BF16 ? 2 : 1;
  RelayJob job[2] = {};
  int n = 0;
  uint8_t* dst = (uint8_t*)ws;
  auto add = [&](const void* src, int64_t rows, int64_t row_bytes, int64_t pitch) {
    job[n] = RelayJob{(const uint8_t*)src, dst, rows, row_bytes, pitch, round128(row_bytes)};
    dst += rows * job[n].dst_pitch;
    return job[n++].dst;
  };
  if (!aligned_rows(o->a, o->lda * e)) {
    o->a = add(o->a, o->M, o->K * e, o->lda * e);
    o->lda = o->a_k = round128(o->K * e) / e;
  }
  if (!aligned_rows(o->b, o->ldb * e)) {
    const int64_t inner = e == 2 ? o->N : o->K;
    o->b = add(o->b, e == 2 ? o->K : o->N, inner * e, o->ldb * e);
    o->ldb = o->b_in = round128(inner * e) / e;
  }
  if (n == 0) return TO_OK;
  const int64_t cap = (int64_t)sm_count() * 8;
  int blocks[2] = {0, 0};
  for (int i = 0; i < n; ++i)
    blocks[i] = (int)std::min<int64_t>(
        ceil_div(job[i].rows * (job[i].dst_pitch / 16), kRelayThreads * kRelayBatch), cap);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks[0] + blocks[1]), 1, 1);
  cfg.blockDim = dim3(kRelayThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, k_linear_relay, job[0], job[1], blocks[0]);
  if (err != cudaSuccess) return cuda_fail(err, "linear epilogue: operand copies launch");
  return check_launch("linear epilogue: operand copies");
}

}  // namespace tob
