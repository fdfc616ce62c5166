// Low-rank adapters of many requests beside a shared projection:
//   y[m] = x[m] W^T + c_a (x[m] A_a^T) B_a^T,  a = ids[m] (-1: x[m] W^T alone),
// BF16 x, A [S, r, K], B [S, N, r]; W in any format that the projections take with BF16 x and one scale tensor.
//
// shrink_kernel: t[m, j] = c_a * x[m] . A_a[j] in FP32; a CTA takes one token and kRanks rows of its A, its threads share
// K with 16-byte loads. The projection then runs as it is, with FP32 output, and expand_kernel adds t[m] . B_a[n] to it in
// FP32 and rounds once. Every sum has a fixed order.
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"

namespace klab {
namespace {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kRanks = 4;  // rows of A per CTA
constexpr int kMaxRank = 256;

struct AdapterParams {
  const unsigned short* x;
  const unsigned short* a;
  const unsigned short* b;
  const float* c;
  const int* ids;
  float* t;         // [m, rank]
  const float* y0;  // [m, n] the projection
  void* out;
  int* status;
  int m, n, k, rank, adapters, ldo, out_f32;
};

__device__ __forceinline__ void fma8(uint4 x, uint4 w, float& s0, float& s1) {
  s0 = fma_rn(bf16lo(x.x), bf16lo(w.x), s0), s1 = fma_rn(bf16hi(x.x), bf16hi(w.x), s1);
  s0 = fma_rn(bf16lo(x.y), bf16lo(w.y), s0), s1 = fma_rn(bf16hi(x.y), bf16hi(w.y), s1);
  s0 = fma_rn(bf16lo(x.z), bf16lo(w.z), s0), s1 = fma_rn(bf16hi(x.z), bf16hi(w.z), s1);
  s0 = fma_rn(bf16lo(x.w), bf16lo(w.w), s0), s1 = fma_rn(bf16hi(x.w), bf16hi(w.w), s1);
}

__global__ void __launch_bounds__(kAdThreads) shrink_kernel(const AdapterParams p) {
  __shared__ float part[kAdWarps][kRanks];
  grid_dependency_wait();
  grid_launch_dependents();
  const int m = blockIdx.y, j0 = blockIdx.x * kRanks;  // rank is a multiple of 8
  const int id = p.ids[m];
  if (id < 0 || id >= p.adapters) {
    if (id != -1 && threadIdx.x == 0 && blockIdx.x == 0) record_status(p.status, kStatusBadAdapter);
    return;
  }
  const uint4* x = reinterpret_cast<const uint4*>(p.x + static_cast<long long>(m) * p.k);
  const uint4* a[kRanks];
#pragma unroll
  for (int j = 0; j < kRanks; ++j)
    a[j] = reinterpret_cast<const uint4*>(p.a + (static_cast<long long>(id) * p.rank + j0 + j) * p.k);
  float s0[kRanks] = {}, s1[kRanks] = {};
  const int chunks = p.k / 8;
#pragma unroll 2
  for (int i = threadIdx.x; i < chunks; i += kAdThreads) {
    const uint4 xv = __ldg(x + i);
    uint4 av[kRanks];
#pragma unroll
    for (int j = 0; j < kRanks; ++j) av[j] = ldg128_stream(a[j] + i);
#pragma unroll
    for (int j = 0; j < kRanks; ++j) fma8(xv, av[j], s0[j], s1[j]);
  }
#pragma unroll
  for (int j = 0; j < kRanks; ++j) {
    const float s = warp_allsum(add_rn(s0[j], s1[j]));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = s;
  }
  __syncthreads();
  if (threadIdx.x < kRanks) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kAdWarps; ++w) s = add_rn(s, part[w][threadIdx.x]);
    p.t[m * p.rank + j0 + threadIdx.x] = mul_rn(s, p.c[id]);
  }
}

__global__ void __launch_bounds__(kAdThreads) expand_kernel(const AdapterParams p) {
  __shared__ float t[kMaxRank];
  grid_dependency_wait();
  grid_launch_dependents();
  const int m = blockIdx.y, n = blockIdx.x * kAdThreads + threadIdx.x;
  const int id = p.ids[m];
  const bool has = id >= 0 && id < p.adapters;
  if (has)
    for (int j = threadIdx.x; j < p.rank; j += kAdThreads) t[j] = p.t[m * p.rank + j];
  __syncthreads();
  if (n >= p.n) return;
  float y = p.y0[static_cast<long long>(m) * p.n + n];
  if (has) {
    const uint4* b = reinterpret_cast<const uint4*>(p.b + (static_cast<long long>(id) * p.n + n) * p.rank);
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll 4
    for (int j = 0; j < p.rank / 8; ++j) {
      const uint4 w = __ldg(b + j);
      const float* tj = t + 8 * j;
      s0 = fma_rn(tj[0], bf16lo(w.x), s0), s1 = fma_rn(tj[1], bf16hi(w.x), s1);
      s0 = fma_rn(tj[2], bf16lo(w.y), s0), s1 = fma_rn(tj[3], bf16hi(w.y), s1);
      s0 = fma_rn(tj[4], bf16lo(w.z), s0), s1 = fma_rn(tj[5], bf16hi(w.z), s1);
      s0 = fma_rn(tj[6], bf16lo(w.w), s0), s1 = fma_rn(tj[7], bf16hi(w.w), s1);
    }
    y = add_rn(y, add_rn(s0, s1));
  }
  const long long at = static_cast<long long>(m) * p.ldo + n;
  if (p.out_f32)
    static_cast<float*>(p.out)[at] = y;
  else
    static_cast<unsigned short*>(p.out)[at] = f32_to_bf16_rn(y);
}

template <typename Kernel>
int launch_adapter(Kernel kernel, dim3 grid, const AdapterParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kAdThreads);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = klab_get_option(KLAB_OPT_PDL) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace
}  // namespace klab

extern "C" {

KLAB_API long long klab_adapter_scratch(int m, int n, int rank) {
  if (m <= 0 || n <= 0 || rank <= 0) return KLAB_E_INVALID;
  const long long t = (static_cast<long long>(m) * rank * 4 + 127) / 128 * 128;
  return t + static_cast<long long>(m) * n * 4;
}

KLAB_API int klab_adapter_linear(int wfmt, const void* x, const void* w, const void* aux, const void* a, const void* b,
                                 const float* c, const int* ids, void* out, int out_dtype, int m, int n, int k, int rank,
                                 int adapters, void* scratch, long long scratch_bytes, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  using namespace klab;
  if (!x || !w || !a || !b || !c || !ids || !out || !scratch || m <= 0 || n <= 0 || k <= 0 || rank <= 0 || adapters <= 0)
    return KLAB_E_INVALID;
  if (wfmt != KLAB_W_BF16 && wfmt != KLAB_W_CBF16 && wfmt != KLAB_W_I8_ROW && wfmt != KLAB_W_I8_G64 &&
      wfmt != KLAB_W_FP4_G32H)
    return KLAB_E_UNSUPPORTED;
  if (out_dtype != KLAB_DT_BF16 && out_dtype != KLAB_DT_F32) return KLAB_E_UNSUPPORTED;
  if (rank % 8 || rank > kMaxRank || k % 8 || m > 65535) return KLAB_E_SHAPE;
  const uintptr_t mis = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) |
                        reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(scratch);
  if (mis & 15) return KLAB_E_ALIGN;
  if (scratch_bytes < klab_adapter_scratch(m, n, rank)) return KLAB_E_INVALID;
  AdapterParams p{};
  p.x = static_cast<const unsigned short*>(x);
  p.a = static_cast<const unsigned short*>(a);
  p.b = static_cast<const unsigned short*>(b);
  p.c = c;
  p.ids = ids;
  p.t = static_cast<float*>(scratch);
  float* y0 = p.t + (static_cast<long long>(m) * rank * 4 + 127) / 128 * 32;
  p.y0 = y0;
  p.out = out;
  p.status = device_status_address();
  p.m = m;
  p.n = n;
  p.k = k;
  p.rank = rank;
  p.adapters = adapters;
  p.ldo = n;
  p.out_f32 = out_dtype == KLAB_DT_F32;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc = launch_adapter(shrink_kernel, dim3(rank / kRanks, m), p, s);
  if (rc) return rc;
  rc = klab_gemv(wfmt, KLAB_DT_BF16, x, k, w, aux, nullptr, y0, n, KLAB_DT_F32, m, n, k, workspace, workspace_bytes,
                 stream);
  if (rc) return rc;
  return launch_adapter(expand_kernel, dim3((n + kAdThreads - 1) / kAdThreads, m), p, s);
}

}  // extern "C"
