// Rows of keys and values into 4-bit pages (store) and back (read): the cache that kv_attn.cu reads. The layout and the
// format are in kv_pages.cuh.
//
// Store: a thread takes 4 dims of one (token, kv head) of K and of V with one 8-byte load each; the 8 threads of a
// group of 32 dims find max|x| by a butterfly, s = RN16(min(max / 7, 65504)), and each value's code is
// clamp(RNE(x / s), -7, 7) + 8 with x / s the correctly rounded quotient, so the codes are those of the definition, ties
// included (x has at most 11 significant bits and s 11, hence |x / s - (k + 1/2)| is 0 or above 2^-13, far beyond the
// quotient's rounding). NaN counts as 0; an infinity takes the largest code. A slot of -1 is skipped.
// Read: the inverse, (code - 8) * s in FP32 (exact) and one rounding to the output's type; a slot of -1 gives zeros.
//
// What bounds them: the bytes, 4 in and 1.125 out per pair of values (store of 16-bit rows).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"
#include "kv_pages.cuh"

namespace klab {
namespace {

constexpr int kStoreThreads = 256;

struct RowParams {
  const void* k;
  const void* v;
  long long k_stride, v_stride, k_head, v_head;  // elements between tokens and between heads
  unsigned short* pages;
  const int* slots;
  void* k_out;
  void* v_out;
  int* status;
  unsigned threads;
  int num_pages, kv_heads, dim, page_shift;
};

template <bool kBf16>
__device__ __forceinline__ void widen4(uint2 w, float (&x)[4]) {
  if (kBf16) {
    x[0] = bf16lo(w.x), x[1] = bf16hi(w.x), x[2] = bf16lo(w.y), x[3] = bf16hi(w.y);
  } else {
    x[0] = f16lo(w.x), x[1] = f16hi(w.x), x[2] = f16lo(w.y), x[3] = f16hi(w.y);
  }
}

// The 4 codes of x and, through `scale`, the group's FP16 scale. Called by all 8 lanes of the group.
__device__ __forceinline__ unsigned short quantize4(float (&x)[4], unsigned short& scale) {
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (x[e] != x[e]) x[e] = 0.0f;
    top = fmaxf(top, fabsf(x[e]));
  }
#pragma unroll
  for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const __half s16 = __float2half_rn(fminf(__fdiv_rn(top, 7.0f), 65504.0f));
  scale = __half_as_ushort(s16);
  const float s = __half2float(s16);
  unsigned piece = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float code = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(x[e], s)), -7.0f), 7.0f) : 0.0f;
    piece |= static_cast<unsigned>(static_cast<int>(code) + 8) << (4 * e);
  }
  return static_cast<unsigned short>(piece);
}

template <bool kBf16>
__global__ void __launch_bounds__(kStoreThreads) kv_store_kernel(const RowParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const unsigned at = blockIdx.x * kStoreThreads + threadIdx.x;
  const unsigned per_head = p.dim / 4, per_token = per_head * p.kv_heads;
  const unsigned token = at / per_token, rest = at - token * per_token;
  const int head = rest / per_head, c = rest - head * per_head;
  // A thread past the end stays for the groups' butterflies.
  const int slot = at < p.threads ? p.slots[token] : -1;
  const long long block = kv_block_offset(slot, head, p.num_pages, p.kv_heads, p.page_shift, p.dim);
  if (slot != -1 && block < 0) record_status(p.status, kStatusBadPage);
  float k[4] = {}, v[4] = {};
  if (block >= 0) {
    const auto* ks = static_cast<const unsigned short*>(p.k) + token * p.k_stride + head * p.k_head + 4 * c;
    const auto* vs = static_cast<const unsigned short*>(p.v) + token * p.v_stride + head * p.v_head + 4 * c;
    widen4<kBf16>(__ldg(reinterpret_cast<const uint2*>(ks)), k);
    widen4<kBf16>(__ldg(reinterpret_cast<const uint2*>(vs)), v);
  }
  unsigned short k_scale, v_scale;
  const unsigned short k_piece = quantize4(k, k_scale), v_piece = quantize4(v, v_scale);
  if (block < 0) return;
  unsigned short* to = p.pages + block / 2;
  const int r = slot & (kKvBlock - 1);
  to[kv_k_piece(r, c, p.dim)] = k_piece;
  to[kv_v_piece(r, c, p.dim)] = v_piece;
  if ((c & 7) == 0) {
    to[kv_k_scale(r, c >> 3, p.dim)] = k_scale;
    to[kv_v_scale(r, c >> 3, p.dim)] = v_scale;
  }
}

template <int kOut>
__device__ __forceinline__ void put4(void* out, unsigned at, unsigned piece, float s) {
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(static_cast<int>(piece >> (4 * e) & 15u) - 8) * s;
  if (kOut == KLAB_DT_F32) {
    reinterpret_cast<float4*>(out)[at] = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    unsigned w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (kOut == KLAB_DT_BF16)
        w[e] = f32_to_bf16_rn(x[2 * e]) | static_cast<unsigned>(f32_to_bf16_rn(x[2 * e + 1])) << 16;
      else
        w[e] = __half_as_ushort(__float2half_rn(x[2 * e])) |
               static_cast<unsigned>(__half_as_ushort(__float2half_rn(x[2 * e + 1]))) << 16;
    }
    reinterpret_cast<uint2*>(out)[at] = make_uint2(w[0], w[1]);
  }
}

template <int kOut>
__global__ void __launch_bounds__(kStoreThreads) kv_read_kernel(const RowParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const unsigned at = blockIdx.x * kStoreThreads + threadIdx.x;
  if (at >= p.threads) return;
  const unsigned per_head = p.dim / 4, per_token = per_head * p.kv_heads;
  const unsigned token = at / per_token, rest = at - token * per_token;
  const int head = rest / per_head, c = rest - head * per_head;
  const int slot = p.slots[token];
  const long long block = kv_block_offset(slot, head, p.num_pages, p.kv_heads, p.page_shift, p.dim);
  unsigned k_piece = 0x8888u, v_piece = 0x8888u;
  float k_scale = 0.0f, v_scale = 0.0f;
  if (block >= 0) {
    const unsigned short* from = p.pages + block / 2;
    const int r = slot & (kKvBlock - 1);
    k_piece = from[kv_k_piece(r, c, p.dim)];
    v_piece = from[kv_v_piece(r, c, p.dim)];
    k_scale = f16_to_f32(from[kv_k_scale(r, c >> 3, p.dim)]);
    v_scale = f16_to_f32(from[kv_v_scale(r, c >> 3, p.dim)]);
  } else if (slot != -1) {
    record_status(p.status, kStatusBadPage);
  }
  put4<kOut>(p.k_out, at, k_piece, k_scale);
  put4<kOut>(p.v_out, at, v_piece, v_scale);
}

int check_pages(const void* pages, const void* slots, int tokens, int num_pages, int page_size, int kv_heads, int dim) {
  if (!pages || !slots || tokens <= 0 || num_pages <= 0 || kv_heads <= 0) return KLAB_E_INVALID;
  if (!kv_page_size_ok(page_size) || !kv_dim_ok(dim) || static_cast<long long>(num_pages) * page_size > INT_MAX)
    return KLAB_E_SHAPE;
  if (static_cast<long long>(tokens) * kv_heads * (dim / 4) > INT_MAX) return KLAB_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(pages) & 15) return KLAB_E_ALIGN;
  return 0;
}

template <typename Kernel>
int launch_rows(Kernel kernel, const RowParams& p, void* stream) {
  const unsigned blocks = (p.threads + kStoreThreads - 1) / kStoreThreads;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kStoreThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = klab_get_option(KLAB_OPT_PDL) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace
}  // namespace klab

extern "C" {

KLAB_API long long klab_kv_block_offset(int slot, int head, int num_pages, int kv_heads, int page_size, int dim) {
  using namespace klab;
  if (!kv_page_size_ok(page_size) || !kv_dim_ok(dim) || num_pages <= 0 || kv_heads <= 0 || head < 0 || head >= kv_heads)
    return -1;
  return kv_block_offset(slot, head, num_pages, kv_heads, kv_page_shift(page_size), dim);
}

KLAB_API int klab_kv_store(const void* k, const void* v, int dtype, long long k_stride, long long v_stride,
                           long long k_head, long long v_head, void* pages, const int* slots, int tokens, int num_pages,
                           int page_size, int kv_heads, int dim, void* stream) {
  using namespace klab;
  if (!k || !v) return KLAB_E_INVALID;
  int rc = check_pages(pages, slots, tokens, num_pages, page_size, kv_heads, dim);
  if (rc) return rc;
  if (dtype != KLAB_DT_BF16 && dtype != KLAB_DT_F16) return KLAB_E_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 7 ||
      (k_stride | v_stride | k_head | v_head) & 3)
    return KLAB_E_ALIGN;
  RowParams p = {};
  p.k = k;
  p.v = v;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.k_head = k_head;
  p.v_head = v_head;
  p.pages = static_cast<unsigned short*>(pages);
  p.slots = slots;
  p.status = device_status_address();
  p.num_pages = num_pages;
  p.threads = static_cast<unsigned>(tokens) * kv_heads * (dim / 4);
  p.kv_heads = kv_heads;
  p.dim = dim;
  p.page_shift = kv_page_shift(page_size);
  return dtype == KLAB_DT_BF16 ? launch_rows(kv_store_kernel<true>, p, stream)
                               : launch_rows(kv_store_kernel<false>, p, stream);
}

KLAB_API int klab_kv_read(const void* pages, const int* slots, void* k_out, void* v_out, int dtype, int tokens,
                          int num_pages, int page_size, int kv_heads, int dim, void* stream) {
  using namespace klab;
  if (!k_out || !v_out) return KLAB_E_INVALID;
  int rc = check_pages(pages, slots, tokens, num_pages, page_size, kv_heads, dim);
  if (rc) return rc;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return KLAB_E_ALIGN;
  RowParams p = {};
  p.pages = static_cast<unsigned short*>(const_cast<void*>(pages));
  p.slots = slots;
  p.k_out = k_out;
  p.v_out = v_out;
  p.status = device_status_address();
  p.num_pages = num_pages;
  p.threads = static_cast<unsigned>(tokens) * kv_heads * (dim / 4);
  p.kv_heads = kv_heads;
  p.dim = dim;
  p.page_shift = kv_page_shift(page_size);
  switch (dtype) {
    case KLAB_DT_BF16: return launch_rows(kv_read_kernel<KLAB_DT_BF16>, p, stream);
    case KLAB_DT_F16: return launch_rows(kv_read_kernel<KLAB_DT_F16>, p, stream);
    case KLAB_DT_F32: return launch_rows(kv_read_kernel<KLAB_DT_F32>, p, stream);
    default: return KLAB_E_UNSUPPORTED;
  }
}

}  // extern "C"
