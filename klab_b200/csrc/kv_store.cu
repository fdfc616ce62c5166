// Rows of keys and values into 4-bit pages (store) and back (read): the cache that kv_attn.cu reads. The layout and the
// format are in kv_pages.cuh.
//
// Store: a thread takes 8 dims of one (token, kv head) of K and of V with one 16-byte load each; the 4 threads of a group
// of 32 dims find max|x| on the 16-bit patterns, s = RN16(min(max / 7, 65504)), and each value's code is
// clamp(RNE(x / s), -7, 7) + 8. The quotient: q = x r with r = RN(1 / s), then q += (x - q s) r. It is within an ulp of
// x / s, and exact where x / s is a float, as the ties k + 1/2 are; x has at most 11 significant bits and s 11, so
// |x / s - (k + 1/2)| is 0 or above 2^-13, and RNE(q) is RNE(x / s), ties included. Adding 1.5 * 2^23 + 8 rounds to the
// nearest even whole number and leaves the code in the low bits. Groups whose scale is under FP16's normal range or at its
// end, and those with NaN (counted as 0) or infinities (the largest code), are clamped first. A slot of -1 is skipped.
// Lanes of two neighbouring tokens join their halves of the V words where their slots are a pair (all of a prompt but its
// ends); other tokens write halves.
// Read: the inverse, (code - 8) * s in FP32 (exact) and one rounding to the output's type; a slot of -1 gives zeros.
//
// What bounds them: the bytes, 4 in and 1.125 out per pair of values (store of 16-bit rows), and about 100 instructions a
// thread beside them.
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
  unsigned threads, tokens;
  int num_pages, kv_heads, dim, page_shift, wide;
};

constexpr float kCodeMagic = 12582912.0f + 8.0f;  // 1.5 * 2^23 + 8: adding it leaves round(q) + 8 in the low bits
// Sum over i < 8 of the other bits of 1.5 * 2^23, shifted by 4 i.
constexpr unsigned kCodeExcess = 0x4b400000u + 0xb4000000u + 0x40000000u;

template <bool kBf16>
__device__ __forceinline__ f2 widen2(unsigned w) {
  return kBf16 ? f2{bf16lo(w), bf16hi(w)} : f2{f16lo(w), f16hi(w)};
}

__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  unsigned long long ra, rb, rd;
  asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
  f2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
  return d;
}

// The 8 codes of the values in v and, through `scale`, the group's FP16 scale. Called by all 4 lanes of the group.
template <bool kBf16>
__device__ __forceinline__ unsigned quantize8(uint4 v, unsigned short& scale) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
  constexpr unsigned kInf = kBf16 ? 0x7f80u : 0x7c00u;
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
  most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const unsigned bits = max(most & 0xffffu, most >> 16);
  float top = kBf16 ? __uint_as_float(bits << 16) : f16_to_f32(static_cast<unsigned short>(bits));
  f2 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = widen2<kBf16>(w[i]);
  // Any lane with an odd group sends its warp through the full path, which gives ordinary groups the same codes.
  if (__any_sync(0xffffffffu, bits >= kInf)) {
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (x[i].x != x[i].x) x[i].x = 0.0f;
      if (x[i].y != x[i].y) x[i].y = 0.0f;
      top = fmaxf(top, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  }
  const __half s16 = __float2half_rn(fminf(__fdiv_rn(top, 7.0f), 65504.0f));
  scale = __half_as_ushort(s16);
  const float s = __half2float(s16);
  if (s == 0.0f) return 0x88888888u;
  if (s < 6.103515625e-5f || s >= 65504.0f) {  // x / s may pass 7
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i].x = fminf(fmaxf(x[i].x, -7.0f * s), 7.0f * s);
      x[i].y = fminf(fmaxf(x[i].y, -7.0f * s), 7.0f * s);
    }
  }
  const float r = __frcp_rn(s);
  const f2 r2 = {r, r}, minus = {-s, -s}, magic = {kCodeMagic, kCodeMagic};
  unsigned codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f2 q = mul2(x[i], r2);
    q = fma2(fma2(q, minus, x[i]), r2, q);
    q = add2(q, magic);
    codes += __float_as_uint(q.x) << (8 * i);
    codes += __float_as_uint(q.y) << (8 * i + 4);
  }
  return codes - kCodeExcess;
}

// Token, head and 8-dim run of a thread: runs, then the two tokens of a pair, then heads, then pairs.
struct Place {
  unsigned token;
  int head, c, slot;
  long long block;
};

template <int D>
__device__ __forceinline__ Place place_of(const RowParams& p, unsigned at) {
  Place w;
  constexpr unsigned kRuns = D / 8;
  w.c = at % kRuns;
  const unsigned rest = at / (2 * kRuns), pair = rest / p.kv_heads;
  w.head = rest - pair * p.kv_heads;
  w.token = 2 * pair + at / kRuns % 2;
  w.slot = w.token < p.tokens ? p.slots[w.token] : -1;
  w.block = kv_block_offset(w.slot, w.head, p.num_pages, p.kv_heads, p.page_shift, D);
  if (w.slot != -1 && w.block < 0) record_status(p.status, kStatusBadPage);
  return w;
}

template <bool kBf16, int D>
__global__ void __launch_bounds__(kStoreThreads) kv_store_kernel(const RowParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const unsigned at = blockIdx.x * kStoreThreads + threadIdx.x;
  const Place w = place_of<D>(p, at);  // a thread past the end has a slot of -1 and stays for the shuffles
  uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
  if (w.block >= 0) {
    const long long row = w.token;
    const auto* ks = static_cast<const unsigned short*>(p.k) + row * p.k_stride + w.head * p.k_head + 8 * w.c;
    const auto* vs = static_cast<const unsigned short*>(p.v) + row * p.v_stride + w.head * p.v_head + 8 * w.c;
    if (p.wide) {
      k = ldg128_stream(ks);
      v = ldg128_stream(vs);
    } else {  // rows on 8-byte boundaries
      const uint2 k0 = __ldg(reinterpret_cast<const uint2*>(ks)), k1 = __ldg(reinterpret_cast<const uint2*>(ks) + 1);
      const uint2 v0 = __ldg(reinterpret_cast<const uint2*>(vs)), v1 = __ldg(reinterpret_cast<const uint2*>(vs) + 1);
      k = make_uint4(k0.x, k0.y, k1.x, k1.y);
      v = make_uint4(v0.x, v0.y, v1.x, v1.y);
    }
  }
  unsigned short k_scale, v_scale;
  const unsigned k_codes = quantize8<kBf16>(k, k_scale), v_codes = quantize8<kBf16>(v, v_scale);
  // The other token of the pair: its V codes and slot (heads of 256 take a warp each and write halves).
  constexpr int other = D / 8;
  const unsigned v_other = __shfl_xor_sync(0xffffffffu, v_codes, other & 31);
  const int slot_other = __shfl_xor_sync(0xffffffffu, w.slot, other & 31);
  if (w.block < 0) return;
  unsigned short* to = p.pages + w.block / 2;
  const int r = w.slot & (kKvBlock - 1);
  *reinterpret_cast<unsigned*>(to + kv_k_piece(r, 2 * w.c, D)) = k_codes;
  // Pieces 2 c and 2 c + 1 (dims 8 c .. + 3, 8 c + 4 .. + 7): neighbouring g of one group.
  if (other < 32 && slot_other == (w.slot ^ 1)) {
    if ((w.slot & 1) == 0)
      *reinterpret_cast<unsigned*>(to + kv_v_piece(r, 2 * w.c, D)) = __byte_perm(v_codes, v_other, 0x5410);
    else
      *reinterpret_cast<unsigned*>(to + kv_v_piece(r & ~1, 2 * w.c + 1, D)) = __byte_perm(v_other, v_codes, 0x7632);
  } else {
    to[kv_v_piece(r, 2 * w.c, D)] = static_cast<unsigned short>(v_codes);
    to[kv_v_piece(r, 2 * w.c + 1, D)] = static_cast<unsigned short>(v_codes >> 16);
  }
  if ((w.c & 3) == 0) {
    to[kv_k_scale(r, w.c >> 2, D)] = k_scale;
    to[kv_v_scale(r, w.c >> 2, D)] = v_scale;
  }
}

template <int kOut>
__device__ __forceinline__ void put8(void* out, long long at, unsigned codes, float s) {
  f2 x[4];
  const f2 s2 = {s, s}, back = {-kCodeMagic, -kCodeMagic};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f2 u = {__uint_as_float((codes >> (8 * i) & 15u) | 0x4b400000u),
                  __uint_as_float((codes >> (8 * i + 4) & 15u) | 0x4b400000u)};
    x[i] = mul2(add2(u, back), s2);
  }
  if (kOut == KLAB_DT_F32) {
    float4* to = reinterpret_cast<float4*>(out) + 2 * at;
    to[0] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
    to[1] = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
  } else {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kOut == KLAB_DT_BF16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[i].y), "f"(x[i].x));
      else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[i].y), "f"(x[i].x));
    }
    reinterpret_cast<uint4*>(out)[at] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int kOut, int D>
__global__ void __launch_bounds__(kStoreThreads) kv_read_kernel(const RowParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const unsigned at = blockIdx.x * kStoreThreads + threadIdx.x;
  const Place w = place_of<D>(p, at);
  if (w.token >= p.tokens) return;
  unsigned k_codes = 0x88888888u, v_codes = 0x88888888u;
  float k_scale = 0.0f, v_scale = 0.0f;
  if (w.block >= 0) {
    const unsigned short* from = p.pages + w.block / 2;
    const int r = w.slot & (kKvBlock - 1);
    k_codes = *reinterpret_cast<const unsigned*>(from + kv_k_piece(r, 2 * w.c, D));
    v_codes = from[kv_v_piece(r, 2 * w.c, D)] | static_cast<unsigned>(from[kv_v_piece(r, 2 * w.c + 1, D)]) << 16;
    k_scale = f16_to_f32(from[kv_k_scale(r, w.c >> 2, D)]);
    v_scale = f16_to_f32(from[kv_v_scale(r, w.c >> 2, D)]);
  }
  const long long to = (static_cast<long long>(w.token) * p.kv_heads + w.head) * (D / 8) + w.c;
  put8<kOut>(p.k_out, to, k_codes, k_scale);
  put8<kOut>(p.v_out, to, v_codes, v_scale);
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

template <int kOut>
int launch_read(const RowParams& p, void* stream) {
  switch (p.dim) {
    case 64: return launch_rows(kv_read_kernel<kOut, 64>, p, stream);
    case 128: return launch_rows(kv_read_kernel<kOut, 128>, p, stream);
    default: return launch_rows(kv_read_kernel<kOut, 256>, p, stream);
  }
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
  p.wide = !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15 ||
             (k_stride | v_stride | k_head | v_head) & 7);
  p.pages = static_cast<unsigned short*>(pages);
  p.slots = slots;
  p.status = device_status_address();
  p.num_pages = num_pages;
  p.tokens = static_cast<unsigned>(tokens);
  p.threads = (p.tokens + 1) / 2 * 2 * kv_heads * (dim / 8);
  p.kv_heads = kv_heads;
  p.dim = dim;
  p.page_shift = kv_page_shift(page_size);
  const bool bf16 = dtype == KLAB_DT_BF16;
  switch (dim) {
    case 64: return bf16 ? launch_rows(kv_store_kernel<true, 64>, p, stream) : launch_rows(kv_store_kernel<false, 64>, p, stream);
    case 128: return bf16 ? launch_rows(kv_store_kernel<true, 128>, p, stream) : launch_rows(kv_store_kernel<false, 128>, p, stream);
    default: return bf16 ? launch_rows(kv_store_kernel<true, 256>, p, stream) : launch_rows(kv_store_kernel<false, 256>, p, stream);
  }
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
  p.tokens = static_cast<unsigned>(tokens);
  p.threads = (p.tokens + 1) / 2 * 2 * kv_heads * (dim / 8);
  p.kv_heads = kv_heads;
  p.dim = dim;
  p.page_shift = kv_page_shift(page_size);
  switch (dtype) {
    case KLAB_DT_BF16: return launch_read<KLAB_DT_BF16>(p, stream);
    case KLAB_DT_F16: return launch_read<KLAB_DT_F16>(p, stream);
    case KLAB_DT_F32: return launch_read<KLAB_DT_F32>(p, stream);
    default: return KLAB_E_UNSUPPORTED;
  }
}

}  // extern "C"
