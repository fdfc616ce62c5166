// Rows of keys and values into 4-bit pages (store) and back (read): the cache that kv_attn.cu reads. The layout and the
// format are in kv_pages.cuh.
//
// Store: lanes hold 8 dims of a group each (16-byte loads), and the 4 lanes of a group of 32 find max|x| on the 16-bit
// patterns, s = RN16(min(max / 7, 65504)), and each value's code, clamp(RNE(x / s), -7, 7) + 8. With r within an ulp of
// 1 / s, fma(x, r, 1.5 * 2^8) rounds x r to a multiple of 2^-15 and is within 2^-15 of x / s; x and s have at most 11
// significant bits, so |x / s - (k + 1/2)| is 0 or above 2^-13, and what is rounded then to a whole number (nearest, ties to
// even, by adding 1.5 * 2^23 + 8 - 1.5 * 2^8, which leaves the code in the low bits) is RNE(x / s), ties included. In the
// same way max * RN(1 / 7) rounds to the FP16 value that max / 7 does where that is normal: 7 n = 2^j m has no solution for
// an odd n of 12 bits and m of 11, so max / 7 keeps 2^-15 of itself from every tie. Groups whose scale is under FP16's
// normal range or near its end, and those with NaN (counted as 0) or infinities (the largest code), take a longer way with
// a division and clamps, together with the rest of their warp. A slot of -1 is skipped.
//   Few rows: a thread takes 8 dims of K and of V of one token; lanes of two neighbouring tokens join their halves of the V
//   words where their slots are a pair (all of a prompt but its ends); other tokens write halves.
//   Many rows: a thread takes two tokens and 8 dims of each of the 4 groups of a quad (read: 2 at heads of 64): K codes, V codes
//   of a pair of slots and scales are then whole runs of 16 bytes of a block, and the addresses are worked out once for 128
//   values. (Single runs are bound by issue slots there.)
// Read: the inverse, (code - 8) * s in FP32 (exact) and one rounding to the output's type; a slot of -1 gives zeros.
//
// What bounds them: few rows launch and three dependent loads; many rows the bytes, 4 in and 1.125 out per pair of values
// (16384 tokens of 8 heads of 128: store 18.0 us, 4.8 TB/s; read 15.8 us, 5.4 TB/s), in store with loads that 16 warps an SM
// (96 registers) keep too few of in flight, and issue slots 50 % busy.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"
#include "kv_pages.cuh"
#include "launch.cuh"

namespace klab {
namespace {

constexpr int kStoreThreads = 256, kBulkThreads = 128;
// 8-dim runs of K (and of V) from which a thread takes runs of Q groups of two tokens. Read: 1024 tokens of 8 heads of 128
// take 2.5 us either way, 64 take 1.6 us by single runs and 2.3 in bulk, 16384 18.1 and 14.9. Store, of a prompt: 1024
// tokens 2.8 us by single runs and 3.0 in bulk, 4096 6.7 and 6.2, 8192 12.0 and 9.2, 16384 22.5 and 17.4; where no two
// tokens share words of V (one token of each of many requests) 4096 6.4 and 9.4, 16384 22.7 and 24.8; heads of 64 only by
// single runs (16384 tokens 12.3 us and 11.4, but 13.5 and 18.5 where no two tokens share words).
constexpr long long kReadBulkRuns = 128 * 1024, kStoreBulkRuns = 512 * 1024;

struct RowParams {
  const void* k;
  const void* v;
  long long k_stride, v_stride, k_head, v_head;  // elements between tokens and between heads
  unsigned short* pages;
  const int* slots;
  void* k_out;
  void* v_out;
  int* status;
  unsigned tokens;
  int num_pages, kv_heads, dim, page_shift, wide;
};

constexpr float kGridMagic = 384.0f;              // 1.5 * 2^8: a sum with it lies on multiples of 2^-15
constexpr float kCodeMagic = 12582912.0f + 8.0f;  // 1.5 * 2^23 + 8: adding it leaves round(q) + 8 in the low bits
// Sum over i < 8 of the other bits of 1.5 * 2^23, shifted by 4 i.
constexpr unsigned kCodeExcess = 0x4b400000u + 0xb4000000u + 0x40000000u;

template <bool kBf16>
__device__ __forceinline__ f2 widen2(unsigned w) {
  return kBf16 ? f2{bf16lo(w), bf16hi(w)} : f2{f16lo(w), f16hi(w)};
}

template <bool kBf16>
__device__ __forceinline__ void widen8(uint4 v, f2 (&x)[4]) {
  x[0] = widen2<kBf16>(v.x);
  x[1] = widen2<kBf16>(v.y);
  x[2] = widen2<kBf16>(v.z);
  x[3] = widen2<kBf16>(v.w);
}

// max|x| of the lane's 8 values in each half's lanes, as 16-bit patterns; NaN is the largest.
template <bool kBf16>
__device__ __forceinline__ unsigned most8(uint4 v) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
  unsigned most = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 4; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
  return most;
}

// Codes of 8 values with |x| <= 7 (1 + 2^-11) s, s an FP16 value above 0.
__device__ __forceinline__ unsigned codes8(const f2 (&x)[4], float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  const f2 r2 = {r, r}, grid = {kGridMagic, kGridMagic}, magic = {kCodeMagic - kGridMagic, kCodeMagic - kGridMagic};
  unsigned codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f2 q = add2(fma2(x[i], r2, grid), magic);
    codes += __float_as_uint(q.x) << (8 * i);
    codes += __float_as_uint(q.y) << (8 * i + 4);
  }
  return codes - kCodeExcess;
}

// Any group: the 8 codes of the values in v and, through `scale`, the FP16 scale. Called by all 4 lanes of the group.
template <bool kBf16>
__device__ __forceinline__ unsigned quantize8(uint4 v, unsigned short& scale) {
  constexpr unsigned kInf = kBf16 ? 0x7f80u : 0x7c00u;
  unsigned most = most8<kBf16>(v);
  most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const unsigned bits = max(most & 0xffffu, most >> 16);
  float top = kBf16 ? __uint_as_float(bits << 16) : f16_to_f32(static_cast<unsigned short>(bits));
  f2 x[4];
  widen8<kBf16>(v, x);
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
  return codes8(x, s);
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
      k = __ldcs(reinterpret_cast<const uint4*>(ks));
      v = __ldcs(reinterpret_cast<const uint4*>(vs));
    } else {  // rows on 8-byte boundaries
      const uint2 k0 = *reinterpret_cast<const uint2*>(ks), k1 = *(reinterpret_cast<const uint2*>(ks) + 1);
      const uint2 v0 = *reinterpret_cast<const uint2*>(vs), v1 = *(reinterpret_cast<const uint2*>(vs) + 1);
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

// Word u of a run of Q 16- or 32-bit words.
template <int Q>
struct alignas(4 * Q) Words {
  unsigned w[Q];
};

// A thread's place among many rows: a pair of tokens, a head and 8 dims (8 t .. 8 t + 7) of each of a quad's Q groups.
struct Pair {
  int head, t, quad;
  unsigned token[2];
  int slot[2];  // -1: skipped
};

template <int D>
__device__ __forceinline__ Pair pair_of(const RowParams& p, unsigned at) {
  constexpr int kQuads = D == 256 ? 2 : 1;
  Pair w;
  w.t = at % 4;
  w.quad = at / 4 % kQuads;
  const unsigned rest = at / (4 * kQuads), pair = rest / p.kv_heads;
  w.head = rest - pair * p.kv_heads;
#pragma unroll
  for (int i = 0; i < 2; ++i) w.token[i] = 2 * pair + i;
  return w;
}

__device__ __forceinline__ int slot_of(const RowParams& p, unsigned token) {
  return token < p.tokens ? p.slots[token] : -1;
}

template <int D>
__device__ __forceinline__ long long block_of(const RowParams& p, int head, int slot) {
  const long long block = kv_block_offset(slot, head, p.num_pages, p.kv_heads, p.page_shift, D);
  if (slot != -1 && block < 0) record_status(p.status, kStatusBadPage);
  return block;
}

// Codes and scales of both tokens' Q groups. Ordinary groups have a scale in FP16's normal range, below its end; when a
// warp meets another, all of its groups go the way that holds for any.
template <bool kBf16, int Q>
__device__ __forceinline__ void quantize_pair(const uint4 (&x)[2][Q], unsigned (&codes)[2][Q], unsigned short (&scales)[2][Q]) {
  constexpr unsigned kLow = kBf16 ? 0x3a00u : 0x1000u;   // 2^-11: scales of 7 * 10^-5
  constexpr unsigned kHigh = kBf16 ? 0x4880u : 0x7c00u;  // 2^18: scales of 37449
  unsigned most[Q], top = 0, low = 0xffffffffu;
#pragma unroll
  for (int u = 0; u < Q; ++u) {
    const unsigned m0 = most8<kBf16>(x[0][u]), m1 = most8<kBf16>(x[1][u]);
    most[u] = __vmaxu2(__byte_perm(m0, m1, 0x5410), __byte_perm(m0, m1, 0x7632));  // token 0 low, token 1 high
    most[u] = __vmaxu2(most[u], __shfl_xor_sync(0xffffffffu, most[u], 1));
    most[u] = __vmaxu2(most[u], __shfl_xor_sync(0xffffffffu, most[u], 2));
    top = __vmaxu2(top, most[u]);
    low = __vminu2(low, most[u]);
  }
  const bool odd = max(top & 0xffffu, top >> 16) >= kHigh || min(low & 0xffffu, low >> 16) < kLow;
  if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < Q; ++u) codes[i][u] = quantize8<kBf16>(x[i][u], scales[i][u]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      const f2 m = widen2<kBf16>(most[u]);
      const __half s = __float2half_rn((i ? m.y : m.x) * (1.0f / 7.0f));
      scales[i][u] = __half_as_ushort(s);
      f2 v[4];
      widen8<kBf16>(x[i][u], v);
      codes[i][u] = codes8(v, __half2float(s));
    }
}

template <int D, int Q>
__device__ __forceinline__ void read_rows(const void* from, long long stride, long long head, const RowParams& p, const Pair& w,
                                          uint4 (&x)[2][Q]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto* row = static_cast<const unsigned short*>(from) + w.token[i] * stride + w.head * head + 128 * w.quad + 8 * w.t;
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      x[i][u] = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);  // skipped: any ordinary value
      if (w.slot[i] == -1) continue;
      if (p.wide) {
        x[i][u] = __ldcs(reinterpret_cast<const uint4*>(row + 32 * u));
      } else {  // rows on 8-byte boundaries
        const uint2* half = reinterpret_cast<const uint2*>(row + 32 * u);
        const uint2 a = half[0], b = half[1];
        x[i][u] = make_uint4(a.x, a.y, b.x, b.y);
      }
    }
  }
}

// Turns a 4 x 4 matrix over the lanes of a group: lane t's words are those of its 8 dims by group; after it, lane t has
// group t, word j from lane j. All lanes of the warp call it.
__device__ __forceinline__ void turn(unsigned (&w)[4], int t) {
#pragma unroll
  for (int u = 0; u < 4; u += 2) {
    const unsigned got = __shfl_xor_sync(0xffffffffu, t & 1 ? w[u] : w[u + 1], 1);
    (t & 1 ? w[u] : w[u + 1]) = got;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const unsigned got = __shfl_xor_sync(0xffffffffu, t & 2 ? w[u] : w[u + 2], 2);
    (t & 2 ? w[u] : w[u + 2]) = got;
  }
}

template <bool kBf16, int D>
__global__ void __launch_bounds__(kBulkThreads, 5) kv_store_bulk_kernel(const RowParams p) {
  constexpr int Q = 4;
  grid_dependency_wait();
  grid_launch_dependents();
  Pair w = pair_of<D>(p, blockIdx.x * kBulkThreads + threadIdx.x);  // past the end: no slots, stays for the shuffles
  // Tokens whose slots are a pair, even and odd, lie in the same words of V and are stored by one thread. A thread has the
  // pairs that begin at its two tokens and those of the two that are in no pair: one pass, and a second one where its first
  // token stands alone and a pair begins at its second (a prompt of odd length before one that begins at an even slot).
  const unsigned first = w.token[0];
  const int before = first > 0 ? slot_of(p, first - 1) : -1, s0 = slot_of(p, first), s1 = slot_of(p, first + 1),
            after = slot_of(p, first + 2);
  const auto begins = [](int a, int b) { return a >= 0 && a % 2 == 0 && b == a + 1; };
  const bool ended = begins(before, s0), next = begins(s1, after);
  bool joined = begins(s0, s1), again = false;
  w.slot[0] = ended ? -1 : s0;
  w.slot[1] = s1;
  if (next) {
    again = w.slot[0] != -1;
    joined = !again;
    w.slot[1] = again ? -1 : after;
    if (!again) w.slot[0] = s1, w.token[0] = first + 1, w.token[1] = first + 2;
  }
  while (true) {
    uint4 x[2][Q], y[2][Q];
    read_rows<D, Q>(p.k, p.k_stride, p.k_head, p, w, x);
    read_rows<D, Q>(p.v, p.v_stride, p.v_head, p, w, y);
    unsigned short* to[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long block = block_of<D>(p, w.head, w.slot[i]);
      to[i] = block < 0 ? nullptr : p.pages + block / 2;
    }
    unsigned codes[2][Q];
    unsigned short scales[2][Q];
    quantize_pair<kBf16, Q>(x, codes, scales);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!to[i]) continue;
      const int r = w.slot[i] & (kKvBlock - 1);
      Words<Q> c;
#pragma unroll
      for (int u = 0; u < Q; ++u) c.w[u] = codes[i][u];
      *reinterpret_cast<Words<Q>*>(to[i] + kv_k_piece(r, 32 * w.quad + 2 * w.t, D)) = c;
      if (w.t == 0) {
        Words<Q / 2> s;
#pragma unroll
        for (int u = 0; u < Q / 2; ++u) s.w[u] = scales[i][2 * u] | static_cast<unsigned>(scales[i][2 * u + 1]) << 16;
        *reinterpret_cast<Words<Q / 2>*>(to[i] + kv_k_scale(r, 4 * w.quad, D)) = s;
      }
    }
    quantize_pair<kBf16, Q>(y, codes, scales);
    if (joined && to[0]) {
      const int r = w.slot[0] & (kKvBlock - 1);
      Words<Q> lo, hi, s;
#pragma unroll
      for (int u = 0; u < Q; ++u) {
        lo.w[u] = __byte_perm(codes[0][u], codes[1][u], 0x5410);
        hi.w[u] = __byte_perm(codes[0][u], codes[1][u], 0x7632);
        s.w[u] = scales[0][u] | static_cast<unsigned>(scales[1][u]) << 16;
      }
      // Pieces 2 t and 2 t + 1 of a group (dims 8 t .. + 3, 8 t + 4 .. + 7): neighbouring g.
      *reinterpret_cast<Words<Q>*>(to[0] + kv_v_piece(r, 32 * w.quad + 2 * w.t, D)) = lo;
      *reinterpret_cast<Words<Q>*>(to[0] + kv_v_piece(r, 32 * w.quad + 2 * w.t + 1, D)) = hi;
      if (w.t == 0) *reinterpret_cast<Words<Q>*>(to[0] + kv_v_scale(r, 4 * w.quad, D)) = s;
    }
    if (__any_sync(0xffffffffu, !joined)) {  // halves of words: a lane takes one group, so that lanes share sectors
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        turn(codes[i], w.t);
        if (joined || !to[i]) continue;
        const int r = w.slot[i] & (kKvBlock - 1), group = 4 * w.quad + w.t;
#pragma unroll
        for (int j = 0; j < Q; ++j) {
          const int c = 8 * group + 2 * j;
          to[i][kv_v_piece(r, c, D)] = static_cast<unsigned short>(codes[i][j]);
          to[i][kv_v_piece(r, c + 1, D)] = static_cast<unsigned short>(codes[i][j] >> 16);
        }
        unsigned short scale = scales[i][0];  // the group's
#pragma unroll
        for (int u = 1; u < Q; ++u)
          if (w.t == u) scale = scales[i][u];
        to[i][kv_v_scale(r, group, D)] = scale;
      }
    }
    if (!__any_sync(0xffffffffu, again)) return;
    w.token[0] = first + 1, w.token[1] = first + 2;
    w.slot[0] = again ? s1 : -1, w.slot[1] = again ? after : -1;
    joined = true, again = false;
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

template <int kOut, int D>
__global__ void __launch_bounds__(kBulkThreads) kv_read_bulk_kernel(const RowParams p) {
  constexpr int Q = D / 32 < 4 ? D / 32 : 4;
  grid_dependency_wait();
  grid_launch_dependents();
  const Pair w = pair_of<D>(p, blockIdx.x * kBulkThreads + threadIdx.x);
  const int slots[2] = {slot_of(p, w.token[0]), slot_of(p, w.token[1])};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (w.token[i] >= p.tokens) return;
    const long long block = block_of<D>(p, w.head, slots[i]);
    Words<Q> k, lo, hi, vs;
    Words<Q / 2> ks;
#pragma unroll
    for (int u = 0; u < Q; ++u) k.w[u] = lo.w[u] = hi.w[u] = 0x88888888u, vs.w[u] = ks.w[u / 2] = 0u;
    const int r = slots[i] & (kKvBlock - 1);
    if (block >= 0) {
      const unsigned short* from = p.pages + block / 2;
      k = *reinterpret_cast<const Words<Q>*>(from + kv_k_piece(r, 32 * w.quad + 2 * w.t, D));
      ks = *reinterpret_cast<const Words<Q / 2>*>(from + kv_k_scale(r, 4 * w.quad, D));
      lo = *reinterpret_cast<const Words<Q>*>(from + kv_v_piece(r & ~1, 32 * w.quad + 2 * w.t, D));
      hi = *reinterpret_cast<const Words<Q>*>(from + kv_v_piece(r & ~1, 32 * w.quad + 2 * w.t + 1, D));
      vs = *reinterpret_cast<const Words<Q>*>(from + kv_v_scale(r & ~1, 4 * w.quad, D));
    }
    const unsigned half = r & 1 ? 0x7632u : 0x5410u;
    const long long to = (static_cast<long long>(w.token[i]) * p.kv_heads + w.head) * (D / 8) + 16 * w.quad + w.t;
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      put8<kOut>(p.k_out, to + 4 * u, k.w[u], f16_to_f32(static_cast<unsigned short>(ks.w[u / 2] >> (u % 2 * 16))));
      put8<kOut>(p.v_out, to + 4 * u, __byte_perm(lo.w[u], hi.w[u], half),
                 f16_to_f32(static_cast<unsigned short>(vs.w[u] >> (r % 2 * 16))));
    }
  }
}

int check_pages(const void* pages, const void* slots, int tokens, int num_pages, int page_size, int kv_heads, int dim) {
  if (!pages || !slots || tokens <= 0 || num_pages <= 0 || kv_heads <= 0) return KLAB_E_INVALID;
  if (!kv_page_size_ok(page_size) || !kv_dim_ok(dim) || static_cast<long long>(num_pages) * page_size > INT_MAX)
    return KLAB_E_SHAPE;
  if (static_cast<long long>(tokens) * kv_heads * (dim / 4) > INT_MAX) return KLAB_E_SHAPE;
  if (reinterpret_cast<uintptr_t>(pages) & 15) return KLAB_E_ALIGN;
  return 0;
}

int launch_rows(void (*kernel)(RowParams), unsigned threads, unsigned block, const RowParams& p, void* stream) {
  return launch_dependent(kernel, dim3((threads + block - 1) / block), block, 0, stream, p);
}

// One thread for 8 dims of a token, or for 8 dims of 2 or 4 groups of a pair of tokens.
template <bool kBf16, int D>
int launch_store(const RowParams& p, void* stream) {
  const unsigned pairs = (p.tokens + 1) / 2 * p.kv_heads;
  if constexpr (D >= 128) {
    if (pairs * (D / 4ll) >= kStoreBulkRuns)
      return launch_rows(kv_store_bulk_kernel<kBf16, D>, pairs * (D / 32), kBulkThreads, p, stream);
  }
  return launch_rows(kv_store_kernel<kBf16, D>, pairs * (D / 4), kStoreThreads, p, stream);
}

template <int kOut, int D>
int launch_read(const RowParams& p, void* stream) {
  const unsigned pairs = (p.tokens + 1) / 2 * p.kv_heads;
  if (pairs * (D / 4ll) < kReadBulkRuns)
    return launch_rows(kv_read_kernel<kOut, D>, pairs * (D / 4), kStoreThreads, p, stream);
  return launch_rows(kv_read_bulk_kernel<kOut, D>, pairs * (D == 256 ? 8 : 4), kBulkThreads, p, stream);
}

template <int kOut>
int launch_read(const RowParams& p, void* stream) {
  switch (p.dim) {
    case 64: return launch_read<kOut, 64>(p, stream);
    case 128: return launch_read<kOut, 128>(p, stream);
    default: return launch_read<kOut, 256>(p, stream);
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
  p.kv_heads = kv_heads;
  p.dim = dim;
  p.page_shift = kv_page_shift(page_size);
  const bool bf16 = dtype == KLAB_DT_BF16;
  switch (dim) {
    case 64: return bf16 ? launch_store<true, 64>(p, stream) : launch_store<false, 64>(p, stream);
    case 128: return bf16 ? launch_store<true, 128>(p, stream) : launch_store<false, 128>(p, stream);
    default: return bf16 ? launch_store<true, 256>(p, stream) : launch_store<false, 256>(p, stream);
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
