// Attention of a batch of requests over 4-bit K/V pages (kv_pages.cuh): for row (token j of request i, query head),
// out = sum_p softmax_p(scale * q . K_p) V_p over the positions p < length_i - new_i + j + 1, grouped query heads, ragged
// lengths read from device memory. Stands beside the single-sequence BF16 attention of decode_attn.cu.
//
// Work: an item is (request, tile of rows, run of 16-token blocks); CTA (item, kv head) has 4 warps that take the run's
// blocks in turn. The rows of a kv head are its query heads times the request's new tokens, in tiles of 8 or 16. The run
// length comes from the lengths themselves (every CTA adds up all requests), so uneven batches and single long ones fill
// the machine alike; a run that is not the whole request leaves its sums in scratch, and combine_kernel joins them in the
// order of the runs (a second launch, because per-call scratch then needs no zeroed counters: two captured graphs or two
// streams never share any).
//
// Per block and warp (K and V codes and scales: one bulk copy of 18 * D bytes into the warp's ring):
//   S^T = K Q^T   mma.m16n8k16, A = 16 tokens x 16 dims of codes u as FP16 subnormals (u * 2^-24, exact), B = q in FP16
//                 times a power of two (its row's maximum near 2^10, so nothing that counts is lost); the accumulator starts
//                 at -8 * 2^-24 * sum q of the group, which turns u into u - 8 without an instruction, and is multiplied
//                 by the token's FP32 scale after each group of 32 dims.
//   softmax       in base 2 against a reference exponent `ref` of the row that moves only when a score passes it by 2^4,
//                 so most blocks need no rescale and no cross-lane maximum; sums in FP32.
//   O^T += V^T P' A = 16 dims x 16 tokens of codes (FP16 subnormals), B = P' = p * (V scale of the token and group) in
//                 FP16. `ref` holds P' between 2^-16 and 2^15 with room below for the tail (FP16 subnormals end 2^-32
//                 under the row's largest weight), so the rounding of p and of the product, 2^-11 relative each at most, is
//                 what the FP16 operand costs. sum P' of a group comes from an MMA with ones, and -8 * sum P' turns u into
//                 u - 8 at the end.
// Scores beyond a row's last position are -inf before the softmax, and the scales of tokens beyond the request are zeroed,
// so whatever the allocator left there (NaN scales included) has no part.
//
// What bounds it: HBM for long caches (4.5 bits a value; about 13 instructions a lane per 8 K and 8 V values keep the
// issue slots near half), launch and dependent loads (lengths, table, first block) for short ones.
#include <cuda_fp16.h>

#include <atomic>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"
#include "kv_pages.cuh"

namespace klab {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
#ifndef KLAB_KV_SLOTS
#define KLAB_KV_SLOTS 4  // blocks in flight per warp
#endif
constexpr int kSlots = KLAB_KV_SLOTS;
#ifndef KLAB_KV_MIN_RUN
#define KLAB_KV_MIN_RUN 8  // blocks a run has at least (two per warp)
#endif
constexpr int kMinRun = KLAB_KV_MIN_RUN;
#ifndef KLAB_KV_CTAS_PER_SM
#define KLAB_KV_CTAS_PER_SM 8  // CTAs per SM that the run length aims at
#endif
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kSlack = 4.0f;  // log2 of how far a score may pass the row's reference before it moves

struct RunHeader {
  int run, runs;   // this run, and how many the (request, tile) has; runs = 0: nothing here
  int rows;        // rows of the tile
  int row0;        // its first row within the request: token row0 / group, head row0 % group
  int token0;      // the request's first token
  int pad[3];
};

struct KvAttnParams {
  const unsigned short* q;
  const unsigned char* pages;
  const int* table;
  const int* lengths;
  const int* starts;
  unsigned short* out;
  RunHeader* headers;
  float2* stats;   // [item][kv head][row] (ref, sum)
  float* sums;     // [item][kv head][row][dim]
  int* status;
  long long q_stride;
  int requests, tokens, width, num_pages, page_shift, heads, kv_heads, group, max_new, target;
  float scale_log2e;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                        unsigned b1, const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ unsigned pack_h2(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ unsigned mul_h2(unsigned a, unsigned b) {
  unsigned r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ unsigned max_h2(unsigned a, unsigned b) {
  unsigned r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <int N>
__device__ __forceinline__ void lds_words(unsigned addr, unsigned (&w)[N]) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "words of one run");
  if constexpr (N == 1) {
    w[0] = lds32(addr);
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = lds128(addr + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

// Requests are handed to CTAs by adding up all of them; a request whose lengths make no sense counts nothing.
struct Request {
  int length, fresh, token0;
  bool valid, bad;
};

__device__ __forceinline__ Request load_request(const KvAttnParams& p, int i) {
  Request r;
  r.length = p.lengths[i];
  r.token0 = p.starts[i];
  r.fresh = p.starts[i + 1] - r.token0;
  r.bad = r.fresh < 0 || r.fresh > p.max_new || r.token0 < 0 || r.token0 > p.tokens - max(r.fresh, 0) || r.length < 0 ||
          (static_cast<long long>(r.length) + (1 << p.page_shift) - 1) >> p.page_shift > p.width;
  r.valid = !r.bad && r.fresh > 0;
  return r;
}

__device__ __forceinline__ int blocks_of(int length) { return length > 0 ? (length - 1) / kKvBlock + 1 : 1; }

// Sum over the CTA's threads of v, and the exclusive prefix of this thread in `before`. Two barriers.
__device__ __forceinline__ long long cta_scan(long long v, long long* parts, long long& before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long s = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += up;
  }
  if (lane == 31) parts[warp] = s;
  __syncthreads();
  long long total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += parts[w];
    total += parts[w];
  }
  __syncthreads();
  before = base + s - v;
  return total;
}

template <int NG, int NT, bool kBf16>
__global__ void __launch_bounds__(kThreads) kv_attn_kernel(const KvAttnParams p) {
  constexpr int D = 32 * NG, Q = NG < 4 ? NG : 4, NQ = NG / Q, ROWS = 8 * NT;
  constexpr int kBytes = kv_block_bytes(D);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long bars[kWarps * kSlots];
  __shared__ long long parts[kWarps];
  __shared__ int found[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int item = blockIdx.x, kvh = blockIdx.y;

  if (tid < kWarps * kSlots) mbar_init(smem_addr(bars + tid), 1);
  fence_mbar_init();
  if (tid == 0) found[0] = -1;
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- the item: total blocks over all requests give the run length, a second pass finds the request
  long long mine = 0, before = 0;
  bool bad = false;
  for (int i = tid; i < p.requests; i += kThreads) {
    const Request r = load_request(p, i);
    bad |= r.bad;
    if (r.valid) mine += static_cast<long long>((r.fresh * p.group + ROWS - 1) / ROWS) * blocks_of(r.length);
  }
  if (bad && item == 0 && kvh == 0) record_status(p.status, kStatusBadLength);
  const long long all = cta_scan(mine, parts, before);
  long long want = (all * p.kv_heads + p.target - 1) / p.target;
  const int run_blocks = static_cast<int>(want > kMinRun ? want : kMinRun);
  long long carry = 0;
  for (int base = 0; base < p.requests; base += kThreads) {
    const int i = base + tid;
    Request r{};
    int runs = 0, tiles = 0;
    if (i < p.requests) {
      r = load_request(p, i);
      if (r.valid) {
        tiles = (r.fresh * p.group + ROWS - 1) / ROWS;
        runs = (blocks_of(r.length) + run_blocks - 1) / run_blocks;
      }
    }
    const long long n = static_cast<long long>(tiles) * runs;
    const long long total = cta_scan(n, parts, before);
    const long long at = item - carry - before;
    if (at >= 0 && at < n) {
      found[0] = i;
      found[1] = static_cast<int>(at) / runs;  // tile
      found[2] = static_cast<int>(at) % runs;
      found[3] = runs;
      found[4] = r.length;
      found[5] = r.fresh;
      found[6] = r.token0;
    }
    carry += total;
    if (item < carry) break;  // uniform: every thread sees the same sums
  }
  __syncthreads();
  const int request = found[0];
  if (request < 0) {
    if (tid == 0 && kvh == 0) p.headers[item].runs = 0;
    return;
  }
  const int tile = found[1], run = found[2], runs = found[3], length = found[4], fresh = found[5], token0 = found[6];
  const int row0 = tile * ROWS, rows = min(ROWS, fresh * p.group - row0);
  if (tid == 0 && kvh == 0) {
    RunHeader h{};
    h.run = run, h.runs = runs, h.rows = rows, h.row0 = row0, h.token0 = token0;
    p.headers[item] = h;
  }
  const int first_block = run * run_blocks;
  const int last_block = min(first_block + run_blocks, length > 0 ? blocks_of(length) : 0);
  const int count = max(0, (last_block - first_block - warp + kWarps - 1) / kWarps);  // this warp's blocks
  const int* table = p.table + static_cast<long long>(request) * p.width;
  const int per_page_shift = p.page_shift - 4;

  // ---- the warp's ring: block s of the warp is block first_block + warp + s * kWarps of the request
  const unsigned ring = smem_addr(smem) + warp * kSlots * kBytes;
  const unsigned bar0 = smem_addr(bars + warp * kSlots);
  unsigned skipped = 0;  // slots whose page is no page: nothing is copied and the block counts as masked
  int entry = -1;        // table entries of 32 blocks, one per lane
  auto issue = [&](int s) {
    if ((s & 31) == 0) {
      const int block = first_block + warp + (s + lane) * kWarps;
      entry = s + lane < count ? __ldg(table + (block >> per_page_shift)) : -1;
    }
    const int id = __shfl_sync(0xffffffffu, entry, s & 31), slot = s % kSlots;
    if (id < 0 || id >= p.num_pages) {
      skipped |= 1u << slot;
      if (lane == 0) record_status(p.status, kStatusBadPage);
      return;
    }
    skipped &= ~(1u << slot);
    if (lane == 0) {
      const int block = first_block + warp + s * kWarps;
      const long long at =
          ((static_cast<long long>(id) * p.kv_heads + kvh) << per_page_shift) + (block & ((1 << per_page_shift) - 1));
      fence_proxy_async_smem();  // the slot's last block was read by ordinary loads
      mbar_arrive_expect_tx(bar0 + 8 * slot, kBytes);
      bulk_g2s(ring + slot * kBytes, p.pages + at * kBytes, kBytes, bar0 + 8 * slot);
    }
  };
  for (int s = 0; s < kSlots && s < count; ++s) issue(s);

  // ---- q as B fragments: row g of each 8-row tile, times a power of two; -8 * 2^-24 * sum q per group
  unsigned qb[NT][NG][4];
  float c0[NT][NG][2];        // accumulator start of rows 2 t, 2 t + 1
  float rs[NT][2];            // score factor of rows 2 t, 2 t + 1: scale * log2(e) * 2^24 / (q's power of two)
  int limit[NT][2];           // positions that rows 2 t, 2 t + 1 see
  int least = INT_MAX;        // the smallest limit of the tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = nt * 8 + g;
    const bool there = row < rows;
    const int at = row0 + row, token = at / p.group;
    const unsigned short* src = p.q + (token0 + token) * p.q_stride +
                                static_cast<long long>(kvh * p.group + at - token * p.group) * D;
    uint4 w[NG];
#pragma unroll
    for (int G = 0; G < NG; ++G)
      w[G] = there ? __ldg(reinterpret_cast<const uint4*>(src + 32 * G + 8 * t)) : make_uint4(0u, 0u, 0u, 0u);
    float top = 0.0f;
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const unsigned u[4] = {w[G].x, w[G].y, w[G].z, w[G].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = fmaxf(top, fmaxf(fabsf(kBf16 ? bf16lo(u[e]) : f16lo(u[e])), fabsf(kBf16 ? bf16hi(u[e]) : f16hi(u[e]))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ef = max(static_cast<int>(__float_as_uint(top) >> 23), 11);
    const float up = __uint_as_float(static_cast<unsigned>(264 - ef) << 23);  // 2^(137 - ef): the maximum becomes < 2^11
    const float mine_rs = p.scale_log2e * __uint_as_float(static_cast<unsigned>(ef - 10) << 23) * 16777216.0f;
    float group_sum[NG];
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const unsigned u[4] = {w[G].x, w[G].y, w[G].z, w[G].w};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = (kBf16 ? bf16lo(u[e]) : f16lo(u[e])) * up;
        x[2 * e + 1] = (kBf16 ? bf16hi(u[e]) : f16hi(u[e])) * up;
      }
      // nibble pairs (0, 4), (1, 5) * 16, (2, 6), (3, 7) * 16
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float by = e & 1 ? 0.0625f : 1.0f;
        const unsigned pair = pack_h2(x[e] * by, x[e + 4] * by);
        qb[nt][G][e] = pair;
        sum += (f16lo(pair) + f16hi(pair)) * (e & 1 ? 16.0f : 1.0f);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      group_sum[G] = sum * (-8.0f / 16777216.0f);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // from the lane that holds row 2 t + e as its row g
      const int from = (2 * t + e) * 4;
#pragma unroll
      for (int G = 0; G < NG; ++G) c0[nt][G][e] = __shfl_sync(0xffffffffu, group_sum[G], from);
      rs[nt][e] = __shfl_sync(0xffffffffu, mine_rs, from);
      const int r = nt * 8 + 2 * t + e;
      limit[nt][e] = r < rows ? length - fresh + (row0 + r) / p.group + 1 : 0;
    }
  }
  least = length - fresh + row0 / p.group + 1;
  if (rows < ROWS) least = min(least, length);  // rows that are not there: masked or not, they are never written

  float o[NT][2 * NG][4], ones[NT][NG][4], l[NT][2], ref[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
#pragma unroll
    for (int G = 0; G < NG; ++G)
#pragma unroll
      for (int e = 0; e < 4; ++e) ones[nt][G][e] = 0.0f;
    l[nt][0] = l[nt][1] = 0.0f;
    ref[nt][0] = ref[nt][1] = kNegInf;
  }
  int vexp = -3;                    // log2 of the V scales that `ref` allows for (below 2^3 of it)
  unsigned vbound = 0u;             // 2^(vexp + 3) as an FP16 pair; 0 until the first block
  unsigned phases = 0;              // parity of each slot
  bool live = true;

  for (int s = 0; s < count; ++s) {
    const int slot = s % kSlots, block = first_block + warp + s * kWarps;
    if (skipped >> slot & 1) {
      if (s + kSlots < count) issue(s + kSlots);
      continue;
    }
    if (!mbar_wait(bar0 + 8 * slot, phases >> slot & 1)) {
      if (lane == 0) record_status(p.status, kStatusMbarTimeout);
      live = false;
    }
    live = __all_sync(0xffffffffu, live);
    if (!live) {  // leave, after a bounded wait for the warp's other copies in flight
      for (int k = s + 1; k < count && k < s + kSlots; ++k)
        if (!(skipped >> (k % kSlots) & 1)) (void)mbar_wait(bar0 + 8 * (k % kSlots), phases >> (k % kSlots) & 1);
      break;
    }
    phases ^= 1u << slot;
    const unsigned at = ring + slot * kBytes;
    // K words of tokens g, g + 8; V words of tokens 2 t, 2 t + 1 (j = 0) and 2 t + 8, 2 t + 9 (j = 1)
    unsigned kw[2][NG], vw[2][NG], sv[2][NG], kscale[2][NG / 2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int quad = 0; quad < NQ; ++quad) {
        unsigned a[Q];
        lds_words<Q>(at + quad * (256 * Q) + (g + 8 * j) * (16 * Q) + t * (4 * Q), a);
#pragma unroll
        for (int i = 0; i < Q; ++i) kw[j][quad * Q + i] = a[i];
        lds_words<Q>(at + 8 * D + quad * (256 * Q) + j * (128 * Q) + g * (16 * Q) + t * (4 * Q), a);
#pragma unroll
        for (int i = 0; i < Q; ++i) vw[j][quad * Q + i] = a[i];
      }
      lds_words<NG / 2>(at + 16 * D + (g + 8 * j) * (2 * NG), kscale[j]);
      lds_words<NG>(at + 17 * D + (j * 4 + t) * (4 * NG), sv[j]);
    }
    __syncwarp();
    if (s + kSlots < count) issue(s + kSlots);

    const int pos = block * kKvBlock;
    if (pos + kKvBlock > length) {  // tokens that are not there: scales whatever they are become 0
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int token = pos + 8 * j + 2 * t;
        const unsigned keep = (token < length ? 0x0000ffffu : 0u) | (token + 1 < length ? 0xffff0000u : 0u);
#pragma unroll
        for (int G = 0; G < NG; ++G) sv[j][G] &= keep;
      }
    }

    // ---- S^T = K Q^T
    float x[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] = 0.0f;
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const unsigned a = kw[0][G], b = kw[1][G], ah = a >> 8, bh = b >> 8;
      const float s0 = G & 1 ? f16hi(kscale[0][G / 2]) : f16lo(kscale[0][G / 2]);
      const float s1 = G & 1 ? f16hi(kscale[1][G / 2]) : f16lo(kscale[1][G / 2]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float acc[4];
        const float start[4] = {c0[nt][G][0], c0[nt][G][1], c0[nt][G][0], c0[nt][G][1]};
        mma_f16(acc, a & 0x000f000fu, b & 0x000f000fu, a & 0x00f000f0u, b & 0x00f000f0u, qb[nt][G][0], qb[nt][G][1],
                start);
        mma_f16(acc, ah & 0x000f000fu, bh & 0x000f000fu, ah & 0x00f000f0u, bh & 0x00f000f0u, qb[nt][G][2],
                qb[nt][G][3], acc);
        x[nt][0] = fmaf(acc[0], s0, x[nt][0]);
        x[nt][1] = fmaf(acc[1], s0, x[nt][1]);
        x[nt][2] = fmaf(acc[2], s1, x[nt][2]);
        x[nt][3] = fmaf(acc[3], s1, x[nt][3]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] *= rs[nt][e & 1];
    if (pos + kKvBlock > least) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (pos + g + (e & 2 ? 8 : 0) >= limit[nt][e & 1]) x[nt][e] = kNegInf;
    }

    // ---- does the reference still hold? P' = 2^(x - ref) * V scale stays below 2^15
    unsigned vtop = max_h2(sv[0][0], sv[1][0]);
#pragma unroll
    for (int G = 1; G < NG; ++G) vtop = max_h2(vtop, max_h2(sv[0][G], sv[1][G]));
    bool move = max_h2(vtop, vbound) != vbound;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) move |= x[nt][e] > ref[nt][e & 1] + (8.0f + kSlack) - static_cast<float>(vexp);
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) vtop = max_h2(vtop, __shfl_xor_sync(0xffffffffu, vtop, d));
      const float v = fmaxf(f16lo(vtop), f16hi(vtop));
      const int exponent = static_cast<int>(__float_as_uint(v) >> 23) - 126;  // v < 2^exponent
      const int old = vexp;
      vexp = max(vexp, exponent);
      // 2^(vexp + 3) where FP16 has it, its largest finite value above that
      const int bits = vexp + 3 < 16 ? (vexp + 18) << 10 : 0x7bff;
      vbound = static_cast<unsigned>(bits) * 0x10001u;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(x[nt][e], x[nt][e + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          // ref = (largest score so far) - 8 + vexp
          const float was = ref[nt][e];
          const float now = fmaxf(top - 8.0f, was - static_cast<float>(old)) + static_cast<float>(vexp);
          const float factor = was == kNegInf ? 0.0f : exp2_fast(was - now);
          if (was != kNegInf) {
            l[nt][e] *= factor;
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) o[nt][i][e] *= factor, o[nt][i][e + 2] *= factor;
#pragma unroll
            for (int G = 0; G < NG; ++G) ones[nt][G][e] *= factor, ones[nt][G][e + 2] *= factor;
          }
          ref[nt][e] = now;
        }
    }

    // ---- P, its sums, and P' per group as B fragments (rows x tokens)
    unsigned pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float r = ref[nt][e & 1];
        w[e] = exp2_fast(x[nt][e] - (r == kNegInf ? 0.0f : r));
      }
      l[nt][0] += w[0] + w[2];
      l[nt][1] += w[1] + w[3];
      pb[nt][0] = transpose8x8(pack_h2(w[0], w[1]));
      pb[nt][1] = transpose8x8(pack_h2(w[2], w[3]));
    }

    // ---- O^T += V^T P'
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const unsigned a = vw[0][G], b = vw[1][G], ah = a >> 8, bh = b >> 8;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const unsigned b0 = mul_h2(pb[nt][0], sv[0][G]), b1 = mul_h2(pb[nt][1], sv[1][G]);
        mma_f16(o[nt][2 * G], a & 0x000f000fu, a & 0x00f000f0u, b & 0x000f000fu, b & 0x00f000f0u, b0, b1,
                o[nt][2 * G]);
        mma_f16(o[nt][2 * G + 1], ah & 0x000f000fu, ah & 0x00f000f0u, bh & 0x000f000fu, bh & 0x00f000f0u, b0, b1,
                o[nt][2 * G + 1]);
        mma_f16(ones[nt][G], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, b0, b1, ones[nt][G]);
      }
    }
  }

  // ---- the warps' sums over the ring's memory: [warp][row][dim] and (ref, sum) per warp and row
  __syncthreads();
  float* wo = reinterpret_cast<float*>(smem);
  float2* ws = reinterpret_cast<float2*>(smem + static_cast<size_t>(kWarps) * ROWS * D * 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[nt][e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const int row = nt * 8 + 2 * t + e;
      if (g == 0) ws[warp * ROWS + row] = make_float2(ref[nt][e], sum);
      float* to = wo + (warp * ROWS + row) * D;
#pragma unroll
      for (int G = 0; G < NG; ++G) {
        const float eight = 8.0f * ones[nt][G][e];
        float4 v;
        v.x = fmaf(o[nt][2 * G][e], 16777216.0f, -eight);
        v.y = fmaf(o[nt][2 * G][e + 2], 1048576.0f, -eight);
        v.z = fmaf(o[nt][2 * G + 1][e], 16777216.0f, -eight);
        v.w = fmaf(o[nt][2 * G + 1][e + 2], 1048576.0f, -eight);
        *reinterpret_cast<float4*>(to + 32 * G + 4 * g) = v;
      }
    }
  __syncthreads();
  constexpr int kVec = D / 4;  // float4s of a row
  for (int at = tid; at < rows * kVec; at += kThreads) {
    const int row = at / kVec, c = at - row * kVec;
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ws[w * ROWS + row].x);
    float den = 0.0f;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 st = ws[w * ROWS + row];
      if (st.x == kNegInf && st.y == 0.0f) continue;  // a warp that saw nothing of this row
      const float f = exp2_fast(st.x - top);
      const float4 v = *reinterpret_cast<const float4*>(wo + (w * ROWS + row) * D + 4 * c);
      den = fmaf(f, st.y, den);
      num.x = fmaf(f, v.x, num.x), num.y = fmaf(f, v.y, num.y), num.z = fmaf(f, v.z, num.z), num.w = fmaf(f, v.w, num.w);
    }
    if (runs == 1) {
      const float by = den == 0.0f ? 0.0f : __frcp_rn(den);  // a row that sees no position: 0
      const int r = row0 + row, token = r / p.group;
      unsigned short* to = p.out + (static_cast<long long>(token0 + token) * p.heads + kvh * p.group + r - token * p.group) * D;
      uint2 w;
      if (kBf16) {
        w.x = f32_to_bf16_rn(num.x * by) | static_cast<unsigned>(f32_to_bf16_rn(num.y * by)) << 16;
        w.y = f32_to_bf16_rn(num.z * by) | static_cast<unsigned>(f32_to_bf16_rn(num.w * by)) << 16;
      } else {
        w.x = pack_h2(num.x * by, num.y * by);
        w.y = pack_h2(num.z * by, num.w * by);
      }
      reinterpret_cast<uint2*>(to)[c] = w;
    } else {
      const long long rec = (static_cast<long long>(item) * p.kv_heads + kvh) * ROWS + row;
      if (c == 0) p.stats[rec] = make_float2(top, den);
      reinterpret_cast<float4*>(p.sums + rec * D)[c] = num;
    }
  }
}

// Joins the runs of one (request, tile, kv head): the tile's rows are dealt to the CTAs that made the runs. 128 threads =
// D / 4 float4 columns x the classes that share the runs; the classes' sums are added in order.
template <int D, int ROWS, bool kBf16>
__global__ void __launch_bounds__(kThreads) kv_combine_kernel(const KvAttnParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  float4* part = reinterpret_cast<float4*>(smem);             // [classes][columns]
  float* weight = reinterpret_cast<float*>(smem + 16 * kThreads);  // [runs]
  __shared__ float red[2 * kWarps];
  grid_dependency_wait();
  grid_launch_dependents();
  const RunHeader h = p.headers[blockIdx.x];
  if (h.runs <= 1) return;
  const int kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kCols = D / 4, kClasses = kThreads / kCols;
  const int col = tid % kCols, cls = tid / kCols;
  const long long first = blockIdx.x - h.run;
  for (int row = h.run; row < h.rows; row += h.runs) {
    auto record = [&](int k) { return ((first + k) * p.kv_heads + kvh) * ROWS + row; };
    float top = kNegInf;
    for (int k = tid; k < h.runs; k += kThreads) top = fmaxf(top, __ldcg(p.stats + record(k)).x);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red[w]);
    float den = 0.0f;
    for (int k = tid; k < h.runs; k += kThreads) {
      const float2 st = __ldcg(p.stats + record(k));
      const float f = st.x == kNegInf && st.y == 0.0f ? 0.0f : exp2_fast(st.x - top);
      weight[k] = f;
      den = fmaf(f, st.y, den);
    }
    den = warp_allsum(den);
    if (lane == 0) red[kWarps + warp] = den;
    __syncthreads();
    den = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) den += red[kWarps + w];
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int k = cls; k < h.runs; k += kClasses) {
      const float f = weight[k];
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.sums + record(k) * D) + col);
      if (f != 0.0f)
        num.x = fmaf(f, v.x, num.x), num.y = fmaf(f, v.y, num.y), num.z = fmaf(f, v.z, num.z), num.w = fmaf(f, v.w, num.w);
    }
    part[tid] = num;
    __syncthreads();
    if (cls == 0) {
#pragma unroll
      for (int k = 1; k < kClasses; ++k) {
        const float4 v = part[k * kCols + col];
        num.x += v.x, num.y += v.y, num.z += v.z, num.w += v.w;
      }
      const float by = den == 0.0f ? 0.0f : __frcp_rn(den);
      const int r = h.row0 + row, token = r / p.group;
      unsigned short* to = p.out + (static_cast<long long>(h.token0 + token) * p.heads + kvh * p.group + r - token * p.group) * D;
      uint2 w;
      if (kBf16) {
        w.x = f32_to_bf16_rn(num.x * by) | static_cast<unsigned>(f32_to_bf16_rn(num.y * by)) << 16;
        w.y = f32_to_bf16_rn(num.z * by) | static_cast<unsigned>(f32_to_bf16_rn(num.w * by)) << 16;
      } else {
        w.x = pack_h2(num.x * by, num.y * by);
        w.y = pack_h2(num.z * by, num.w * by);
      }
      reinterpret_cast<uint2*>(to)[col] = w;
    }
    __syncthreads();
  }
}

// What a call launches; the grid and the scratch depend on the shapes alone, so a captured call serves any lengths.
struct KvPlan {
  int tiles_nt;       // 8-row tiles a CTA holds (1 or 2)
  int items, target;
  bool combine;
  size_t headers, stats, sums, total;  // scratch offsets
  size_t smem;
};

int kv_sms(int* sms) {
  static std::atomic<int> cached[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return KLAB_E_UNSUPPORTED;
  int n = cached[dev].load();
  if (!n) {
    err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (err != cudaSuccess) return err;
    cached[dev].store(n);
  }
  *sms = n;
  return 0;
}

int kv_plan(int requests, int width, int page_size, int heads, int kv_heads, int dim, int max_new, KvPlan* plan) {
  if (requests <= 0 || width <= 0 || heads <= 0 || kv_heads <= 0 || max_new <= 0) return KLAB_E_INVALID;
  if (requests > kKvMaxRequests || kv_heads > 65535 || heads % kv_heads || heads / kv_heads > 64 || max_new > kKvMaxNew ||
      !kv_dim_ok(dim) || !kv_page_size_ok(page_size) || static_cast<long long>(width) * page_size > INT_MAX)
    return KLAB_E_SHAPE;
  int sms = 0;
  const int rc = kv_sms(&sms);
  if (rc) return rc;
  const int most_rows = heads / kv_heads * max_new;
  plan->tiles_nt = most_rows > 8 && dim < 256 ? 2 : 1;
  const int rows = 8 * plan->tiles_nt, tiles = (most_rows + rows - 1) / rows;
  const long long runs = (static_cast<long long>(width) * page_size / kKvBlock + kMinRun - 1) / kMinRun;
  plan->target = sms * KLAB_KV_CTAS_PER_SM;
  const long long segments = static_cast<long long>(requests) * tiles;
  long long items = segments + plan->target / kv_heads + 1;
  if (segments * runs < items) items = segments * runs;
  if (items > INT_MAX / 2) return KLAB_E_SHAPE;
  plan->items = static_cast<int>(items);
  plan->combine = runs > 1;
  plan->headers = 0;
  plan->stats = (static_cast<size_t>(items) * sizeof(RunHeader) + 127) / 128 * 128;
  const size_t records = plan->combine ? static_cast<size_t>(items) * kv_heads * rows : 0;
  plan->sums = plan->stats + (records * 8 + 127) / 128 * 128;
  plan->total = plan->sums + records * dim * 4;
  const size_t ring = static_cast<size_t>(kWarps) * kSlots * kv_block_bytes(dim);
  const size_t join = static_cast<size_t>(kWarps) * rows * (dim * 4 + 8);
  plan->smem = ring > join ? ring : join;
  return 0;
}

template <typename... A>
int launch_kv(void (*kernel)(A...), dim3 grid, size_t smem, cudaStream_t stream, const KvAttnParams& p) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = klab_get_option(KLAB_OPT_PDL) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int NG, int NT, bool kBf16>
int run_kv(const KvAttnParams& p, const KvPlan& plan, cudaStream_t stream) {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (!(ready.load() >> dev & 1)) {
    err = cudaFuncSetAttribute(kv_attn_kernel<NG, NT, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(plan.smem));
    if (err != cudaSuccess) return err;
    ready.fetch_or(1ull << dev);
  }
  const dim3 grid(static_cast<unsigned>(plan.items), static_cast<unsigned>(p.kv_heads));
  int rc = launch_kv(kv_attn_kernel<NG, NT, kBf16>, grid, plan.smem, stream, p);
  if (rc || !plan.combine) return rc;
  // At most target / kv_heads + 1 runs share a (request, tile): the weights' room.
  const size_t smem = 16 * kThreads + 4 * (static_cast<size_t>(plan.target / p.kv_heads) + 2);
  return launch_kv(kv_combine_kernel<32 * NG, 8 * NT, kBf16>, grid, smem, stream, p);
}

template <bool kBf16>
int dispatch_kv(int dim, const KvAttnParams& p, const KvPlan& plan, cudaStream_t stream) {
  const bool two = plan.tiles_nt == 2;
  switch (dim) {
    case 64: return two ? run_kv<2, 2, kBf16>(p, plan, stream) : run_kv<2, 1, kBf16>(p, plan, stream);
    case 128: return two ? run_kv<4, 2, kBf16>(p, plan, stream) : run_kv<4, 1, kBf16>(p, plan, stream);
    default: return run_kv<8, 1, kBf16>(p, plan, stream);
  }
}

}  // namespace
}  // namespace klab

extern "C" {

KLAB_API long long klab_kv_attention_scratch(int requests, int width, int page_size, int heads, int kv_heads, int dim,
                                             int max_new) {
  klab::KvPlan plan{};
  const int rc = klab::kv_plan(requests, width, page_size, heads, kv_heads, dim, max_new, &plan);
  if (rc) return rc < 0 ? rc : -rc;
  return static_cast<long long>(plan.total);
}

KLAB_API int klab_kv_attention(const void* q, long long q_stride, int dtype, const void* pages, const int* table,
                               const int* lengths, const int* starts, void* out, void* scratch, long long scratch_bytes,
                               int tokens, int requests, int width, int num_pages, int page_size, int heads,
                               int kv_heads, int dim, int max_new, float scale, void* stream) {
  using namespace klab;
  if (!q || !pages || !table || !lengths || !starts || !out || !scratch || tokens <= 0 || num_pages <= 0)
    return KLAB_E_INVALID;
  if (dtype != KLAB_DT_BF16 && dtype != KLAB_DT_F16) return KLAB_E_UNSUPPORTED;
  KvPlan plan{};
  const int rc = kv_plan(requests, width, page_size, heads, kv_heads, dim, max_new, &plan);
  if (rc) return rc;
  if (static_cast<long long>(num_pages) * page_size > INT_MAX) return KLAB_E_SHAPE;
  if (static_cast<long long>(plan.total) > scratch_bytes) return KLAB_E_INVALID;
  const uintptr_t mis = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages) |
                        reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch);
  if (mis & 15 || q_stride & 7) return KLAB_E_ALIGN;
  KvAttnParams p{};
  unsigned char* base = static_cast<unsigned char*>(scratch);
  p.q = static_cast<const unsigned short*>(q);
  p.pages = static_cast<const unsigned char*>(pages);
  p.table = table;
  p.lengths = lengths;
  p.starts = starts;
  p.out = static_cast<unsigned short*>(out);
  p.headers = reinterpret_cast<RunHeader*>(base + plan.headers);
  p.stats = reinterpret_cast<float2*>(base + plan.stats);
  p.sums = reinterpret_cast<float*>(base + plan.sums);
  p.status = device_status_address();
  p.q_stride = q_stride;
  p.requests = requests;
  p.tokens = tokens;
  p.width = width;
  p.num_pages = num_pages;
  p.page_shift = kv_page_shift(page_size);
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.max_new = max_new;
  p.target = plan.target;
  p.scale_log2e = scale * 1.44269504088896340736f;
  return dtype == KLAB_DT_BF16 ? dispatch_kv<true>(dim, p, plan, static_cast<cudaStream_t>(stream))
                               : dispatch_kv<false>(dim, p, plan, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
