// Attention of a batch of requests over 4-bit K/V pages (kv_pages.cuh): for row (token j of request i, query head),
// out = sum_p softmax_p(scale * q . K_p) V_p over the positions p < length_i - new_i + j + 1, grouped query heads, ragged
// lengths read from device memory. Stands beside the single-sequence BF16 attention of decode_attn.cu.
//
// Work: a segment is a tile of 8 query rows of a request and kv head (its query heads times its new tokens), in units of
// 32 tokens. All segments of a kv head, one behind the other, are cut into equal shares, one for each CTA that the machine
// holds at once (or, while shares are short, every segment into shares of its own that are nearly as long); every CTA adds
// up all requests to find its own, so uneven batches and single long ones fill the machine alike, and its 4 warps take a
// piece's units in turn. A piece that is not a whole segment leaves its sums in scratch, and
// kv_combine_kernel joins them in order (a second launch, because per-call scratch then needs no zeroed counters: two
// captured graphs or two streams never share any). Tables of at most 512 tokens a request are not cut: whole segments are
// dealt, and the second launch is saved.
//
// Per unit and warp (two blocks of 16 tokens: K and V codes and scales, one bulk copy of 18 * D bytes each into the
// warp's ring):
//   S^T = K Q^T   mma.m16n8k16, A = 16 tokens x 16 dims of codes u as FP16 subnormals (u * 2^-24, exact), B = q in FP16
//                 times a power of two (its row's maximum in [2^14, 2^15): exact down to 2^-28 of the row's largest for
//                 BF16 and 2^-25 for FP16, below that off by 2^-35 of it at most; the codes need FP16); each group of 32
//                 dims is multiplied by the token's scale in FP32. -8 * scale * sum q, which turns u into u - 8, is one
//                 more MMA of the scales with the groups' sums of q in two FP16 terms, and starts the sum.
//   softmax       in base 2 against a reference `ref` of the row that moves only when a score passes it by 2^14, so most
//                 units need no rescale and no cross-lane maximum; weights and sums in FP32.
//   O^T += V^T P' A = 16 dims x 16 tokens of codes (FP16 subnormals), B = P' = p * (V scale of the token and group), formed
//                 in FP32 and rounded once to FP16 (2^-11 relative at most, for the tensor cores' sake). `ref` counts the
//                 range of the V scales in (below 2^-7, below 2, or any): p can be 2^22 for weak rows and 2^-1 for strong
//                 ones, and P' stays below 2^15 with room under it for the tail, 2^-34 to 2^-27 of the row's largest weight
//                 where its scale is near its range's. (p rounded to FP16 first saves 3 % for BF16 outputs, adds as much
//                 error again, and leaves FP16 where the scales of one row are far from another's.) sum P' of each group
//                 comes from an MMA with ones, and -8 sum P' turns u into u - 8 at the end, so u and 8 meet the same P' and a
//                 code of 8 stays an exact 0. (One MMA of the scales with p in place of the four with ones saved 1.5 % and
//                 lost that.)
// Scores beyond a row's last position are -inf before the softmax, and the scales of tokens beyond the request are zeroed,
// so whatever the allocator left there (NaN scales included) has no part.
//
// What bounds it: long caches the warps' own chains (about 610 instructions a warp and unit of 4608 bytes at D = 128, issue
// slots 56 % busy with the 12 warps that registers allow, the ALU pipe 51 %, tensor cores 31 %), before HBM: 64 x 8192
// tokens, 8 kv heads of 128, 243 MB in 63.4 us, 3.8 TB/s; 1 x 131072, 151 MB in 38.5 us, 3.9 TB/s. Four CTAs an SM (80
// registers), more shares than CTAs, the next piece's first copies issued ahead and 16 rows a tile all measured the same or
// slower. Short ones launch, dependent loads (lengths, table, first block) and the join (2.8 us): 1 x 300 tokens 4.9 us.
#include <cuda_fp16.h>

#include <atomic>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"
#include "kv_pages.cuh"
#include "launch.cuh"

namespace klab {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 8;  // query rows of a tile (the MMA's N)
// Units of two blocks that a warp's ring holds: a third one takes shared memory and L1 from the third CTA of an SM at heads
// of 64 and 256 (26.4 us against 32.3, 22.2 against 29.8) and changes heads of 128 by 1 %.
constexpr int kSlots = 2;
// Units a CTA takes at least: short batches pay for the sums that every share leaves (1 x 2000 tokens 7.9 us, with 2 units
// 8.4, with 8 units 8.0).
constexpr int kMinShare = 4;
// Up to 64 requests whose equal shares have at most kTry units: every segment gets CTAs of its own where shares of up to
// kSlack units more allow it, since a CTA's second piece starts and ends like its first: 16 x 4096 tokens 14.4 us, with
// equal shares 16.8; 32 x 1000 12.7 and 18.3; 8 x 2048 drafts 11.9 and 13.9. Above kTry equal shares are as good or better
// (32 x 8192 36.6 us, 37.4 with the search; 32 x 4096, just under it, 26.5 and 25.8), and 8 units of slack measure the same.
constexpr int kTry = 40, kSlack = 16;
constexpr int kUnitTokens = 2 * kKvBlock;
// Tables of at most this many units are not cut: 1 x 250 tokens 5.1 us against 6.6 cut, 64 x 512 15.1 against 19.2;
// 1 x 2000 17.0 us whole and 7.9 cut.
constexpr int kWholeUnits = 16;
constexpr float kNegInf = -__builtin_huge_valf();
// A row's weights are 2^(score - ref) with ref = (a score near the largest) - 10 + e, moved when a score passes it by
// 14 - e; V scales below 2^(e + 1) then keep P' below 2^15. e is that of the range of the scales a warp has met: FP16 patterns
// say by their two highest exponent bits whether one is 2^-7 or more, and 2 or more.
constexpr float kRefBelow = 10.0f, kMoveAt = 14.0f;
constexpr float kWeakRange = -8.0f, kPlainRange = 0.0f, kStrongRange = 15.0f;
constexpr unsigned kAboveWeak = 0x60006000u, kAbovePlain = 0x40004000u;

// Of each CTA: where its share begins inside a segment (a tile of rows of a request), what the CTAs from `first` to `last`
// of that segment left in scratch has to be joined.
struct Header {
  int first, last;  // last = -1: nothing to join
  int rows, row0;   // rows of the tile, its first row within the request: token row0 / group, head row0 % group
  int token0;       // the request's first token
  int pad[3];
};

struct KvAttnParams {
  const unsigned short* q;
  const unsigned char* pages;
  const int* table;
  const int* lengths;
  const int* starts;
  unsigned short* out;
  Header* headers;  // [CTA of a kv head]
  float2* stats;    // [CTA of a kv head][kv head][2][row] (ref, sum): records of the CTA's first and last piece
  float* sums;      // [..][dim]
  int* status;
  long long q_stride;
  int requests, tokens, width, num_pages, page_shift, heads, kv_heads, group, group_div, max_new, max_length, whole, fill;
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

__device__ __forceinline__ float lo_f32(unsigned w) { return __low2float(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float hi_f32(unsigned w) { return __high2float(*reinterpret_cast<const __half2*>(&w)); }

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

// row / group for row < 1024 and group <= 64 (div = ceil(2^16 / group): exact while row * (group - 1) < 2^16).
__device__ __forceinline__ int by_group(const KvAttnParams& p, int row) { return (row * p.group_div) >> 16; }

// A request as the lengths say; tiles = 0 for one without new tokens or whose numbers make no sense.
struct Request {
  int length, fresh, token0, tiles, units;
};

__device__ __forceinline__ Request make_request(const KvAttnParams& p, int length, int start, int end, bool& bad) {
  Request r;
  r.length = length;
  r.token0 = start;
  r.fresh = end - start;
  const bool wrong =
      start < 0 || end < start || end > p.tokens || r.fresh > p.max_new || length < 0 || length > p.max_length;
  bad |= wrong;
  r.tiles = wrong ? 0 : (r.fresh * p.group + kRows - 1) / kRows;
  // A request without a token has a unit that sees nothing; segments that are dealt whole count one unit each.
  r.units = length > 0 && !p.whole ? (length - 1) / kUnitTokens + 1 : 1;
  return r;
}

// Units of all (request, tile) one behind the other, requests in order; a CTA takes `share` of them from `pos` on. Every
// warp works its piece out for itself: the loads are the same few lines for the whole machine, and no barrier is needed.
struct Share {
  int pos, end;              // this CTA's units
  int request, tile, unit;   // the segment that holds `pos`, and the unit within it
  int first, last;           // the CTAs that this segment's units went to
  Request r;
};

__device__ __forceinline__ Share find_share(const KvAttnParams& p, int cta, int ctas, bool report, bool& wrong) {
  constexpr int kFlight = 4;  // requests of a lane whose loads are in flight at once
  const int lane = threadIdx.x & 31, each = (p.requests + 31) / 32;
  bool bad = false;
  // Ordinary loads, here and for q and the table: what the launch before wrote while this one was already resident is not
  // read-only data of the kernel.
  auto load = [&](int i, int end) {
    int length = 0, start = 0, stop = 0;
    if (i < end) {
      length = p.lengths[i];
      start = p.starts[i];
      stop = p.starts[i + 1];
    }
    return make_request(p, length, start, stop, bad);
  };
  auto scan = [&](int upto) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += up;
    }
    return upto;
  };
  // A lane adds up a run of `each` requests; the run that holds the share's beginning is then looked through by all.
  Request held[2] = {load(lane * each, p.requests), load(lane * each + 1, each > 1 ? p.requests : 0)};
  int mine = held[0].tiles * held[0].units + held[1].tiles * held[1].units;
  for (int j = 2; j < each; j += kFlight) {
#pragma unroll
    for (int u = 0; u < kFlight; ++u)
      if (j + u < each) {
        const Request q = load(lane * each + j + u, p.requests);
        mine += q.tiles * q.units;
      }
  }
  int upto = scan(mine);
  const int all = __shfl_sync(0xffffffffu, upto, 31);
  wrong = __any_sync(0xffffffffu, bad);
  if (wrong && report) record_status(p.status, kStatusBadLength);
  Share it;
  it.request = it.tile = it.unit = it.first = it.last = 0;
  auto take = [&](const Request& r, int from) {
    it.r.length = __shfl_sync(0xffffffffu, r.length, from);
    it.r.fresh = __shfl_sync(0xffffffffu, r.fresh, from);
    it.r.token0 = __shfl_sync(0xffffffffu, r.token0, from);
    it.r.tiles = __shfl_sync(0xffffffffu, r.tiles, from);
    it.r.units = __shfl_sync(0xffffffffu, r.units, from);
  };
  const int share = max(p.whole ? 1 : kMinShare, (all + ctas - 1) / ctas);
  if (each <= 2 && !p.whole && share <= kTry && (p.requests > 1 || p.max_new * p.group > kRows) &&
      __reduce_add_sync(0xffffffffu, held[0].tiles + held[1].tiles) <= ctas) {
    // CTAs of its own for every segment: a lane counts them for shares of share + lane units.
    const float by = 1.0f / static_cast<float>(share + lane);
    int need = 0;
    auto count_of = [&](const Request& r, int i) {
      return __shfl_sync(0xffffffffu, r.tiles, i) *
             static_cast<int>(ceilf(static_cast<float>(__shfl_sync(0xffffffffu, r.units, i)) * by));
    };
#pragma unroll 4
    for (int i = 0; i < min(p.requests, 32); ++i) need += count_of(held[0], i);
    if (each > 1) {
#pragma unroll 4
      for (int i = 0; i < 32; ++i) need += count_of(held[1], i);
    }
    const unsigned fits = __ballot_sync(0xffffffffu, lane <= kSlack && need <= ctas);
    if (fits) {
      const int own = share + __ffs(fits) - 1;
      int parts[2], count[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) parts[j] = (held[j].units + own - 1) / own, count[j] = held[j].tiles * parts[j];
      const int behind = scan(count[0] + count[1]), total = __shfl_sync(0xffffffffu, behind, 31);
      if (total <= ctas) {
        it.pos = it.end = 0;
        const unsigned owner = __ballot_sync(0xffffffffu, cta < behind);
        if (!owner) return it;  // a CTA too many
        const int from = __ffs(owner) - 1, before = __shfl_sync(0xffffffffu, behind - count[0] - count[1], from);
        const int second = cta - before >= __shfl_sync(0xffffffffu, count[0], from);
        const int rest = cta - before - (second ? __shfl_sync(0xffffffffu, count[0], from) : 0);
        const int n = __shfl_sync(0xffffffffu, second ? parts[1] : parts[0], from);
        Request r = held[0];
        if (second) r = held[1];
        take(r, from);
        it.request = from * each + second;
        it.tile = rest / n;
        const int part = rest - it.tile * n;
        it.unit = part * it.r.units / n;  // n shares of at most kTry + kSlack units: the product is small
        it.end = (part + 1) * it.r.units / n - it.unit;
        it.first = cta - part, it.last = it.first + n - 1;
        return it;
      }
    }
  }
  it.pos = min(static_cast<long long>(cta) * share, static_cast<long long>(all));
  it.end = min(it.pos + share, all);
  if (it.pos >= it.end) return it;
  int left = it.pos;  // units from the start of what `upto` counts
  int base = 0, stop = p.requests;
  Request r = held[0];
  if (each > 1) {
    const int from = __ffs(__ballot_sync(0xffffffffu, left < upto)) - 1;
    left -= __shfl_sync(0xffffffffu, upto - mine, from);
    base = from * each, stop = min(base + each, p.requests);
    r = load(base + lane, stop);
    mine = r.tiles * r.units;
    upto = scan(mine);
  }
  while (true) {
    const unsigned owner = __ballot_sync(0xffffffffu, left < upto);
    if (owner) {
      const int from = __ffs(owner) - 1;
      it.request = base + from;
      take(r, from);
      it.unit = left - __shfl_sync(0xffffffffu, upto - mine, from);
      if (it.r.tiles > 1) {
        it.tile = it.unit / it.r.units;
        it.unit -= it.tile * it.r.units;
      }
      const int begin = it.pos - it.unit;
      it.first = begin / share, it.last = (begin + it.r.units - 1) / share;
      return it;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
    base += 32;
    if (base >= stop) {  // not with lengths that stay as they are during the call
      it.pos = it.end;
      return it;
    }
    r = load(base + lane, stop);
    mine = r.tiles * r.units;
    upto = scan(mine);
  }
}

// The segment behind this one (there is one while pos < end).
__device__ __forceinline__ void next_segment(const KvAttnParams& p, Share& it) {
  it.unit = 0;
  if (++it.tile < it.r.tiles) return;
  it.tile = 0;
  bool bad = false;
  it.r.tiles = 0;
  while (it.r.tiles == 0 && ++it.request < p.requests)
    it.r = make_request(p, p.lengths[it.request], p.starts[it.request], p.starts[it.request + 1], bad);
  if (it.r.tiles == 0) it.pos = it.end;  // not with lengths that stay as they are during the call
}

// Rows of `out` that belong to no request become 0 (this kv head's part, rows dealt to the warps of all CTAs): those before
// the first request's and behind the last one's, and where a request's numbers make no sense all that no other one has.
__device__ __noinline__ void fill_rows(const KvAttnParams& p, int first, int last, bool wrong, int kvh, int dim) {
  const int lane = threadIdx.x & 31, warps = gridDim.x * kWarps;
  const int count = wrong ? p.tokens : first + p.tokens - last;
  for (int i = blockIdx.x * kWarps + (threadIdx.x >> 5); i < count; i += warps) {
    int row = i;
    if (wrong) {
      bool held = false, bad = false;
      for (int r = lane; r < p.requests; r += 32) {
        const Request q = make_request(p, p.lengths[r], p.starts[r], p.starts[r + 1], bad);
        held |= q.tiles > 0 && row >= q.token0 && row < q.token0 + q.fresh;
      }
      if (__any_sync(0xffffffffu, held)) continue;
    } else if (i >= first) {
      row = last + i - first;
    }
    uint4* to = reinterpret_cast<uint4*>(p.out + (static_cast<long long>(row) * p.heads + kvh * p.group) * dim);
    for (int c = lane; c < p.group * dim / 8; c += 32) to[c] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// CTAs per SM the registers are cut for; heads of 256 hold twice the accumulators.
constexpr int kv_resident(int ng) { return ng <= 4 ? 3 : 2; }

__device__ __forceinline__ long long record_of(const KvAttnParams& p, int cta, int kvh, int which) {
  return ((static_cast<long long>(cta) * p.kv_heads + kvh) * 2 + which) * kRows;
}

template <int NG, bool kBf16>
__global__ void __launch_bounds__(kThreads, kv_resident(NG)) kv_attn_kernel(const __grid_constant__ KvAttnParams p) {
  constexpr int D = 32 * NG, Q = NG < 4 ? NG : 4, NQ = NG / Q;
  constexpr int kBytes = kv_block_bytes(D);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long bars[kWarps * kSlots];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, kvh = blockIdx.y;

  if (lane < kSlots) mbar_init(smem_addr(bars + warp * kSlots + lane), 2);  // the warp's own
  fence_mbar_init();
  __syncwarp();
  grid_dependency_wait();
  grid_launch_dependents();

  int before = 0, behind = p.tokens;
  if (p.fill) {
    before = min(max(p.starts[0], 0), p.tokens);
    behind = min(max(p.starts[p.requests], before), p.tokens);
  }
  bool wrong;
  Share it = find_share(p, cta, gridDim.x, cta == 0 && kvh == 0 && warp == 0, wrong);
  if (p.fill && (wrong || before > 0 || behind < p.tokens)) fill_rows(p, before, behind, wrong, kvh, D);
  if (tid == 0 && kvh == 0) {
    Header h{};
    h.last = -1;
    if (it.pos < it.end && it.unit > 0) {  // the share begins inside a segment: others hold its beginning
      h.first = it.first;
      h.last = it.last;
      h.row0 = it.tile * kRows;
      h.rows = min(kRows, it.r.fresh * p.group - h.row0);
      h.token0 = it.r.token0;
    }
    p.headers[cta] = h;
  }
  const unsigned ring = smem_addr(smem) + warp * kSlots * 2 * kBytes;
  const unsigned bar0 = smem_addr(bars + warp * kSlots);
  float* wo = reinterpret_cast<float*>(smem + kWarps * kSlots * 2 * kBytes);  // [warp][row][dim]
  float2* ws = reinterpret_cast<float2*>(wo + kWarps * kRows * D);             // [warp][row] (ref, sum)
  const int per_page_shift = p.page_shift - 4;
  int turn = 0;  // units this warp has sent through its ring before this piece

  while (it.pos < it.end) {
    // ---- one piece: units [it.unit, last_unit) of a segment
    const int last_unit = min(it.r.units, it.unit + it.end - it.pos);
    const int length = it.r.length, fresh = it.r.fresh, token0 = it.r.token0;
    const int row0 = it.tile * kRows, rows = min(kRows, fresh * p.group - row0);
    // q's rows, asked for before the table is waited for: row g of each 8-row tile, dims 32 G + 8 t .. + 7.
    uint4 qw[NG];
    const int row = g, at = row0 + row, token = by_group(p, at);
    const unsigned short* src = p.q + (token0 + token) * p.q_stride +
                                static_cast<long long>(kvh * p.group + at - token * p.group) * D;
#pragma unroll
    for (int G = 0; G < NG; ++G)
      qw[G] = row < rows ? *reinterpret_cast<const uint4*>(src + 32 * G + 8 * t) : make_uint4(0u, 0u, 0u, 0u);
    // Units of two blocks (32 tokens) go to the warps in turn; unit s of this warp begins at block first_block + 2 * (warp +
    // 4 * s).
    const int first_block = 2 * it.unit, last_block = (length + kKvBlock - 1) / kKvBlock;
    const int units = p.whole ? (length + kUnitTokens - 1) / kUnitTokens : last_unit - it.unit;
    const int count = max(0, (units - warp + kWarps - 1) / kWarps);
    const int* table = p.table + static_cast<long long>(it.request) * p.width;

    // ---- the warp's ring. Lane 2 u + b keeps the address of block b of unit u of a window of 16 units and issues its copy;
    // a page that is no page (or a block behind the last) is not copied, its tokens are masked.
    const unsigned char* source = nullptr;
    unsigned issued_ok = 0;  // blocks of the window being issued that have a page
    auto issue = [&](int s) {
      const int u = s & 15, slot = (turn + s) % kSlots;
      if (u == 0) {
        const int block = first_block + 2 * (warp + kWarps * (s + (lane >> 1))) + (lane & 1);
        const bool there = block < last_block;
        const int id = there ? table[block >> per_page_shift] : -1;
        const bool page = id >= 0 && id < p.num_pages;
        if (there && !page) record_status(p.status, kStatusBadPage);
        const long long at =
            ((static_cast<long long>(id) * p.kv_heads + kvh) << per_page_shift) + (block & ((1 << per_page_shift) - 1));
        source = page ? p.pages + at * kBytes : nullptr;
        issued_ok = __ballot_sync(0xffffffffu, page);
      }
      if ((lane >> 1) == u) {
        if (turn + s >= kSlots) fence_proxy_async_smem();  // the slot's last blocks were read by ordinary loads
        mbar_arrive_expect_tx(bar0 + 8 * slot, source ? kBytes : 0);
        if (source) bulk_g2s(ring + (slot * 2 + (lane & 1)) * kBytes, source, kBytes, bar0 + 8 * slot);
      }
    };
    for (int s = 0; s < kSlots && s < count; ++s) issue(s);

    // ---- q as B fragments, times a power of two of its row
    unsigned qb[NG][4];
    unsigned offset[2];     // B fragment of -8 * 2^-24 * sum q, see below
    float rs[2];            // score factor of rows 2 t, 2 t + 1: scale * log2(e) * 2^24 / (q's power of two)
    int limit[2];           // positions that rows 2 t, 2 t + 1 see
    float top = 0.0f;
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const unsigned u[4] = {qw[G].x, qw[G].y, qw[G].z, qw[G].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = fmaxf(top, fmaxf(fabsf(kBf16 ? bf16lo(u[e]) : f16lo(u[e])), fabsf(kBf16 ? bf16hi(u[e]) : f16hi(u[e]))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ef = max(static_cast<int>(__float_as_uint(top) >> 23), 15);
    const float up = __uint_as_float(static_cast<unsigned>(268 - ef) << 23);  // 2^(141 - ef): the maximum becomes < 2^15
    // At most the largest float: scores that far apart are one-hot at any factor of that size, and 0 stays 0.
    const float mine_rs =
        fminf(p.scale_log2e * __uint_as_float(static_cast<unsigned>(ef - 14) << 23) * 16777216.0f, 3.402823466e38f);
    float c0[NG][2];  // of rows 2 t, 2 t + 1
#pragma unroll
    for (int G = 0; G < NG; ++G) {
      const unsigned u[4] = {qw[G].x, qw[G].y, qw[G].z, qw[G].w};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = (kBf16 ? bf16lo(u[e]) : f16lo(u[e])) * up;
        x[2 * e + 1] = (kBf16 ? bf16hi(u[e]) : f16hi(u[e])) * up;
      }
      // nibble pairs (0, 4), (1, 5) * 16, (2, 6), (3, 7) * 16
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float by = e & 1 ? 0.0625f : 1.0f;
        qb[G][e] = pack_h2(x[e] * by, x[e + 4] * by);
      }
      // -2^-21 for the pairs as they are, 16 times that for those that were divided by 16
      constexpr unsigned kOne = 0x80088008u, kSixteen = 0x80808080u;
      const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      float sum[4];
      mma_f16(sum, kOne, kOne, kSixteen, kSixteen, qb[G][0], qb[G][1], zero);
      mma_f16(sum, kOne, kOne, kSixteen, kSixteen, qb[G][2], qb[G][3], sum);
      c0[G][0] = sum[0], c0[G][1] = sum[1];
    }
    // The offsets as a B fragment (k x rows) for an A of the tokens' K scales, in two FP16 terms (2^-25 at worst): slots
    // k = 2 t, 2 t + 1 (and + 8) of lane (g, t) take a pair of groups' high or low term of row g.
#pragma unroll
    for (int half = 0; half < 2; ++half) offset[half] = 0u;
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) {
      float mine[2];  // groups 2 i, 2 i + 1 of row g: lane g / 2 holds rows g & ~1, (g & ~1) + 1
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float even = __shfl_sync(0xffffffffu, c0[2 * i + h][0], g >> 1);
        const float odd = __shfl_sync(0xffffffffu, c0[2 * i + h][1], g >> 1);
        mine[h] = g & 1 ? odd : even;
      }
      const unsigned high = pack_h2(mine[0], mine[1]);
      const unsigned low = pack_h2(mine[0] - lo_f32(high), mine[1] - hi_f32(high));
      if (NG == 8) {
        if (t == i) offset[0] = high, offset[1] = low;
      } else {
        if (t == i) offset[0] = high;
        if (t == i + NG / 2) offset[0] = low;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // from a lane that holds row 2 t + e as its row g
      rs[e] = __shfl_sync(0xffffffffu, mine_rs, (2 * t + e) * 4);
      const int r = 2 * t + e;
      limit[e] = r < rows ? length - fresh + by_group(p, row0 + r) + 1 : 0;
    }
    // The smallest limit of the tile; rows that are not there are never written, masked or not.
    const int least = length - fresh + by_group(p, row0) + 1;

    // ones = sum of P' per group; groups 2 i and 2 i + 1 share an accumulator (rows 0-7 and 8-15 of the A operand).
    float o[2 * NG][4], ones[NG / 2][4], l[2], nref[2];  // nref = -ref
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < NG / 2; ++i) ones[i][e] = 0.0f;
    l[0] = l[1] = 0.0f;
    nref[0] = nref[1] = -kNegInf;
    const int tv = g >> 1;              // the token pair whose V scales this lane holds
    float range = kWeakRange;           // e of the V scales
    unsigned above = kAboveWeak;        // bits that scales of the range do not have
    unsigned ok = 0;            // blocks of the window being read that have a page
    bool live = true;

    for (int s = 0; s < count; ++s) {
      const int slot = (turn + s) % kSlots;
      if ((s & 15) == 0) ok = issued_ok;
      const int pos = (first_block + 2 * (warp + kWarps * s)) * kKvBlock;
      live = mbar_wait(bar0 + 8 * slot, (turn + s) / kSlots & 1);
      live = __all_sync(0xffffffffu, live);
      if (!live) {  // leave, after a bounded wait for the warp's other copies in flight
        if (lane == 0) record_status(p.status, kStatusMbarTimeout);
        for (int k = s + 1; k < count && k < s + kSlots; ++k)
          (void)mbar_wait(bar0 + 8 * ((turn + k) % kSlots), (turn + k) / kSlots & 1);
        break;
      }
      const unsigned at = ring + slot * 2 * kBytes;

      // ---- S^T = K Q^T of tokens g, g + 8 of both blocks
      float x[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        unsigned kw[2][NG], kscale[2][NG / 2], kpair[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int quad = 0; quad < NQ; ++quad) {
            unsigned a[Q];
            lds_words<Q>(at + b * kBytes + quad * (256 * Q) + (g + 8 * j) * (16 * Q) + t * (4 * Q), a);
#pragma unroll
            for (int i = 0; i < Q; ++i) kw[j][quad * Q + i] = a[i];
          }
          lds_words<NG / 2>(at + b * kBytes + 16 * D + (g + 8 * j) * (2 * NG), kscale[j]);
          kpair[j] = lds32(at + b * kBytes + 16 * D + (g + 8 * j) * (2 * NG) + 4 * (t & (NG / 2 - 1)));
        }
        const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_f16(x[b], kpair[0], kpair[1], NG == 8 ? kpair[0] : 0u, NG == 8 ? kpair[1] : 0u, offset[0],
                offset[1], zero);
#pragma unroll
        for (int G = 0; G < NG; ++G) {
          const unsigned a = kw[0][G], c = kw[1][G], ah = a >> 8, ch = c >> 8;
          const float s0 = G & 1 ? hi_f32(kscale[0][G / 2]) : lo_f32(kscale[0][G / 2]);
          const float s1 = G & 1 ? hi_f32(kscale[1][G / 2]) : lo_f32(kscale[1][G / 2]);
          float acc[4];
          const float start[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_f16(acc, a & 0x000f000fu, c & 0x000f000fu, a & 0x00f000f0u, c & 0x00f000f0u, qb[G][0], qb[G][1],
                  start);
          mma_f16(acc, ah & 0x000f000fu, ch & 0x000f000fu, ah & 0x00f000f0u, ch & 0x00f000f0u, qb[G][2],
                  qb[G][3], acc);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float by = e & 2 ? s1 : s0;
            x[b][e] = fmaf(acc[e], by, x[b][e]);
          }
        }
      }

      // ---- V scales of tokens 2 tv, 2 tv + 1 (j = 0) and 2 tv + 8, 2 tv + 9 (j = 1), and scores against the reference
      unsigned sv[2][2][NG];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          lds_words<NG>(at + b * kBytes + 17 * D + (j * 4 + tv) * (4 * NG), sv[b][j]);
      float y[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[b][e] = fmaf(x[b][e], rs[e & 1], nref[e & 1]);
      if (pos + 2 * kKvBlock > least || (ok >> 2 * (s & 15) & 3u) != 3u) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const bool page = ok >> (2 * (s & 15) + b) & 1;
          const int end = page ? length : 0, first = pos + b * kKvBlock;
#pragma unroll
          for (int j = 0; j < 2; ++j) {  // tokens that are not there: scales whatever they are become 0
            const int token = first + 8 * j + 2 * tv;
            const unsigned keep = (token < end ? 0x0000ffffu : 0u) | (token + 1 < end ? 0xffff0000u : 0u);
#pragma unroll
            for (int G = 0; G < NG; ++G) sv[b][j][G] &= keep;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (first + g + (e & 2 ? 8 : 0) >= min(end, limit[e & 1])) x[b][e] = y[b][e] = kNegInf;
        }
      }

      // ---- does the reference still hold, and are the V scales in the range?
      unsigned any = 0u;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int G = 0; G < NG; ++G) any |= sv[b][0][G] | sv[b][1][G];
      float most = kNegInf;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; e += 2) most = fmaxf(most, fmaxf(y[b][e], y[b][e + 1]));
      if (__any_sync(0xffffffffu, most > kMoveAt - range || (any & above))) {
        any = __reduce_or_sync(0xffffffffu, any);
        const float before = range;
        if (any & kAbovePlain)
          range = kStrongRange, above = 0u;
        else if (any & kAboveWeak)
          range = fmaxf(range, kPlainRange), above &= kAbovePlain;
        const float wider = range - before;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(fmaxf(x[0][e], x[0][e + 2]), fmaxf(x[1][e], x[1][e + 2]));
          top = mul_rn(top, rs[e]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const float was = -nref[e], now = fmaxf(top - kRefBelow + range, was + wider);
          if (was != kNegInf) {
            const float factor = exp2_fast(was - now);
            l[e] *= factor;
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) o[i][e] *= factor, o[i][e + 2] *= factor;
#pragma unroll
            for (int i = 0; i < NG / 2; ++i) ones[i][e] *= factor, ones[i][e + 2] *= factor;
          }
          nref[e] = -now;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              // Scores past 2^27 know the weight only to a power of two: the largest score's is in range here, where a
              // fused product would leave the score's own rounding, and no weight passes the limit.
              const float v = x[b][e + h], score = mul_rn(v, rs[e]) - now, limit = kMoveAt - range;
              y[b][e + h] = v == kNegInf ? kNegInf : score > limit ? limit : score;
            }
        }
      }

      // ---- P, its sums, P' per group as B fragments (rows x tokens), O^T += V^T P'
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        unsigned vw[2][NG];
        float w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int quad = 0; quad < NQ; ++quad) {
            unsigned a[Q];
            lds_words<Q>(at + b * kBytes + 8 * D + quad * (256 * Q) + j * (128 * Q) + g * (16 * Q) + t * (4 * Q), a);
#pragma unroll
            for (int i = 0; i < Q; ++i) vw[j][quad * Q + i] = a[i];
          }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = exp2_fast(y[b][e]);
        l[0] += w[0] + w[2];
        l[1] += w[1] + w[3];
#pragma unroll
        for (int G = 0; G < NG; ++G) {
          const unsigned a = vw[0][G], c = vw[1][G], ah = a >> 8, ch = c >> 8;
          const float s0 = f16_to_f32(static_cast<unsigned short>(sv[b][0][G] >> (16 * (g & 1))));
          const float s1 = f16_to_f32(static_cast<unsigned short>(sv[b][1][G] >> (16 * (g & 1))));
          const f2 p0 = mul2({w[0], w[1]}, {s0, s0}), p1 = mul2({w[2], w[3]}, {s1, s1});
          const unsigned b0 = transpose8x8(pack_h2(p0.x, p0.y)), b1 = transpose8x8(pack_h2(p1.x, p1.y));
          mma_f16(o[2 * G], a & 0x000f000fu, a & 0x00f000f0u, c & 0x000f000fu, c & 0x00f000f0u, b0, b1,
                  o[2 * G]);
          mma_f16(o[2 * G + 1], ah & 0x000f000fu, ah & 0x00f000f0u, ch & 0x000f000fu, ch & 0x00f000f0u, b0, b1,
                  o[2 * G + 1]);
          constexpr unsigned kOnes = 0x3c003c00u;
          if (G & 1)
            mma_f16(ones[G / 2], 0u, kOnes, 0u, kOnes, b0, b1, ones[G / 2]);
          else
            mma_f16(ones[G / 2], kOnes, 0u, kOnes, 0u, b0, b1, ones[G / 2]);
        }
      }
      __syncwarp();
      if (s + kSlots < count) issue(s + kSlots);
    }

    turn += count;

    // ---- the warps' sums to shared memory, joined there
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const int row = 2 * t + e;
      if (g == 0) ws[warp * kRows + row] = make_float2(-nref[e], sum);
      float* to = wo + (warp * kRows + row) * D;
#pragma unroll
      for (int G = 0; G < NG; ++G) {
        const float mass = ones[G / 2][G & 1 ? e + 2 : e];
        const float eight = 8.0f * mass;
        float4 v;
        v.x = fmaf(o[2 * G][e], 16777216.0f, -eight);
        v.y = fmaf(o[2 * G][e + 2], 1048576.0f, -eight);
        v.z = fmaf(o[2 * G + 1][e], 16777216.0f, -eight);
        v.w = fmaf(o[2 * G + 1][e + 2], 1048576.0f, -eight);
        *reinterpret_cast<float4*>(to + 32 * G + 4 * g) = v;
      }
    }
    __syncthreads();
    constexpr int kVec = D / 4;  // float4s of a row
    for (int at = tid; at < rows * kVec; at += kThreads) {
      const int row = at / kVec, c = at - row * kVec;
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ws[w * kRows + row].x);
      float den = 0.0f;
      float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 st = ws[w * kRows + row];
        if (st.x == kNegInf && st.y == 0.0f) continue;  // a warp that saw nothing of this row
        const float f = exp2_fast(st.x - top);
        const float4 v = *reinterpret_cast<const float4*>(wo + (w * kRows + row) * D + 4 * c);
        den = fmaf(f, st.y, den);
        num.x = fmaf(f, v.x, num.x), num.y = fmaf(f, v.y, num.y), num.z = fmaf(f, v.z, num.z), num.w = fmaf(f, v.w, num.w);
      }
      if (it.unit == 0 && last_unit == it.r.units) {
        const float by = den == 0.0f ? 0.0f : __frcp_rn(den);  // a row that sees no position: 0
        const int r = row0 + row, token = by_group(p, r);
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
      } else {  // record 0: a piece that continues a segment, record 1: one that begins it
        const long long rec = record_of(p, cta, kvh, it.unit == 0) + row;
        if (c == 0) p.stats[rec] = make_float2(top, den);
        reinterpret_cast<float4*>(p.sums + rec * D)[c] = num;
      }
    }
    it.pos += last_unit - it.unit;
    if (!__syncthreads_and(live)) return;  // a copy never came: the status says so, nothing more is asked for
    if (it.pos < it.end) next_segment(p, it);
  }
}

// Joins what the CTAs first .. last left of one segment (tile of a request, kv head): record 1 of the first, record 0 of the
// others. Its rows * D / 4 columns of 4 are dealt to the CTAs behind the first, `each` (a power of two) to a CTA, whose
// threads share the records of a column in 128 / each classes: every thread reads its records in one go against a reference
// of its own; classes meet by butterflies inside a warp and in order through shared memory.
template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads) kv_combine_kernel(const KvAttnParams p) {
  __shared__ float4 part[kThreads];
  __shared__ float2 part_stat[kThreads];
  grid_dependency_wait();
  grid_launch_dependents();
  const Header h = p.headers[blockIdx.x];
  if (h.last < 0) return;
  const int kvh = blockIdx.y, tid = threadIdx.x;
  constexpr int kCols = D / 4;
  const int parts = h.last - h.first, records = parts + 1, mine = blockIdx.x - h.first - 1;
  const int total = h.rows * kCols, share = (total + parts - 1) / parts;
  int shift = 0;
  while ((1 << shift) < share && shift < 7) ++shift;
  const int each = 1 << shift, classes = kThreads >> shift, cls = tid >> shift;
  for (int base = mine * each; base < total; base += parts * each) {
    const int at = base + (tid & (each - 1)), row = at / kCols, col = at - row * kCols;
    float top = kNegInf, den = 0.0f;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = cls; k0 < records; k0 += 4 * classes) {
      float2 st[4];
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + j * classes;
        st[j] = make_float2(kNegInf, 0.0f);
        v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < records && at < total) {
          const long long record = record_of(p, h.first + k, kvh, k == 0) + row;
          st[j] = __ldcg(p.stats + record);
          v[j] = __ldcg(reinterpret_cast<const float4*>(p.sums + record * D) + col);
        }
      }
      float now = top;
#pragma unroll
      for (int j = 0; j < 4; ++j) now = fmaxf(now, st[j].x);
      const float keep = top == kNegInf ? 0.0f : exp2_fast(top - now);
      if (top != kNegInf) den *= keep, num.x *= keep, num.y *= keep, num.z *= keep, num.w *= keep;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (st[j].x == kNegInf && st[j].y == 0.0f) continue;  // a piece that saw nothing of this row
        const float f = exp2_fast(st[j].x - now);
        den = fmaf(f, st[j].y, den);
        num.x = fmaf(f, v[j].x, num.x), num.y = fmaf(f, v[j].y, num.y);
        num.z = fmaf(f, v[j].z, num.z), num.w = fmaf(f, v[j].w, num.w);
      }
      top = now;
    }
    if (each < 32) {  // the classes inside the warp
      float all = top;
      for (int d = each; d < 32; d <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, d));
      if (!(top == kNegInf && den == 0.0f)) {
        const float f = exp2_fast(top - all);
        den *= f, num.x *= f, num.y *= f, num.z *= f, num.w *= f;
      }
      top = all;
      for (int d = each; d < 32; d <<= 1) {
        den += __shfl_xor_sync(0xffffffffu, den, d);
        num.x += __shfl_xor_sync(0xffffffffu, num.x, d), num.y += __shfl_xor_sync(0xffffffffu, num.y, d);
        num.z += __shfl_xor_sync(0xffffffffu, num.z, d), num.w += __shfl_xor_sync(0xffffffffu, num.w, d);
      }
    }
    const int step = max(each, 32);  // threads between two classes that are left
    part[tid] = num;
    part_stat[tid] = make_float2(top, den);
    __syncthreads();
    if (tid < each && at < total) {
      for (int c = tid + step; c < kThreads; c += step) top = fmaxf(top, part_stat[c].x);
      den = 0.0f, num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int c = tid; c < kThreads; c += step) {
        const float2 st = part_stat[c];
        if (st.x == kNegInf && st.y == 0.0f) continue;
        const float f = exp2_fast(st.x - top);
        const float4 v = part[c];
        den = fmaf(f, st.y, den);
        num.x = fmaf(f, v.x, num.x), num.y = fmaf(f, v.y, num.y), num.z = fmaf(f, v.z, num.z), num.w = fmaf(f, v.w, num.w);
      }
      const float by = den == 0.0f ? 0.0f : __frcp_rn(den);
      const int r = h.row0 + row, token = by_group(p, r);
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
  bool whole;         // segments go to CTAs whole
  int ctas;           // per kv head
  bool combine;
  size_t headers, stats, sums, total;  // scratch offsets
  size_t smem;
};

int kv_plan(int requests, int width, int page_size, int heads, int kv_heads, int dim, int max_new, KvPlan* plan) {
  if (requests <= 0 || width <= 0 || heads <= 0 || kv_heads <= 0 || max_new <= 0) return KLAB_E_INVALID;
  if (requests > kKvMaxRequests || kv_heads > 65535 || heads % kv_heads || heads / kv_heads > KLAB_KV_MAX_GROUP ||
      max_new > kKvMaxNew || !kv_dim_ok(dim) || !kv_page_size_ok(page_size) ||
      static_cast<long long>(width) * page_size > INT_MAX)
    return KLAB_E_SHAPE;
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc) return rc;
  const int tiles = (heads / kv_heads * max_new + kRows - 1) / kRows;
  const long long units = (static_cast<long long>(width) * page_size - 1) / kUnitTokens + 1;
  plan->whole = units <= kWholeUnits;
  const long long most = static_cast<long long>(requests) * tiles * (plan->whole ? 1 : units);
  if (most > INT_MAX) return KLAB_E_SHAPE;
  // One CTA for each place on the machine, dealt evenly to the kv heads; fewer where the table cannot hold more shares.
  const long long places = static_cast<long long>(sms) * kv_resident(dim / kKvGroup) / kv_heads;
  const long long shares = plan->whole ? most : (most + kMinShare - 1) / kMinShare;
  plan->ctas = static_cast<int>(shares < places ? shares : places > 1 ? places : 1);
  plan->combine = plan->ctas > 1 && !plan->whole;
  plan->headers = 0;
  plan->stats = (static_cast<size_t>(plan->ctas) * sizeof(Header) + 127) / 128 * 128;
  const size_t records = plan->combine ? static_cast<size_t>(plan->ctas) * kv_heads * 2 * kRows : 0;
  plan->sums = plan->stats + (records * 8 + 127) / 128 * 128;
  plan->total = plan->sums + records * dim * 4;
  const size_t ring = static_cast<size_t>(kWarps) * kSlots * 2 * kv_block_bytes(dim);
  const size_t join = static_cast<size_t>(kWarps) * kRows * (dim * 4 + 8);
  plan->smem = ring + join;
  return 0;
}

template <int NG, bool kBf16>
int run_kv(const KvAttnParams& p, const KvPlan& plan, cudaStream_t stream) {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (!(ready.load() >> dev & 1)) {
    err = cudaFuncSetAttribute(kv_attn_kernel<NG, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(plan.smem));
    if (err != cudaSuccess) return err;
    ready.fetch_or(1ull << dev);
  }
  const dim3 grid(static_cast<unsigned>(plan.ctas), static_cast<unsigned>(p.kv_heads));
  int rc = launch_dependent(kv_attn_kernel<NG, kBf16>, grid, kThreads, plan.smem, stream, p);
  if (rc || !plan.combine) return rc;
  return launch_dependent(kv_combine_kernel<32 * NG, kBf16>, grid, kThreads, 0, stream, p);
}

template <bool kBf16>
int dispatch_kv(int dim, const KvAttnParams& p, const KvPlan& plan, cudaStream_t stream) {
  switch (dim) {
    case 64: return run_kv<2, kBf16>(p, plan, stream);
    case 128: return run_kv<4, kBf16>(p, plan, stream);
    default: return run_kv<8, kBf16>(p, plan, stream);
  }
}

int run_attention(const void* q, long long q_stride, int dtype, const void* pages, const int* table,
                 const int* lengths, const int* starts, void* out, void* scratch, long long scratch_bytes, int tokens,
                 int requests, int width, int num_pages, int page_size, int heads, int kv_heads, int dim, int max_new,
                 float scale, void* stream, bool fill) {
  if (!q || !pages || !table || !lengths || !starts || !out || !scratch || tokens <= 0 || num_pages <= 0)
    return KLAB_E_INVALID;
  if (dtype != KLAB_DT_BF16 && dtype != KLAB_DT_F16) return KLAB_E_UNSUPPORTED;
  if (!(scale > 0.0f) || scale > 3.0e38f) return KLAB_E_INVALID;
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
  p.headers = reinterpret_cast<Header*>(base + plan.headers);
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
  p.group_div = (65536 + p.group - 1) / p.group;
  p.max_length = width * page_size;
  p.whole = plan.whole;
  p.max_new = max_new;
  p.fill = fill;
  p.scale_log2e = scale * 1.44269504088896340736f;
  return dtype == KLAB_DT_BF16 ? dispatch_kv<true>(dim, p, plan, static_cast<cudaStream_t>(stream))
                               : dispatch_kv<false>(dim, p, plan, static_cast<cudaStream_t>(stream));
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
  return klab::run_attention(q, q_stride, dtype, pages, table, lengths, starts, out, scratch, scratch_bytes, tokens, requests,
                             width, num_pages, page_size, heads, kv_heads, dim, max_new, scale, stream, false);
}

KLAB_API int klab_kv_attention_new(const void* q, long long q_stride, int dtype, const void* pages, const int* table,
                               const int* lengths, const int* starts, void* out, void* scratch, long long scratch_bytes,
                               int tokens, int requests, int width, int num_pages, int page_size, int heads,
                               int kv_heads, int dim, int max_new, float scale, void* stream) {
  return klab::run_attention(q, q_stride, dtype, pages, table, lengths, starts, out, scratch, scratch_bytes, tokens, requests,
                             width, num_pages, page_size, heads, kv_heads, dim, max_new, scale, stream, true);
}

}  // extern "C"
