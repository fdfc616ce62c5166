// Low-rank adapters of many requests beside a shared projection:
//   y[m] = x[m] W^T + c_a (x[m] A_a^T) B_a^T,  a = ids[m] (-1: x[m] W^T alone),
// BF16 x, A [S, r, K], B [S, N, r]; W in any format that the projections take with BF16 x and one scale tensor.
//
// BF16, INT8 per-row and E2M1/FP16-per-32 weights with 16-byte rows: two launches.
//   adapter_stream_kernel reads, for each tile of 16 tokens, W once and every token's A (one adapter's again for each of
//   its tokens, from L2), as one list of work: a block is 128 rows (8 warps x 16 rows) of W, or 8 groups of 16 rows of the
//   tokens' A (token m's adapter against x, of which column m counts), and a unit is 128 or 256 bytes of each of its rows.
//   The units, block by block, are cut into equal shares, two CTAs to an SM (a block into shares of its own where that
//   costs little), so any N and K and any number of adapters keep every SM reading to the end. A warp copies its units into
//   a ring of its own (cp.async, whole runs of a row at a time: 64-byte runs straight into registers measured 36.9 us where
//   this took 31.3) and multiplies its 16 rows by up to 16 tokens on mma.m16n8k16 with FP32 sums: lane (g, t) takes 16
//   bytes of rows g and g + 8 as A fragments (the k slots of an MMA may be any columns as long as x's are the same); x lies
//   in shared memory in fragment order. Weights, INT8 codes and E2M1 values are exact in BF16 and meet x as it is, so every
//   product is exact whatever else the row holds; E2M1 groups are multiplied by their FP16 scale in FP32. What a share
//   holds of a block goes to scratch in FP32.
//   adapter_join_kernel adds the shares of each block in order, forms t = c (x A^T) the same way, and writes
//   y + t . B_a[n] with one rounding.
//   More than 16 rows are tiles of 16 that read W again each, from L2 where it holds it (the projections alone do the same,
//   and take longer: BF16 M = 128 1022 us against 126, INT8 173 against 131).
// Other formats: shrink_kernel (t in FP32), the projection as it is with FP32 output, expand_kernel (the sum, one rounding).
// Either form takes parts of the rows one behind the other where the FP32 sums of all would pass 64 MiB.
//
// What bounds it: BF16 the copies while the units stream (M = 16, 14336 -> 4096, rank 64: 148 MB of W and distinct adapters
// in 31.8 us, 4.7 TB/s over all; issue slots 36 % busy, warps waiting for data), around it launch, the staging of x and the
// join (3 us). INT8 and E2M1 are bound by issue too (51 and 55 % busy, the ALU pipe 60 and 48 %): a code costs two
// instructions on its way to BF16. M = 1, 4096 -> 4096 BF16 7.5 us; M = 8, 4096 -> 14336 INT8 17.1; M = 16 E2M1 25.6.
#include <atomic>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "klab_b200.h"
#include "klab_kernels.h"
#include "launch.cuh"

namespace klab {
namespace {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kRanks = 4;  // rows of A per CTA
constexpr int kMaxRank = KLAB_ADAPTER_MAX_RANK;

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
    // Not by read-only loads: this kernel may already be here while the launch before writes what it reads.
    const uint4 xv = __ldcg(x + i);
    uint4 av[kRanks];
#pragma unroll
    for (int j = 0; j < kRanks; ++j) av[j] = __ldcg(a[j] + i);
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
      const uint4 w = __ldcg(b + j);
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

// ---------------------------------------------------------------- streaming form

enum AdKind : int { AD_BF16 = 0, AD_I8 = 1, AD_FP4 = 2 };

constexpr int kAsWarps = 8;
constexpr int kAsThreads = 32 * kAsWarps;
constexpr int kAsRows = 16 * kAsWarps;   // rows of a block
constexpr int kAsTokens = 16;            // tokens of a call's tile
constexpr int kAsWindow = 32 * 1024;     // x in shared memory
constexpr int kAsMinShare = 2;           // units of a share: fewer would only add records to join
// Every block gets CTAs of its own where shares grow by at most so many units: a second piece stages x again and starts its
// ring anew. M = 4, 1856 -> 1000 BF16 4.7 us (equal shares 6.1), M = 16, 4096 -> 14336 E2M1 25.6 (26.3), M = 8 INT8 17.1
// (17.3); 8 units gain nothing more.
constexpr int kAsSlack = 4;
// CTAs to a place from which on blocks are not cut: the last round is then short, and no sums are joined. 4096 -> 14336 BF16,
// M = 64 67 us (with 1: 76), M = 128 126 (137); 4096 -> 4096 INT8, M = 1024 276 us (with 8: 333). Cut for one tile alone, as
// tiles of 16 rows run one behind the other, M = 128 took 158 and M = 2048, 4096 -> 4096 880 (599 now).
constexpr int kAsWaves = 4;
// FP32 sums that one pair of launches leaves; calls of more rows are made of several, on the same scratch.
constexpr size_t kAsScratch = 64ull << 20;

// Bytes of a row in a unit and units of a warp in flight, by the kind of W. Longer runs of a row are better for HBM, shorter
// units even out short shares: M = 8, 4096 -> 14336 BF16 takes 23.3 us with 256-byte units and 24.6 with 128 (M = 16,
// 14336 -> 4096 31.8 and 31.6), the same in INT8 (half the bytes) 17.7 and 17.1.
__host__ __device__ constexpr int as_unit(int kind) { return kind == AD_BF16 ? 256 : 128; }
__host__ __device__ constexpr int as_depth(int kind) { return kind == AD_BF16 ? 2 : 3; }

// A warp's ring in shared memory: units of 16 rows.
__host__ __device__ constexpr int as_slot(int kind) { return 16 * as_unit(kind); }
__host__ __device__ constexpr int as_smem(int kind) { return kAsWindow + kAsWarps * as_depth(kind) * as_slot(kind); }

// Columns per 64-byte step and 16-byte x pieces (8 columns of a token) per lane and step.
__host__ __device__ constexpr int as_cols(int kind) { return kind == AD_BF16 ? 32 : kind == AD_I8 ? 64 : 128; }
__host__ __device__ constexpr int as_pieces(int kind) { return as_cols(kind) / 32; }

struct StreamParams {
  const unsigned short* x;
  const unsigned char* w;
  const void* side;      // INT8: FP32 [N]; E2M1: FP16 [N, K / 32]
  const unsigned short* a;
  const unsigned short* b;
  const float* c;
  const int* ids;
  float* w_part;         // [tile][block][piece][token][128]
  float* a_part;         // [tile][block][piece][128]
  void* out;
  int* status;
  long long row_bytes;
  int m, n, k, rank, adapters, ldo, out_f32;
  int groups;                    // 16-row groups of an adapter's A
  int a_blocks, w_blocks;        // per tile of 16 tokens
  int a_units, w_units;          // units of a block
  int share, a_pieces, w_pieces; // units of a CTA; most shares that meet in a block
  int a_parts, w_parts;          // CTAs of a block where none takes parts of two (w_parts = 0: equal shares)
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// INT8 codes and E2M1 values are taken times 2^-24, which the join takes back: their scales, which bring a sum into range,
// come after it, and without it |x| of 2^121 makes a sum of codes infinite whose result is not. (Products of |x| under 2^-102
// then reach FP32's subnormals.)
constexpr float kAsUp = 16777216.0f;

// Four INT8 codes times 2^-24 as two BF16 pairs, exact: with the code's low 7 bits u and its sign s, 0x3700 | u is
// (128 + u) 2^-24 and 0x3700 | s << 7 is (128 + 128 s) 2^-24.
__device__ __forceinline__ void i8_pairs(unsigned w, unsigned& lo, unsigned& hi) {
  const unsigned u = w & 0x7f7f7f7fu, s = w & 0x80808080u;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(__byte_perm(u, 0x37373737u, 0x4140)), "r"(__byte_perm(s, 0x37373737u, 0x4140)));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(__byte_perm(u, 0x37373737u, 0x4342)), "r"(__byte_perm(s, 0x37373737u, 0x4342)));
}

// E2M1 values J and J + 4 of a word times 2^-24 as a BF16 pair, exact: the code's two exponent bits and one mantissa bit at
// BF16's lowest exponent bits and highest mantissa bit are the value times 2^-126, BF16 subnormal included.
template <int J>
__device__ __forceinline__ unsigned e2m1_pair(unsigned w) {
  const unsigned size = (J == 0 ? w << 6 : J == 1 ? w << 2 : J == 2 ? w >> 2 : w >> 6) & 0x01c001c0u;
  const unsigned by = ((J == 3 ? w : w << (12 - 4 * J)) & 0x80008000u) ^ 0x72807280u;  // +- 2^102
  unsigned d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(size), "r"(by));
  return d;
}

__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// One piece of a share: units [u0, u1) of a block of kind KIND, for this warp's 16 rows at `base` (nullptr: no rows), of
// which `rows` exist; `ring` is the warp's ring. Sums of row g (+ 8) and tokens 2 t (+ 1) of each
// 8-token block end in `sum`.
template <int KIND, int NB, int UNIT, int DEPTH>
__device__ __forceinline__ void stream_piece(const StreamParams& p, const unsigned char* base, long long row_bytes,
                                             const unsigned short* scales, int rows, int u0, int u1, int token0,
                                             unsigned char* xs, unsigned ring, float (&sum)[NB][4], bool first) {
  constexpr int P = as_pieces(KIND), COLS = as_cols(KIND);
  constexpr int kUnitSteps = UNIT / 64, kSlot = 16 * UNIT;  // an MMA step takes 64 bytes of each row
  constexpr int kStepBytes = P * NB * 512;  // x of one step
  constexpr int kSteps = kAsWindow / kStepBytes / kUnitSteps * kUnitSteps;  // steps of a window
  const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const bool has0 = base && g < rows, has1 = base && g + 8 < rows;
  // Copies go by rows: kRun lanes take a row's bytes of the unit, so HBM sees whole runs of sectors.
  constexpr int kRun = UNIT / 16, kRowsAtOnce = 32 / kRun;
  const int sub = lane / kRun, chunk = lane % kRun;
  const unsigned char* mine = base + sub * row_bytes + 16 * chunk;
  // Chunk c of row r at c ^ 4 (r mod 2) for fragments of 16 bytes (rows g, four chunks each), at c ^ (r mod 8) for words of
  // a chunk (rows g): neither meets a bank twice.
  static_assert(KIND != AD_FP4 || kRowsAtOnce == 4, "row j + sub, j a multiple of 4: the chunk's bit 2 turns with j's");
  const unsigned to0 = ring + sub * UNIT + ((KIND == AD_FP4 ? chunk ^ sub : chunk ^ ((sub & 1) << 2)) << 4);
  int slot = 0;
  auto copy = [&](int u) {  // unit u into the ring's next slot; nothing past the piece, the rows or a row's end
    const long long at = static_cast<long long>(u) * UNIT;
    const bool in = u < u1 && base && at + 16 * chunk < row_bytes;
    const unsigned to = to0 + slot * kSlot;
#pragma unroll
    for (int j = 0; j < 16; j += kRowsAtOnce) {
      const bool there = in && j + sub < rows;
      copy16((KIND == AD_FP4 ? to ^ ((j & 4) << 4) : to) + j * UNIT,
             there ? static_cast<const void*>(mine + at + j * row_bytes) : p.x, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
  };
  // E2M1: the scales of rows g and g + 8 for the four steps of a unit, a unit ahead in registers.
  const int srow = p.k / 32;  // scales of a row, four to a step
  const unsigned short* q0 = scales + static_cast<long long>(g) * srow;
  const unsigned short* q1 = q0 + 8ll * srow;
  const bool scales_vec = (srow & 3) == 0 && (reinterpret_cast<uintptr_t>(scales) & 7) == 0;
  constexpr int kHeld = KIND == AD_FP4 ? kUnitSteps : 1;
  uint2 next0[kHeld], next1[kHeld];
  auto fetch_scales = [&](int u) {
    if constexpr (KIND == AD_FP4) {
#pragma unroll
      for (int j = 0; j < kUnitSteps; ++j) {
        const int i0 = 4 * (u * kUnitSteps + j);
        next0[j] = next1[j] = make_uint2(0u, 0u);
        if (scales_vec) {
          if (u < u1 && i0 < srow && has0) next0[j] = __ldcg(reinterpret_cast<const uint2*>(q0 + i0));
          if (u < u1 && i0 < srow && has1) next1[j] = __ldcg(reinterpret_cast<const uint2*>(q1 + i0));
        } else {
          unsigned short v[8] = {};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (u < u1 && i0 + i < srow) {
              if (has0) v[i] = __ldcg(q0 + i0 + i);
              if (has1) v[4 + i] = __ldcg(q1 + i0 + i);
            }
          next0[j] = make_uint2(v[0] | static_cast<unsigned>(v[1]) << 16, v[2] | static_cast<unsigned>(v[3]) << 16);
          next1[j] = make_uint2(v[4] | static_cast<unsigned>(v[5]) << 16, v[6] | static_cast<unsigned>(v[7]) << 16);
        }
      }
    }
  };
  // Before the previous kernel has ended only L2 is asked for the first units: it may still be writing them.
  if (first) {
    if (base && lane < min(rows, 16)) {
      const long long at = static_cast<long long>(u0) * UNIT, left = row_bytes - at;
      bulk_prefetch_l2(base + lane * row_bytes + at,
                       static_cast<unsigned>(min(left, static_cast<long long>(min(DEPTH, u1 - u0) * UNIT))));
    }
    grid_dependency_wait();
    grid_launch_dependents();
  }
#pragma unroll
  for (int j = 0; j < DEPTH; ++j) copy(u0 + j);
  fetch_scales(u0);
  const int s_end = kUnitSteps * u1;
  for (int s0 = kUnitSteps * u0; s0 < s_end; s0 += kSteps) {
    const int steps = min(kSteps, s_end - s0);
    // ---- x of the window: piece i of step s of lane (g, t) holds columns COLS s + (INT8: 16 t + 8 i, else 32 i + 8 t)
    __syncthreads();  // the last window is read
    const int pieces = steps * P * NB * 32;
    auto fetch = [&](int i) {
      const int ln = i & 31, piece = (i >> 5) / NB % P, s = (i >> 5) / (NB * P);
      const int col = COLS * (s0 + s) + (KIND == AD_I8 ? 16 * (ln & 3) + 8 * piece : 32 * piece + 8 * (ln & 3));
      const int token = token0 + (i >> 5) % NB * 8 + (ln >> 2);
      return i < pieces && token < p.m && col < p.k
                 ? __ldcg(reinterpret_cast<const uint4*>(p.x + static_cast<long long>(token) * p.k + col))
                 : make_uint4(0u, 0u, 0u, 0u);
    };
    constexpr int kBatch = 8;  // loads of x in flight per thread
    for (int i0 = tid; i0 < pieces; i0 += kBatch * kAsThreads) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) v[j] = fetch(i0 + j * kAsThreads);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kAsThreads;
        if constexpr (KIND == AD_FP4)  // columns j and j + 4 in a word, as e2m1_pair gives the weights
          v[j] = make_uint4(__byte_perm(v[j].x, v[j].z, 0x5410), __byte_perm(v[j].x, v[j].z, 0x7632),
                            __byte_perm(v[j].y, v[j].w, 0x5410), __byte_perm(v[j].y, v[j].w, 0x7632));
        if (i < pieces) reinterpret_cast<uint4*>(xs)[i] = v[j];
      }
    }
    __syncthreads();
    // ---- the window's steps
    float acc[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[b][e] = 0.0f;
    unsigned at = smem_addr(xs) + 16 * lane;
    for (int s = 0; s < steps; s += kUnitSteps, at += kUnitSteps * kStepBytes) {
      const int unit = (s0 + s) / kUnitSteps;
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
      __syncwarp();  // every lane's copies of the unit
      const unsigned from = ring + slot * kSlot + g * UNIT;
      uint4 v[kUnitSteps][2];
#pragma unroll
      for (int j = 0; j < kUnitSteps; ++j) {
        if constexpr (KIND == AD_FP4) {  // word t of the step's four groups
          unsigned c[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned at = from + (((4 * j + i) ^ g) << 4) + 4 * t;
            c[0][i] = lds32(at), c[1][i] = lds32(at + 8 * UNIT);
          }
          v[j][0] = make_uint4(c[0][0], c[0][1], c[0][2], c[0][3]), v[j][1] = make_uint4(c[1][0], c[1][1], c[1][2], c[1][3]);
        } else {
          const unsigned c = ((4 * j + t) ^ ((g & 1) << 2)) << 4;
          v[j][0] = lds128(from + c), v[j][1] = lds128(from + c + 8 * UNIT);
        }
      }
      uint2 now0[kHeld], now1[kHeld];
      if constexpr (KIND == AD_FP4) {
#pragma unroll
        for (int j = 0; j < kUnitSteps; ++j) now0[j] = next0[j], now1[j] = next1[j];
        fetch_scales(unit + 1);
      }
      __syncwarp();  // the slot is read
      copy(unit + DEPTH);
#pragma unroll
      for (int j = 0; j < kUnitSteps; ++j) {
        const uint4 v0 = v[j][0], v1 = v[j][1];
        const unsigned xat = at + j * kStepBytes;
        if constexpr (KIND == AD_BF16) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint4 xv = lds128(xat + b * 512);
            const unsigned a0[4] = {v0.x, v1.x, v0.y, v1.y}, a1[4] = {v0.z, v1.z, v0.w, v1.w};
            mma_bf16(acc[b], a0, xv.x, xv.y);
            mma_bf16(acc[b], a1, xv.z, xv.w);
          }
        } else if constexpr (KIND == AD_I8) {
          const unsigned c0[4] = {v0.x, v0.y, v0.z, v0.w}, c1[4] = {v1.x, v1.y, v1.z, v1.w};
          uint4 xv[NB][2];
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) xv[b][i] = lds128(xat + (i * NB + b) * 512);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            unsigned a[4];
            i8_pairs(c0[i], a[0], a[2]);
            i8_pairs(c1[i], a[1], a[3]);
#pragma unroll
            for (int b = 0; b < NB; ++b)
              mma_bf16(acc[b], a, i & 1 ? xv[b][i >> 1].z : xv[b][i >> 1].x, i & 1 ? xv[b][i >> 1].w : xv[b][i >> 1].y);
          }
        } else {
          const unsigned c0[4] = {v0.x, v0.y, v0.z, v0.w}, c1[4] = {v1.x, v1.y, v1.z, v1.w};
          const unsigned g0[2] = {now0[j].x, now0[j].y}, g1[2] = {now1[j].x, now1[j].y};
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // group i of the step: columns 8 t .. 8 t + 7 of it
            const unsigned a0[4] = {e2m1_pair<0>(c0[i]), e2m1_pair<0>(c1[i]), e2m1_pair<1>(c0[i]), e2m1_pair<1>(c1[i])};
            const unsigned a1[4] = {e2m1_pair<2>(c0[i]), e2m1_pair<2>(c1[i]), e2m1_pair<3>(c0[i]), e2m1_pair<3>(c1[i])};
            const float h0 = f16_to_f32(static_cast<unsigned short>(g0[i >> 1] >> (16 * (i & 1))));
            const float h1 = f16_to_f32(static_cast<unsigned short>(g1[i >> 1] >> (16 * (i & 1))));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const uint4 xv = lds128(xat + (i * NB + b) * 512);
              float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_bf16(d, a0, xv.x, xv.y);
              mma_bf16(d, a1, xv.z, xv.w);
              acc[b][0] = fma_rn(d[0], h0, acc[b][0]), acc[b][1] = fma_rn(d[1], h0, acc[b][1]);
              acc[b][2] = fma_rn(d[2], h1, acc[b][2]), acc[b][3] = fma_rn(d[3], h1, acc[b][3]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[b][e] += acc[b][e];
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // what is left copied nothing
  __syncwarp();  // the ring is free for the next piece
}

template <int KIND, int NB>
__global__ void __launch_bounds__(kAsThreads, 2) adapter_stream_kernel(const StreamParams p) {
  extern __shared__ __align__(128) unsigned char xs[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.y, token0 = tile * kAsTokens;
  const unsigned ring = smem_addr(xs) + kAsWindow + warp * as_depth(KIND) * as_slot(KIND);
  const int a_total = p.a_blocks * p.a_units, total = a_total + p.w_blocks * p.w_units;
  int pos = p.w_parts ? 0 : min(static_cast<long long>(blockIdx.x) * p.share, static_cast<long long>(total));
  const int end = p.w_parts ? 1 : min(pos + p.share, total);
  bool first = true;
  while (pos < end) {
    bool is_a;
    int block, u0, u1, piece;
    if (p.w_parts) {  // one piece
      const int a_ctas = p.a_blocks * p.a_parts, cta = blockIdx.x;
      is_a = cta < a_ctas;
      const int parts = is_a ? p.a_parts : p.w_parts, units = is_a ? p.a_units : p.w_units, at = is_a ? cta : cta - a_ctas;
      block = at / parts, piece = at - block * parts;
      u0 = static_cast<int>(static_cast<long long>(piece) * units / parts);
      u1 = static_cast<int>(static_cast<long long>(piece + 1) * units / parts);
      pos = end;
    } else {
      is_a = pos < a_total;
      const int units = is_a ? p.a_units : p.w_units, from = is_a ? 0 : a_total;
      block = (pos - from) / units, u0 = pos - from - block * units, u1 = min(units, u0 + end - pos);
      piece = blockIdx.x - (from + block * units) / p.share;
      pos += u1 - u0;
    }
    float sum[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[b][e] = 0.0f;
    if (is_a) {
      if (first) {  // ids belong to the call, the weights below depend on them
        grid_dependency_wait();
        grid_launch_dependents();
        first = false;
      }
      const int group = block * kAsWarps + warp, token = token0 + group / p.groups, rg = group % p.groups;
      const bool there = group < kAsTokens * p.groups && token < p.m;
      const int id = there ? __ldcg(p.ids + token) : -1;
      const bool has = id >= 0 && id < p.adapters;
      if (there && !has && id != -1 && lane == 0) record_status(p.status, kStatusBadAdapter);
      const unsigned char* base = has ? reinterpret_cast<const unsigned char*>(
                                            p.a + (static_cast<long long>(id) * p.rank + 16 * rg) * p.k)
                                      : nullptr;
      stream_piece<AD_BF16, NB, as_unit(KIND), as_depth(KIND)>(p, base, 2ll * p.k, nullptr, min(16, p.rank - 16 * rg), u0, u1,
                                                               token0, xs, ring, sum, false);
      if (has) {
        const int column = token - token0;
        float* to = p.a_part + ((static_cast<long long>(tile) * p.a_blocks + block) * p.a_pieces + piece) * kAsRows + 16 * warp;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (8 * b + 2 * t + (e & 1) == column) to[g + (e & 2 ? 8 : 0)] = sum[b][e];
      }
    } else {
      const int row0 = block * kAsRows + 16 * warp, rows = p.n - row0;
      const unsigned short* scales =
          KIND == AD_FP4 ? static_cast<const unsigned short*>(p.side) + static_cast<long long>(row0) * (p.k / 32) : nullptr;
      stream_piece<KIND, NB, as_unit(KIND), as_depth(KIND)>(p, rows > 0 ? p.w + row0 * p.row_bytes : nullptr, p.row_bytes,
                                                            scales, rows, u0, u1, token0, xs, ring, sum, first);
      first = false;
      const int tokens = min(kAsTokens, p.m - token0);
      float* to = p.w_part + (((static_cast<long long>(tile) * p.w_blocks + block) * p.w_pieces + piece) * kAsTokens) * kAsRows +
                  16 * warp;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int token = 8 * b + 2 * t + (e & 1);
          if (token < tokens) to[token * kAsRows + g + (e & 2 ? 8 : 0)] = sum[b][e];
        }
    }
  }
}

// 128 rows of one token, a thread per row. The token's adapter and its rows of B are read before the streaming kernel has
// ended: all its CTAs have then passed their wait for what came before the call.
template <int KIND>
__global__ void __launch_bounds__(kAsRows) adapter_join_kernel(const StreamParams p) {
  __shared__ __align__(16) float ts[kMaxRank];
  const int tid = threadIdx.x, block = blockIdx.x, row = block * kAsRows + tid, token = blockIdx.y;
  const int tile = token / kAsTokens, slot = token % kAsTokens;
  constexpr int kHeld = 8;  // 16-byte runs of B that are asked for ahead
  const int id = __ldcg(p.ids + token);
  const bool has = id >= 0 && id < p.adapters;
  const uint4* b = reinterpret_cast<const uint4*>(p.b + (static_cast<long long>(has ? id : 0) * p.n + min(row, p.n - 1)) * p.rank);
  const int runs = has ? p.rank / 8 : 0;
  uint4 held[kHeld];
#pragma unroll
  for (int r = 0; r < kHeld; ++r) held[r] = r < runs ? __ldcg(b + r) : make_uint4(0u, 0u, 0u, 0u);
  const float c = has ? __ldcg(p.c + id) : 0.0f;
  const float scale = KIND == AD_I8 ? __ldcg(static_cast<const float*>(p.side) + min(row, p.n - 1)) * kAsUp : kAsUp;
  grid_dependency_wait();
  grid_launch_dependents();
  // The shares of the block, in order.
  const int begin = p.a_blocks * p.a_units + block * p.w_units;
  const int pieces = p.w_parts ? p.w_parts : (begin + p.w_units - 1) / p.share - begin / p.share + 1;
  const float* from = p.w_part + ((static_cast<long long>(tile) * p.w_blocks + block) * p.w_pieces * kAsTokens + slot) * kAsRows + tid;
  float y = 0.0f;
  for (int q0 = 0; q0 < pieces; q0 += 8) {
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q)
      v[q] = q0 + q < pieces ? __ldcg(from + static_cast<long long>(q0 + q) * kAsTokens * kAsRows) : 0.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) y += v[q];
  }
  for (int r = tid; r < 8 * runs; r += kAsRows) {
    const int group = slot * p.groups + r / 16, ablock = group / kAsWarps;
    const int abegin = ablock * p.a_units;
    const int apieces = p.w_parts ? p.a_parts : (abegin + p.a_units - 1) / p.share - abegin / p.share + 1;
    const float* src = p.a_part + (static_cast<long long>(tile) * p.a_blocks + ablock) * p.a_pieces * kAsRows +
                       16 * (group % kAsWarps) + r % 16;
    float t = 0.0f;
    for (int q0 = 0; q0 < apieces; q0 += 8) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = q0 + q < apieces ? __ldcg(src + static_cast<long long>(q0 + q) * kAsRows) : 0.0f;
#pragma unroll
      for (int q = 0; q < 8; ++q) t += v[q];
    }
    ts[r] = mul_rn(t, c);
  }
  __syncthreads();
  if (row >= p.n) return;
  if (KIND != AD_BF16) y = mul_rn(y, scale);
  if (has) {
    float s0 = 0.0f, s1 = 0.0f;
    auto dot = [&](uint4 w, int r) {
      const float4 lo = reinterpret_cast<const float4*>(ts)[2 * r], hi = reinterpret_cast<const float4*>(ts)[2 * r + 1];
      s0 = fma_rn(lo.x, bf16lo(w.x), s0), s1 = fma_rn(lo.y, bf16hi(w.x), s1);
      s0 = fma_rn(lo.z, bf16lo(w.y), s0), s1 = fma_rn(lo.w, bf16hi(w.y), s1);
      s0 = fma_rn(hi.x, bf16lo(w.z), s0), s1 = fma_rn(hi.y, bf16hi(w.z), s1);
      s0 = fma_rn(hi.z, bf16lo(w.w), s0), s1 = fma_rn(hi.w, bf16hi(w.w), s1);
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
      if (r < runs) dot(held[r], r);
    for (int r = kHeld; r < runs; ++r) dot(__ldcg(b + r), r);
    y = add_rn(y, add_rn(s0, s1));
  }
  const long long at = static_cast<long long>(token) * p.ldo + row;
  if (p.out_f32)
    static_cast<float*>(p.out)[at] = y;
  else
    static_cast<unsigned short*>(p.out)[at] = f32_to_bf16_rn(y);
}

struct StreamPlan {
  int ctas, tiles;
  size_t a_part, total;
};

bool stream_kind(int wfmt, int* kind) {
  if (wfmt == KLAB_W_BF16) return *kind = AD_BF16, true;
  if (wfmt == KLAB_W_I8_ROW) return *kind = AD_I8, true;
  if (wfmt == KLAB_W_FP4_G32H) return *kind = AD_FP4, true;
  return false;
}

// Fills the shares of p (m, n, k, rank set) for `places` CTAs, which the tiles of 16 tokens share. Blocks are cut while that
// fills the machine; from kAsWaves CTAs to a place on each is a share of its own, and its tile's sums are kept once.
StreamPlan plan_stream(int kind, StreamParams& p, int places) {
  StreamPlan s{};
  p.row_bytes = kind == AD_BF16 ? 2ll * p.k : kind == AD_I8 ? p.k : p.k / 2;
  p.groups = (p.rank + 15) / 16;
  s.tiles = (p.m + kAsTokens - 1) / kAsTokens;
  const int tokens = p.m < kAsTokens ? p.m : kAsTokens;
  p.a_blocks = (tokens * p.groups + kAsWarps - 1) / kAsWarps;
  p.w_blocks = (p.n + kAsRows - 1) / kAsRows;
  p.a_units = static_cast<int>((2ll * p.k + as_unit(kind) - 1) / as_unit(kind));
  p.w_units = static_cast<int>((p.row_bytes + as_unit(kind) - 1) / as_unit(kind));
  const long long blocks = static_cast<long long>(p.a_blocks) + p.w_blocks;
  if (blocks * s.tiles >= static_cast<long long>(kAsWaves) * places) {
    p.a_parts = p.w_parts = p.a_pieces = p.w_pieces = 1;
    s.ctas = static_cast<int>(blocks);
  } else {
    const int here = places > s.tiles ? places / s.tiles : 1;
    const long long total = static_cast<long long>(p.a_blocks) * p.a_units + static_cast<long long>(p.w_blocks) * p.w_units;
    const long long share = (total + here - 1) / here;
    p.share = static_cast<int>(share < kAsMinShare ? kAsMinShare : share);
    s.ctas = static_cast<int>((total + p.share - 1) / p.share);
    p.a_pieces = (p.a_units - 1) / p.share + 2;
    p.w_pieces = (p.w_units - 1) / p.share + 2;
    p.a_parts = p.w_parts = 0;
    for (int own = p.share; own <= p.share + kAsSlack; ++own) {
      const int a_parts = (p.a_units + own - 1) / own, w_parts = (p.w_units + own - 1) / own;
      const long long ctas = static_cast<long long>(p.a_blocks) * a_parts + static_cast<long long>(p.w_blocks) * w_parts;
      if (ctas > here) continue;
      p.a_parts = p.a_pieces = a_parts, p.w_parts = p.w_pieces = w_parts;
      s.ctas = static_cast<int>(ctas);
      break;
    }
  }
  s.a_part = static_cast<size_t>(s.tiles) * p.w_blocks * p.w_pieces * kAsTokens * kAsRows * 4;
  s.total = s.a_part + static_cast<size_t>(s.tiles) * p.a_blocks * p.a_pieces * kAsRows * 4;
  return s;
}

// Rows of x that one pair of launches takes, a whole number of tiles: all, or as many as leave their FP32 sums in kAsScratch
// bytes (one tile at least).
int stream_rows(int kind, int m, int n, int k, int rank, int places) {
  StreamParams p{};
  p.m = m, p.n = n, p.k = k, p.rank = rank;
  const StreamPlan s = plan_stream(kind, p, places);
  if (s.total <= kAsScratch) return m;
  const size_t tile = (static_cast<size_t>(p.w_blocks) * kAsTokens + p.a_blocks) * kAsRows * 4;
  const size_t tiles = tile < kAsScratch ? kAsScratch / tile : 1;
  return static_cast<long long>(tiles) * kAsTokens < m ? static_cast<int>(tiles) * kAsTokens : m;
}

// The same for the form of three launches, whose scratch holds t and the projection in FP32. Every part has more than 16 rows
// (or is the whole call), so that the projection asks for no more workspace than for all rows.
int plain_rows(int m, int n, int rank) {
  const size_t row = (static_cast<size_t>(n) + rank) * 4, rows = kAsScratch / row / kAsTokens * kAsTokens;
  const int most = rows > 2 * kAsTokens ? static_cast<int>(rows < 65536 ? rows : 65536) : 2 * kAsTokens;
  return m - most > kAsTokens ? most : m;
}

// Bytes of t, and of t and the projection, for up to `rows` rows of the call and the few behind the last part.
size_t plain_t(int rows, int rank) { return (static_cast<size_t>(rows) * rank * 4 + 127) / 128 * 128; }
size_t plain_scratch(int m, int n, int rank) {
  const int rows = plain_rows(m, n, rank), held = rows < m ? rows + kAsTokens : m;
  return plain_t(held, rank) + static_cast<size_t>(held) * n * 4;
}

template <int KIND, int NB>
int run_stream(const StreamParams& p, const StreamPlan& plan, cudaStream_t stream) {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (!(ready.load() >> dev & 1)) {
    err = cudaFuncSetAttribute(adapter_stream_kernel<KIND, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, as_smem(KIND));
    if (err != cudaSuccess) return err;
    ready.fetch_or(1ull << dev);
  }
  const int rc = launch_dependent(adapter_stream_kernel<KIND, NB>, dim3(plan.ctas, plan.tiles), kAsThreads, as_smem(KIND),
                                  stream, p);
  if (rc) return rc;
  return launch_dependent(adapter_join_kernel<KIND>, dim3(p.w_blocks, p.m), kAsRows, 0, stream, p);
}

}  // namespace
}  // namespace klab

extern "C" {

KLAB_API long long klab_adapter_scratch(int wfmt, int m, int n, int k, int rank) {
  using namespace klab;
  if (m <= 0 || n <= 0 || k <= 0 || rank <= 0) return KLAB_E_INVALID;
  size_t need = plain_scratch(m, n, rank);  // streamed formats with rows off 16-byte boundaries too
  int kind = 0, sms = 0;
  if (stream_kind(wfmt, &kind)) {
    const int rc = device_sms(&sms);
    if (rc) return rc < 0 ? rc : -rc;
    const int rows = stream_rows(kind, m, n, k, rank, 2 * sms);
    for (const int part : {rows, m % rows}) {
      if (!part) continue;
      StreamParams p{};
      p.m = part, p.n = n, p.k = k, p.rank = rank;
      const size_t total = plan_stream(kind, p, 2 * sms).total;
      if (total > need) need = total;
    }
  }
  return static_cast<long long>(need);
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
  if (scratch_bytes < klab_adapter_scratch(wfmt, m, n, k, rank)) return KLAB_E_INVALID;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int out_bytes = out_dtype == KLAB_DT_F32 ? 4 : 2;
  int kind = 0;
  if (stream_kind(wfmt, &kind)) {
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    const int rows = stream_rows(kind, m, n, k, rank, 2 * sms);
    StreamParams q{};
    q.m = rows, q.n = n, q.k = k, q.rank = rank;
    plan_stream(kind, q, 2 * sms);
    if ((reinterpret_cast<uintptr_t>(w) & 15) == 0 && q.row_bytes % 16 == 0 &&
        static_cast<long long>(q.a_blocks) * q.a_units + static_cast<long long>(q.w_blocks) * q.w_units < INT_MAX) {
      if (kind != AD_BF16 && !aux) return KLAB_E_INVALID;
      if (kind == AD_FP4 && k % 32) return KLAB_E_SHAPE;
      q.w = static_cast<const unsigned char*>(w);
      q.side = aux;
      q.a = static_cast<const unsigned short*>(a);
      q.b = static_cast<const unsigned short*>(b);
      q.c = c;
      q.w_part = static_cast<float*>(scratch);
      q.status = device_status_address();
      q.adapters = adapters;
      q.ldo = n;
      q.out_f32 = out_dtype == KLAB_DT_F32;
      for (int m0 = 0; m0 < m; m0 += rows) {
        q.m = m - m0 < rows ? m - m0 : rows;
        const StreamPlan plan = plan_stream(kind, q, 2 * sms);
        q.a_part = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + plan.a_part);
        q.x = static_cast<const unsigned short*>(x) + static_cast<long long>(m0) * k;
        q.ids = ids + m0;
        q.out = static_cast<unsigned char*>(out) + static_cast<long long>(m0) * n * out_bytes;
        const bool one = q.m <= 8;
        int rc;
        if (kind == AD_BF16)
          rc = one ? run_stream<AD_BF16, 1>(q, plan, s) : run_stream<AD_BF16, 2>(q, plan, s);
        else if (kind == AD_I8)
          rc = one ? run_stream<AD_I8, 1>(q, plan, s) : run_stream<AD_I8, 2>(q, plan, s);
        else
          rc = one ? run_stream<AD_FP4, 1>(q, plan, s) : run_stream<AD_FP4, 2>(q, plan, s);
        if (rc) return rc;
      }
      return 0;
    }
  }
  AdapterParams p{};
  p.a = static_cast<const unsigned short*>(a);
  p.b = static_cast<const unsigned short*>(b);
  p.c = c;
  p.status = device_status_address();
  p.n = n;
  p.k = k;
  p.rank = rank;
  p.adapters = adapters;
  p.ldo = n;
  p.out_f32 = out_dtype == KLAB_DT_F32;
  p.t = static_cast<float*>(scratch);
  const int part = plain_rows(m, n, rank);
  for (int m0 = 0; m0 < m; m0 += p.m) {
    p.m = m - m0 - part > kAsTokens ? part : m - m0;
    float* y0 = p.t + plain_t(p.m, rank) / 4;
    p.y0 = y0;
    p.x = static_cast<const unsigned short*>(x) + static_cast<long long>(m0) * k;
    p.ids = ids + m0;
    p.out = static_cast<unsigned char*>(out) + static_cast<long long>(m0) * n * out_bytes;
    int rc = launch_dependent(shrink_kernel, dim3(rank / kRanks, p.m), kAdThreads, 0, s, p);
    if (rc) return rc;
    rc = klab_gemv(wfmt, KLAB_DT_BF16, p.x, k, w, aux, nullptr, y0, n, KLAB_DT_F32, p.m, n, k, workspace, workspace_bytes, stream);
    if (rc) return rc;
    rc = launch_dependent(expand_kernel, dim3((n + kAdThreads - 1) / kAdThreads, p.m), kAdThreads, 0, s, p);
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
