// Layout of the 4-bit K/V pages (kv_tables.cu, kv_store.cu, kv_attn.cu).
//
// pages: uint8 [num_pages][kv_heads][page_size / 16][block], a block = 16 tokens of one kv head:
//   K codes   8 * D bytes   32-bit word (quad, r, t, i): dims 32 G + 8 t .. + 7 of token r, low nibble first
//   V codes   8 * D bytes   32-bit word (quad, j, g, t, i): dims 32 G + 4 g .. + 3, low nibble first, of token
//                           r = 8 j + 2 t in the low half and of token r + 1 in the high half
//   K scales  D bytes       fp16 (r, G)
//   V scales  D bytes       fp16 (j, t, G, r mod 2)
// with D the head dimension, NG = D / 32 groups of 32 dims, Q = min(NG, 4), G = Q * quad + i.
// A value is (code - 8) * scale; scale = RN16(min(max|x| / 7, 65504)) over the group's 32 dims.
//
// The order is that of the attention kernel's matrix fragments: lane (g, t) of a warp reads its K words of
// token g (and g + 8) as one run, and its V words of four tokens as two runs, and a mask with 0x000f000f or
// 0x00f000f0 turns a word into a pair of FP16 subnormals u * 2^-24 (or 16 u * 2^-24): no conversion, no shift
// for half of the pairs.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "klab_b200.h"

namespace klab {

constexpr int kKvGroup = 32;        // dims that share a scale
constexpr int kKvBlock = 16;        // tokens of a block
constexpr int kKvMaxRequests = KLAB_KV_MAX_REQUESTS;
constexpr int kKvMaxNew = KLAB_KV_MAX_NEW;

__host__ __device__ constexpr int kv_block_bytes(int dim) { return 18 * dim; }

// Byte offset of the block that holds token `slot` of kv head `head`, or -1 when the slot lies outside the pages; a page
// has 2^page_shift tokens. Offsets of a long cache pass 32 bits.
__host__ __device__ inline long long kv_block_offset(int slot, int head, int num_pages, int kv_heads, int page_shift,
                                                     int dim) {
  if (slot < 0 || (slot >> page_shift) >= num_pages) return -1;
  const long long page = slot >> page_shift;
  const int block = (slot & ((1 << page_shift) - 1)) / kKvBlock;
  return (((page * kv_heads + head) << (page_shift - 4)) + block) * kv_block_bytes(dim);
}

// Offsets inside a block, in 16-bit units, of piece c (dims 4 c .. 4 c + 3) and of group G's scale of token r.
__host__ __device__ inline int kv_k_piece(int r, int c, int dim) {
  const int ng = dim / kKvGroup, q = ng < 4 ? ng : 4, group = c >> 3, g = c & 7;
  return group / q * (128 * q) + r * (8 * q) + (g >> 1) * (2 * q) + group % q * 2 + (g & 1);
}
__host__ __device__ inline int kv_v_piece(int r, int c, int dim) {
  const int ng = dim / kKvGroup, q = ng < 4 ? ng : 4, group = c >> 3, g = c & 7;
  return 4 * dim + group / q * (128 * q) + (r >> 3) * (64 * q) + g * (8 * q) + ((r & 7) >> 1) * (2 * q) +
         group % q * 2 + (r & 1);
}
__host__ __device__ inline int kv_k_scale(int r, int group, int dim) { return 8 * dim + r * (dim / kKvGroup) + group; }
__host__ __device__ inline int kv_v_scale(int r, int group, int dim) {
  return 8 * dim + dim / 2 + ((r >> 3) * 4 + ((r & 7) >> 1)) * (dim / 16) + group * 2 + (r & 1);
}

inline bool kv_page_size_ok(int page_size) {
  return page_size >= kKvBlock && page_size <= 1024 && (page_size & (page_size - 1)) == 0;
}
inline int kv_page_shift(int page_size) {
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  return shift;
}
inline bool kv_dim_ok(int dim) { return dim == 64 || dim == 128 || dim == 256; }

}  // namespace klab
