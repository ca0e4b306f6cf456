// A key-value cache held in 4 bits, in pages.
//
// A value is one of +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} (a code: sign, two bits of exponent, one of
// mantissa) times the power of two 2^(byte - 127) that 32 neighbouring channels of a token share;
// byte 255: one of the 32 was not finite, and all read as NaN. A page holds `page` tokens (a
// multiple of 32) of every key-value head in four arrays, first the pages, then the heads:
//
//   k         [page][dim / 2]               channels 2 i and 2 i + 1 in byte i's low and high half
//   k_scales  [page / 32][4][dim / 32][8]   token 32 a + 4 c + b at [a][b][:][c]
//   v         [page / tb][16][tb][dim / 32] token tb a + b, channels dim / 16 n ... at [a][n][b], tb = 512 / dim
//   v_scales  [page / 32][dim / 32][32]     token 32 a + b at [a][:][b]
//
// A wave that attends to 32 tokens then takes every operand in whole pieces: a token's row of k is
// the contracted index of the scores, 16 bytes a lane; 8 tokens of v's channel slice n are 32
// contiguous bytes (dim 128) or 16 (dim 64), the contracted index of the second product.
#pragma once

#include "bq_common.h"

namespace bq {

struct Kv4 {
  uint8_t *k, *ks, *v, *vs;
  int pages, heads, page;  // page: tokens a page
  const int* table;        // [B][width]: the pages of each sequence, in order
  int width;
  FastDiv by_page, by_blocks;  // division by page, by page / 32
};

// Checks a cache's description and fills the kernels' form of it.
int kv4_of(const char* what, const bq_kv4_cache* c, const int* table, int64_t B, int64_t width, Kv4* out);

// Where a token lies: of page `at` (checked by the caller), head h, place `off`.
template <int DIM>
struct Kv4At {
  static constexpr int TB = 512 / DIM, CB = DIM / 32;  // tokens a v block, scale blocks a token
  static __device__ __forceinline__ size_t row(const Kv4& c, int at, int h, int off) {
    return ((size_t)at * c.heads + h) * c.page + off;
  }
  // of the first token of v's block and of the 32 tokens that share a block of scales
  static __device__ __forceinline__ size_t k(size_t row) { return row * (DIM / 2); }
  static __device__ __forceinline__ size_t v(size_t row, int off, int n) {
    return (row - off % TB) * (DIM / 2) + (n * TB + off % TB) * CB;
  }
  static __device__ __forceinline__ size_t ks(size_t row, int off, int block) {
    return (row - (off & 31)) * CB + (((off & 3) * CB + block) << 3) + ((off & 31) >> 2);
  }
  static __device__ __forceinline__ size_t vs(size_t row, int off, int block) {
    return (row - (off & 31)) * CB + block * 32 + (off & 31);
  }
};

// A token's page, or -1 (outside the table, or no page of the cache).
__device__ __forceinline__ int kv4_page(const Kv4& c, int b, int page_index) {
  if ((unsigned)page_index >= (unsigned)c.width) return -1;
  const int at = c.table[(size_t)b * c.width + page_index];
  return (unsigned)at < (unsigned)c.pages ? at : -1;
}

// Elements of the callers' types.
enum { KV4_F32 = 0, KV4_BF16 = 1, KV4_F16 = 2 };

}  // namespace bq
