// The 4-bit cache of tpx_packed.h as the kernels see it: places of tokens, and where a page keeps what.
#pragma once
#include "../../include/tpx_packed.h"
#include "tpx_common.cuh"

namespace tpx {

constexpr int kI4Page = 32;   // tokens of a page
constexpr int kI4Group = 64;  // values that share a scale and a minimum

// byte offsets within one head of a page
template <int H>
struct I4 {
  static constexpr int G = H / kI4Group;
  static constexpr int CODES = kI4Page * H / 2, PARAMS = kI4Page * G * 4;
  static constexpr int KC = 0, KP = CODES, VC = CODES + PARAMS, VP = 2 * CODES + PARAMS;
  static constexpr int BYTES = 2 * (CODES + PARAMS);  // 36 H
};

struct I4Cache {
  uint8_t* pool;
  const int32_t *table, *lengths;
  int pages, cols, B, Nkv;
};

// The word of 8 values from dimension d (a multiple of 8) of the page's token t: index among the K or V code words
__host__ __device__ __forceinline__ int i4_k_word(int H, int t, int d) { return t * (H / 8) + (d % 32 / 8) * (H / 32) + d / 32; }
__host__ __device__ __forceinline__ int i4_v_word(int H, int t, int d) {
  return ((((t / 8) * 8 + d % 64 / 8) * 4 + t % 4) * 2 + t % 8 / 4) * (H / 64) + d / 64;
}

// The sequence that token row `row` belongs to, -1 if none. cu may be any int32s: the result is in [-1, B).
__device__ __forceinline__ int i4_sequence(const int32_t* cu, int B, int row) {
  if (!cu) return row < B ? row : -1;
  int lo = 0, hi = B;  // cu[lo] <= row < cu[hi] where it is in any
  if (row < cu[0] || row >= cu[B]) return -1;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (cu[m] <= row) lo = m;
    else hi = m;
  }
  return lo;
}

// Head `n` of the page of place t of sequence b, or null
__device__ __forceinline__ uint8_t* i4_head(const I4Cache& c, int b, int64_t t, int n, int bytes) {
  if (t < 0 || t >= (int64_t)c.cols * kI4Page) return nullptr;
  const int page = c.table[(int64_t)b * c.cols + (int)(t / kI4Page)];
  if (page < 0 || page >= c.pages) return nullptr;
  return c.pool + ((int64_t)page * c.Nkv + n) * bytes;
}

int i4_cache_of(const TpxInt4Cache* a, I4Cache* c);  // checks the sizes and pointers

}  // namespace tpx
