// The key/value cache's layout, exponents and bounds (include/supra_kv.h), for the kernels and for host code.
#pragma once

#include <stdint.h>

#include "supra_kv.h"

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define SA_HD __host__ __device__ __forceinline__
#else
#define SA_HD inline
#endif

namespace sa {

constexpr int kKvBlock = SA_KV_BLOCK;
constexpr int kKvMaxBlocks = 1 << 25;  // columns of a block table: token positions stay below 2^30

// Byte offset of a page's head: K and V tiles of 32 x D codes.
SA_HD int64_t kv_tile(int64_t page, int Hkv, int h, int D) { return (page * Hkv + h) * (int64_t)(kKvBlock * D); }
// Place of token t's code inside the 32 codes of one V element d, and of (t, d) inside a K tile.
SA_HD int kv_v_slot(int t) { return 16 * ((t >> 2) & 1) + 4 * (t >> 3) + (t & 3); }
SA_HD int kv_k_place(int t, int d) { return (d >> 5) * 1024 + t * 32 + (d & 31); }

SA_HD bool kv_page_ok(int32_t page, int pages) { return (uint32_t)page < (uint32_t)pages; }

// Exponent byte of a page whose largest finite magnitude has the float32 bits `amax` (sign 0): the smallest e with
// amax <= 448 * 2^(e - 127), 448 = 1.75 * 2^8. 0 at least, which zeros and magnitudes below 2^-119 take.
SA_HD int kv_exponent(uint32_t amax) {
  const int x = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return x > 0 ? x : 0;
}

// float32 bits of 2^n: 0 below -126, n at most 127.
SA_HD uint32_t kv_pow2_bits(int n) { return n < -126 ? 0u : (uint32_t)(n + 127) << 23; }

// A sequence's bounds, whatever the device arrays say (the argument checks bound T, max_rows and max_blocks).
struct KvSeq {
  int len;      // tokens in the cache
  int rows;     // rows of the call's row tensors
  int row0;     // the first of them
  int first;    // position of the first row's token; may be negative
};

SA_HD KvSeq kv_seq(const sa_kv_seqs& s, int b) {
  KvSeq q;
  const int cap = s.max_blocks * kKvBlock;
  int n = s.seq_len[b];
  n = n < 0 ? 0 : n > cap ? cap : n;
  int64_t r0 = (int64_t)b * s.max_rows, r = s.max_rows;
  if (s.row_start) {
    r0 = s.row_start[b];
    r = (int64_t)s.row_start[b + 1] - r0;
  }
  if (r < 0 || r0 < 0 || r0 >= s.T) r = 0;
  const int64_t first = (int64_t)n - r;
  if (r > s.max_rows) r = s.max_rows;
  if (r > s.T - r0) r = r > 0 ? s.T - r0 : 0;
  q.len = n;
  q.rows = (int)r;
  q.row0 = (int)r0;
  q.first = (int)(first < -(1 << 30) ? -(1 << 30) : first);
  return q;
}

}  // namespace sa
