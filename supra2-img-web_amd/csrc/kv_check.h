// Argument checks shared by the cache's entry points.
#pragma once

#include <stdint.h>

#include "kv_layout.h"
#include "status.h"

namespace sa {

constexpr int64_t kKvMaxStride = (int64_t)1 << 40;
constexpr int64_t kKvMaxThreads = ((int64_t)1 << 32) - 1;  // of one launch

inline int kv_type_bytes(int32_t dtype) { return dtype == SA_DT_F32 ? 4 : dtype == SA_DT_F16 || dtype == SA_DT_BF16 ? 2 : 0; }

inline int kv_check_dtype(int32_t dtype) {
  if (kv_type_bytes(dtype)) return SA_OK;
  if (dtype >= SA_DT_F32 && dtype <= SA_DT_F8_E5M2)
    return fail(SA_ERR_UNSUPPORTED, "dtype %d: the rows are SA_DT_F32, SA_DT_F16 or SA_DT_BF16", dtype);
  return fail(SA_ERR_INVALID, "unknown dtype %d", dtype);
}

// n rows of `width` elements every `ld` from base + off, in bytes.
struct KvRows {
  const char* lo;
  int64_t ld, width, n;
  const char* hi() const { return n > 0 ? lo + (n - 1) * ld + width : lo; }
};

// Offsets and strides in elements, validated; `name` for the message. ld 0 means width.
inline int kv_rows(const void* base, int64_t off, int64_t ld, int64_t width, int64_t n, int size, const char* name, KvRows* out) {
  if (!base) return fail(SA_ERR_INVALID, "%s must be a non-NULL device pointer", name);
  if ((uintptr_t)base % size != 0) return fail(SA_ERR_INVALID, "%s is not aligned to its type", name);
  if (off < 0 || off >= kKvMaxStride || ld < 0 || ld >= kKvMaxStride)
    return fail(SA_ERR_INVALID, "offset and row stride of %s must be in [0, 2^40)", name);
  if (ld == 0) ld = width;
  if (ld < width) return fail(SA_ERR_INVALID, "row stride %lld of %s is below its row of %lld", (long long)ld, name, (long long)width);
  int64_t span = 0;
  if (__builtin_mul_overflow(n > 0 ? n - 1 : 0, ld * size, &span) || span > INT64_MAX / 4)
    return fail(SA_ERR_INVALID, "the extent of %s overflows 64-bit addresses", name);
  *out = {(const char*)base + off * size, ld * size, width * size, n};
  return SA_OK;
}

inline bool kv_overlap(const void* a, int64_t abytes, const void* b, int64_t bbytes) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  return abytes > 0 && bbytes > 0 && a0 < b0 + (uintptr_t)bbytes && b0 < a0 + (uintptr_t)abytes;
}

// Whether two sets of rows share a byte. Column blocks of the same rows (one stride) do not; other strides whose
// ranges meet count as overlapping.
inline bool kv_overlap(const KvRows& a, const KvRows& b) {
  if (!kv_overlap(a.lo, a.hi() - a.lo, b.lo, b.hi() - b.lo)) return false;
  if (a.ld != b.ld) return true;
  int64_t d = (int64_t)((uintptr_t)b.lo - (uintptr_t)a.lo) % a.ld;
  if (d < 0) d += a.ld;
  return d < a.width || d + b.width > a.ld;
}
inline bool kv_overlap(const KvRows& a, const void* p, int64_t bytes) { return kv_overlap(a.lo, a.hi() - a.lo, p, bytes); }

inline int kv_check_cache(const sa_kv_cache& c) {
  if (c.pages <= 0 || c.Hkv <= 0) return fail(SA_ERR_INVALID, "pages and Hkv must be positive (got %d, %d)", c.pages, c.Hkv);
  if (c.reserved != 0) return fail(SA_ERR_INVALID, "the cache's reserved field must be 0");
  if (c.D != 64 && c.D != 128 && c.D != 256) {
    if (c.D <= 0) return fail(SA_ERR_INVALID, "head dim %d", c.D);
    return fail(SA_ERR_UNSUPPORTED, "head dim %d: the cache holds 64, 128 or 256", c.D);
  }
  if (c.Hkv > 4096) return fail(SA_ERR_UNSUPPORTED, "%d key heads (at most 4096)", c.Hkv);
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return fail(SA_ERR_INVALID, "the cache's pointers must be non-NULL device pointers");
  if (((uintptr_t)c.k | (uintptr_t)c.v) & 15) return fail(SA_ERR_INVALID, "the cache's k and v must be 16-byte aligned");
  const int64_t bytes = (int64_t)c.pages * c.Hkv * kKvBlock * c.D, scales = (int64_t)c.pages * c.Hkv;
  if (kv_overlap(c.k, bytes, c.v, bytes) || kv_overlap(c.k_scale, scales, c.v_scale, scales) || kv_overlap(c.k, bytes, c.k_scale, scales) ||
      kv_overlap(c.k, bytes, c.v_scale, scales) || kv_overlap(c.v, bytes, c.k_scale, scales) || kv_overlap(c.v, bytes, c.v_scale, scales))
    return fail(SA_ERR_ALIAS, "the cache's arrays overlap");
  return SA_OK;
}

// B == 0 or T == 0 (nothing to do) passes with NULL arrays.
inline int kv_check_seqs(const sa_kv_seqs& s) {
  if (s.B < 0 || s.T < 0 || s.max_rows < 0 || s.max_blocks < 0) return fail(SA_ERR_INVALID, "B, T, max_rows and max_blocks must be >= 0");
  if (s.B > (1 << 20)) return fail(SA_ERR_UNSUPPORTED, "%d sequences (at most 2^20)", s.B);
  if (s.max_blocks > kKvMaxBlocks) return fail(SA_ERR_UNSUPPORTED, "max_blocks %d (at most 2^25)", s.max_blocks);
  if (s.B == 0 || s.T == 0 || s.max_rows == 0) return SA_OK;
  if (!s.seq_len || (s.max_blocks > 0 && !s.block_table)) return fail(SA_ERR_INVALID, "seq_len and block_table must be non-NULL device pointers");
  if (!s.row_start && (int64_t)s.B * s.max_rows > s.T)
    return fail(SA_ERR_INVALID, "without row_start, T = %d must hold max_rows = %d rows of each of %d sequences", s.T, s.max_rows, s.B);
  return SA_OK;
}

inline bool kv_nothing(const sa_kv_seqs& s) { return s.B == 0 || s.T == 0 || s.max_rows == 0; }

// Whether rows that are written share a byte with an array of the sequences.
inline bool kv_overlap_seqs(const KvRows& r, const sa_kv_seqs& s) {
  return kv_overlap(r, s.seq_len, 4LL * s.B) || kv_overlap(r, s.block_table, 4LL * s.B * s.max_blocks) ||
         (s.row_start && kv_overlap(r, s.row_start, 4LL * (s.B + 1)));
}
inline bool kv_overlap_cache(const KvRows& r, const sa_kv_cache& c) {
  const int64_t scales = (int64_t)c.pages * c.Hkv, bytes = scales * kKvBlock * c.D;
  return kv_overlap(r, c.k, bytes) || kv_overlap(r, c.v, bytes) || kv_overlap(r, c.k_scale, scales) || kv_overlap(r, c.v_scale, scales);
}

}  // namespace sa
