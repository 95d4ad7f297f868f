// The 8-bit key/value cache written and read back (include/supra_kv.h).
//
// A page and head of K or V is one tile of 32 tokens x D codes with one exponent byte. Both kernels give a wave one
// such tile: what it reads and writes is contiguous on the cache's side and whole rows' heads on the other, and
// the page's scale is a reduction inside the wave. Which sequence, page and head that is follows from the
// workgroup index and the device's own lengths; waves beyond a sequence's pages end at once.
//
// Quantising: with e the page's exponent byte, code = e4m3(x * 2^(127 - e)). The factor is a power of two, so the
// product is exact (or below every e4m3 value's half), and v_cvt_pk_fp8_f32 rounds it once, to nearest even. A
// page that holds earlier tokens keeps max(its exponent, the new tokens'): codes that must move to a larger scale
// are decoded, multiplied by a power of two and rounded the same way.
//
// Bound: HBM traffic (rows in, a quarter to a half of it out).

#include <hip/hip_runtime.h>

#include "common.h"
#include "kv_check.h"
#include "kv_layout.h"
#include "row_types.h"

namespace sa {

namespace {

constexpr int kWaves = 4;  // tiles per workgroup

struct KvMove {
  sa_kv_cache c;
  sa_kv_seqs s;
  char* k;  // the rows (offset included)
  char* v;
  int64_t ldk, ldv;  // bytes
  int blocks;        // tiles of one head that a sequence's rows can touch
  int64_t tiles;     // B * blocks * Hkv * 2
};

// The tile of one wave: (sequence, block of 32 positions, head, K or V). Consecutive waves take the heads of one
// block, which share the rows' lines.
struct Tile {
  KvSeq q;
  int h;
  bool is_v;
  int lo, hi;     // rows' tokens inside the block: places [lo, hi), lo < hi
  int row;        // row of place 0 (of the rows [lo, hi) it is a valid one)
  int32_t page;   // -1: none
};

__device__ __forceinline__ bool kv_tile_of(const KvMove& a, int64_t i, Tile* t) {
  if (i >= a.tiles) return false;
  t->is_v = i & 1;
  i >>= 1;
  t->h = (int)(i % a.c.Hkv);
  i /= a.c.Hkv;
  const int n = (int)(i % a.blocks), b = (int)(i / a.blocks);
  t->q = kv_seq(a.s, b);
  const KvSeq& q = t->q;
  if (q.rows == 0) return false;
  const int last = q.first + q.rows;       // one past the last row's position
  const int block = (q.first >> 5) + n;    // of 32 positions; negative ones hold no token
  t->lo = q.first - 32 * block;
  t->hi = last - 32 * block;
  t->row = q.row0 - t->lo;
  if (t->lo < 0) t->lo = 0;
  if (t->hi > 32) t->hi = 32;
  if (t->lo >= t->hi) return false;
  t->page = -1;
  if (block >= 0 && block < a.s.max_blocks) {
    const int32_t p = a.s.block_table[(int64_t)b * a.s.max_blocks + block];
    if (kv_page_ok(p, a.c.pages)) t->page = p;
  }
  return true;
}

// Bits of |x| for the scale: infinities and NaN do not count.
__device__ __forceinline__ uint32_t amax_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t y = __shfl_xor(x, m);
    x = x > y ? x : y;
  }
  return x;
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// The four codes of w at a scale 1/factor times as large: decoded, multiplied, rounded.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float factor) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return encode4(a[0] * factor, a[1] * factor, b[0] * factor, b[1] * factor);
}

__device__ __forceinline__ int new_exponent(int e, uint8_t* scale, bool keeps, int* old) {
  *old = 0;
  if (keeps) {
    *old = min((int)*scale, 254);
    e = max(e, *old);
  }
  return e;
}

template <typename T, int D, bool ALIGNED>
__global__ __launch_bounds__(64 * kWaves) void kv_write_kernel(KvMove a) {
  const int lane = threadIdx.x & 63;
  Tile t;
  if (!kv_tile_of(a, (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), &t)) return;
  if (t.page < 0) return;
  const int64_t at = kv_tile(t.page, a.c.Hkv, t.h, D);
  const bool keeps = t.lo > 0 && t.q.first > 0;  // the block holds earlier tokens: places [0, lo)
  uint8_t* scale = (t.is_v ? a.c.v_scale : a.c.k_scale) + (int64_t)t.page * a.c.Hkv + t.h;
  if (!t.is_v) {
    // 16 codes per lane and step: token and 16 channels, D/16 lanes across a token's row
    constexpr int N = D / 32, R = D / 16;
    float x[N][16];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * 64 + lane, tok = id / R, d = id % R * 16;
      if (tok >= t.lo && tok < t.hi) {
        load_row<T, 16, ALIGNED>(reinterpret_cast<const T*>(a.k + (int64_t)(t.row + tok) * a.ldk) + t.h * D + d, x[i]);
#pragma unroll
        for (int j = 0; j < 16; ++j) m = max(m, amax_bits(x[i][j]));
      }
    }
    int old;
    const int e = new_exponent(kv_exponent(wave_max(m)), scale, keeps, &old);
    const float factor = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e); e <= 254
    const bool grows = keeps && e > old;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * 64 + lane, tok = id / R, d = id % R * 16;
      uint8_t* p = a.c.k + at + kv_k_place(tok, d);
      uint32_t w[4];
      if (tok >= t.lo && tok < t.hi) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = encode4(x[i][4 * j] * factor, x[i][4 * j + 1] * factor, x[i][4 * j + 2] * factor, x[i][4 * j + 3] * factor);
        store_words<16>(p, w);
      } else if (grows && tok < t.lo) {
        load_words<16>(p, w);
        const float f = __uint_as_float(kv_pow2_bits(old - e));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = rescale4(w[j], f);
        store_words<16>(p, w);
      }
    }
    if (lane == 0) *scale = (uint8_t)e;
  } else {
    // D/64 channels per lane, all 32 tokens of each: the transposed tile needs no exchange between lanes
    constexpr int E = D / 64;
    float x[32][E];
    uint32_t m = 0;
#pragma unroll
    for (int tok = 0; tok < 32; ++tok) {
#pragma unroll
      for (int j = 0; j < E; ++j) x[tok][j] = 0.f;
      if (tok >= t.lo && tok < t.hi) {
        load_row<T, E, ALIGNED>(reinterpret_cast<const T*>(a.v + (int64_t)(t.row + tok) * a.ldv) + t.h * D + lane * E, x[tok]);
#pragma unroll
        for (int j = 0; j < E; ++j) m = max(m, amax_bits(x[tok][j]));
      }
    }
    int old;
    const int e = new_exponent(kv_exponent(wave_max(m)), scale, keeps, &old);
    const float factor = __uint_as_float((uint32_t)(254 - e) << 23);
    const bool grows = keeps && e > old, whole = t.lo == 0 && t.hi == 32;
    const float f = __uint_as_float(kv_pow2_bits(old - e));
    const uint32_t news = (t.hi == 32 ? 0xffffffffu : (1u << t.hi) - 1u) & ~((1u << t.lo) - 1u), olds = (1u << t.lo) - 1u;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      uint8_t* p = a.c.v + at + (lane * E + j) * 32;
      uint32_t w[8], had[8];
      if (!whole) load_words<32>(p, had);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int tok = 8 * (k & 3) + 4 * (k >> 2);  // the four tokens of word k
        w[k] = encode4(x[tok][j] * factor, x[tok + 1][j] * factor, x[tok + 2][j] * factor, x[tok + 3][j] * factor);
        if (!whole) {
          uint32_t moved = had[k];
          if (grows) moved = rescale4(had[k], f);
          uint32_t mn = 0, mo = 0;  // bytes of new and of earlier tokens
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            mn |= (news >> (tok + r) & 1u) ? 0xffu << (8 * r) : 0u;
            mo |= (olds >> (tok + r) & 1u) ? 0xffu << (8 * r) : 0u;
          }
          w[k] = (w[k] & mn) | (moved & mo) | (had[k] & ~(mn | mo));
        }
      }
      store_words<32>(p, w);
    }
    if (lane == 0) *scale = (uint8_t)e;
  }
}

template <typename T, int D, bool ALIGNED>
__global__ __launch_bounds__(64 * kWaves) void kv_read_kernel(KvMove a) {
  const int lane = threadIdx.x & 63;
  Tile t;
  if (!kv_tile_of(a, (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), &t)) return;
  const bool none = t.page < 0;
  const int64_t page = none ? 0 : t.page, at = kv_tile(page, a.c.Hkv, t.h, D);
  const int e = (t.is_v ? a.c.v_scale : a.c.k_scale)[page * a.c.Hkv + t.h];
  // 2^(e - 127), down to the subnormal 2^-127: exact products either way
  const float factor = none ? 0.f : e == 0 ? 0x1p-127f : __uint_as_float((uint32_t)min(e, 254) << 23);
  if (!t.is_v) {
    constexpr int N = D / 32, R = D / 16;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * 64 + lane, tok = id / R, d = id % R * 16;
      if (tok < t.lo || tok >= t.hi) continue;
      uint32_t w[4] = {0, 0, 0, 0};
      if (!none) load_words<16>(a.c.k + at + kv_k_place(tok, d), w);
      float x[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
        x[4 * j] = lo[0] * factor, x[4 * j + 1] = lo[1] * factor, x[4 * j + 2] = hi[0] * factor, x[4 * j + 3] = hi[1] * factor;
      }
      store_row<T, 16, ALIGNED>(reinterpret_cast<T*>(a.k + (int64_t)(t.row + tok) * a.ldk) + t.h * D + d, x);
    }
  } else {
    constexpr int E = D / 64;
    uint32_t w[E][8];
#pragma unroll
    for (int j = 0; j < E; ++j) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[j][k] = 0;
      if (!none) load_words<32>(a.c.v + at + (lane * E + j) * 32, w[j]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x[4][E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j][k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j][k], true);
        x[0][j] = lo[0] * factor, x[1][j] = lo[1] * factor, x[2][j] = hi[0] * factor, x[3][j] = hi[1] * factor;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = 8 * (k & 3) + 4 * (k >> 2) + r;
        if (tok >= t.lo && tok < t.hi)
          store_row<T, E, ALIGNED>(reinterpret_cast<T*>(a.v + (int64_t)(t.row + tok) * a.ldv) + t.h * D + lane * E, x[r]);
      }
    }
  }
}

template <typename T, int D>
hipError_t launch_d(const KvMove& a, bool write, bool aligned, hipStream_t stream) {
  const dim3 grid((unsigned)((a.tiles + kWaves - 1) / kWaves)), block(64 * kWaves);
  if (write) {
    if (aligned) hipLaunchKernelGGL((kv_write_kernel<T, D, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv_write_kernel<T, D, false>), grid, block, 0, stream, a);
  } else {
    if (aligned) hipLaunchKernelGGL((kv_read_kernel<T, D, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv_read_kernel<T, D, false>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const KvMove& a, bool write, bool aligned, hipStream_t stream) {
  return a.c.D == 64 ? launch_d<T, 64>(a, write, aligned, stream)
         : a.c.D == 128 ? launch_d<T, 128>(a, write, aligned, stream) : launch_d<T, 256>(a, write, aligned, stream);
}

// Both calls: checks, then one launch.
int kv_move(const sa_kv_rows_args* a, bool write, void* stream) {
  if (a == nullptr) return fail(SA_ERR_INVALID, "args is NULL");
  if (a->struct_size != sizeof(sa_kv_rows_args))
    return fail(SA_ERR_INVALID, "struct_size %u does not match sizeof(sa_kv_rows_args) = %zu", a->struct_size, sizeof(sa_kv_rows_args));
  int rc = kv_check_dtype(a->dtype);
  if (rc == SA_OK) rc = kv_check_cache(a->cache);
  if (rc == SA_OK) rc = kv_check_seqs(a->seqs);
  if (rc != SA_OK) return rc;
  if (kv_nothing(a->seqs)) return ok();
  const int size = kv_type_bytes(a->dtype);
  const int64_t width = (int64_t)a->cache.Hkv * a->cache.D;
  KvRows k, v;
  rc = kv_rows(a->k, a->k_off, a->ldk, width, a->seqs.T, size, "k", &k);
  if (rc == SA_OK) rc = kv_rows(a->v, a->v_off, a->ldv, width, a->seqs.T, size, "v", &v);
  if (rc != SA_OK) return rc;
  if (kv_overlap_cache(k, a->cache) || kv_overlap_cache(v, a->cache)) return fail(SA_ERR_ALIAS, "the rows overlap the cache");
  if (!write) {
    if (kv_overlap(k, v)) return fail(SA_ERR_ALIAS, "k overlaps v");
    if (kv_overlap_seqs(k, a->seqs) || kv_overlap_seqs(v, a->seqs)) return fail(SA_ERR_ALIAS, "k or v overlaps the sequences' arrays");
  }
  KvMove m;
  m.c = a->cache;
  m.s = a->seqs;
  m.k = const_cast<char*>(k.lo);
  m.v = const_cast<char*>(v.lo);
  m.ldk = k.ld;
  m.ldv = v.ld;
  const int64_t blocks = ((int64_t)a->seqs.max_rows + 30) / 32 + 1;  // r tokens touch at most (r + 62) / 32 blocks
  m.blocks = (int)blocks;
  m.tiles = a->seqs.B * blocks * a->cache.Hkv * 2;
  if (m.tiles > (int64_t)0x7fffffff * kWaves) return fail(SA_ERR_UNSUPPORTED, "%lld tiles in one call", (long long)m.tiles);
  // every access of the aligned kernels is of 16 bytes or of a lane's channels at a multiple of them
  const bool aligned = (((uintptr_t)k.lo | (uintptr_t)v.lo | (uintptr_t)k.ld | (uintptr_t)v.ld) & 15) == 0;
  const hipError_t e = a->dtype == SA_DT_F32   ? launch_t<float>(m, write, aligned, (hipStream_t)stream)
                       : a->dtype == SA_DT_F16 ? launch_t<_Float16>(m, write, aligned, (hipStream_t)stream)
                                               : launch_t<__bf16>(m, write, aligned, (hipStream_t)stream);
  return e == hipSuccess ? ok() : hip_fail(e, write ? "kv_write" : "kv_read");
}

}  // namespace

}  // namespace sa

using sa::fail;
using sa::ok;

extern "C" {

int64_t sa_kv_cache_bytes(int32_t pages, int32_t Hkv, int32_t D) {
  if (pages <= 0 || Hkv <= 0 || D <= 0) return fail(SA_ERR_INVALID, "pages, Hkv and D must be positive (got %d, %d, %d)", pages, Hkv, D);
  if (D != 64 && D != 128 && D != 256) return fail(SA_ERR_UNSUPPORTED, "head dim %d: the cache holds 64, 128 or 256", D);
  if (Hkv > 4096) return fail(SA_ERR_UNSUPPORTED, "%d key heads (at most 4096)", Hkv);
  ok();
  return (int64_t)pages * Hkv * SA_KV_BLOCK * D;
}

int sa_kv_write(const sa_kv_rows_args* args, void* stream) { return sa::kv_move(args, true, stream); }

int sa_kv_read(const sa_kv_rows_args* args, void* stream) { return sa::kv_move(args, false, stream); }

}  // extern "C"
