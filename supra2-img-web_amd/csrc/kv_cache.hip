// The 8-bit key/value cache written and read back (include/supra_kv.h).
//
// A page and head of K or V is one tile of 32 tokens x D codes with one exponent byte. Both kernels give a wave one
// such tile: what it reads and writes is contiguous on the cache's side and whole rows' heads on the other, and
// the page's scale is a reduction inside the wave, so the rows are read once and stay in registers until it is known.
// Which sequence, page and head that is follows from the workgroup index and the device's own lengths; waves beyond a
// sequence's pages end at once. Two waves to a workgroup: four hold its registers until the slowest is done (33 us
// against 36 for the prompts below, with the earlier codes of a page loaded only by waves that must keep some).
//
// Quantising: with e the page's exponent byte, code = e4m3(x * 2^(127 - e)). v_cvt_scalef32_pk_fp8_* takes the
// factor as a power of two and rounds once, to nearest even (46 us with a multiplication and a conversion each). A
// page that holds earlier tokens keeps max(its exponent, the new tokens'): codes that must move to a larger scale
// are decoded, which is exact, and rounded at the new one the same way.
//
// Bound: HBM traffic. Written and read back: 5 prompts of 1 .. 4095 tokens, 8 heads x 128, bfloat16, 33 us for 129 MB,
// 3.9 TB/s (a copy of 4 GiB reaches 4.6). One new token of each of 64 sequences, 13 us for both launches: latency, a page
// rewritten for a token.

#include <hip/hip_runtime.h>

#include "common.h"
#include "kv_check.h"
#include "kv_layout.h"
#include "row_types.h"

namespace sa {

namespace {

constexpr int kWaves = 2;  // tiles per workgroup

struct KvMove {
  sa_kv_cache c;
  sa_kv_seqs s;
  char* k;  // the rows (offset included)
  char* v;
  int64_t ldk, ldv;  // bytes
  int blocks;        // tiles of one head that a sequence's rows can touch
  uint32_t tiles;    // B * blocks * Hkv * 2
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

__device__ __forceinline__ bool kv_tile_of(const KvMove& a, uint32_t i, Tile* t) {
  if (i >= a.tiles) return false;
  t->is_v = i & 1;
  i >>= 1;
  const uint32_t heads = (uint32_t)a.c.Hkv, blocks = (uint32_t)a.blocks;
  t->h = (int)(i % heads);
  i /= heads;
  const int n = (int)(i % blocks), b = (int)(i / blocks);
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

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, m));
  return x;
}

// Two neighbouring elements as they come from memory, and what the kernels do to them: the larger magnitude, two
// codes at a scale, two elements of two codes.
template <typename T>
struct Pair {
  uint32_t w;
  typedef T T2 __attribute__((ext_vector_type(2)));
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  static constexpr uint16_t kInf = __is_same(T, __bf16) ? 0x7f80 : 0x7c00;  // bits of infinity

  __device__ __forceinline__ void put(T a, T b) { w = __builtin_bit_cast(uint32_t, T2{a, b}); }
  __device__ __forceinline__ T2 both() const { return __builtin_bit_cast(T2, w); }
  // Running maximum of both halves' magnitudes (as bits, which order like the magnitudes); the float32 bits of it.
  __device__ __forceinline__ static void most(uint32_t& m, Pair p, bool finite) {
    u16x2 a = __builtin_bit_cast(u16x2, p.w & 0x7fff7fffu);
    if (finite) {
      a[0] = a[0] < kInf ? a[0] : (uint16_t)0;
      a[1] = a[1] < kInf ? a[1] : (uint16_t)0;
    }
    m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), a));
  }
  __device__ __forceinline__ static uint32_t f32_bits(uint32_t m) {
    const uint16_t x = (uint16_t)max(m & 0xffffu, m >> 16);
    return __float_as_uint((float)__builtin_bit_cast(T, x));
  }
};

template <>
struct Pair<float> {
  float a, b;
  __device__ __forceinline__ void put(float x, float y) { a = x, b = y; }
  __device__ __forceinline__ static void most(uint32_t& m, Pair p, bool finite) {
    uint32_t x = __float_as_uint(p.a) & 0x7fffffffu, y = __float_as_uint(p.b) & 0x7fffffffu;
    if (finite) {
      x = x < 0x7f800000u ? x : 0u;
      y = y < 0x7f800000u ? y : 0u;
    }
    m = max(m, max(x, y));
  }
  __device__ __forceinline__ static uint32_t f32_bits(uint32_t m) { return m; }
};

typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

// Codes of a pair's elements / scale, scale a power of two, in one rounding to nearest even, into half HI of `to`.
template <bool HI, typename T>
__device__ __forceinline__ i16x2 codes2(i16x2 to, Pair<T> p, float scale) {
  if constexpr (__is_same(T, float)) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(to, p.a, p.b, scale, HI);
  else if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(to, p.both(), scale, HI);
  else return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(to, p.both(), scale, HI);
}
template <typename T>
__device__ __forceinline__ uint32_t codes4(Pair<T> p, Pair<T> q, float scale) {
  i16x2 w = {0, 0};
  w = codes2<false>(w, p, scale);
  return __builtin_bit_cast(uint32_t, codes2<true>(w, q, scale));
}

// The values (code * scale, rounded to T once) of half HI's two codes.
template <bool HI, typename T>
__device__ __forceinline__ Pair<T> values2(uint32_t w, float scale) {
  Pair<T> p;
  if constexpr (__is_same(T, float)) {
    const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, HI);
    p.put(x[0], x[1]);
  } else if constexpr (__is_same(T, _Float16)) {
    p.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  } else {
    p.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  }
  return p;
}

template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void load_pairs(const T* p, Pair<T> (&x)[N]) {
  static_assert(sizeof(Pair<T>) == 2 * sizeof(T), "pairs are their elements' bytes");
  if constexpr (ALIGNED) {
    uint32_t w[N * sizeof(T) / 2];
    load_words<N * 2 * sizeof(T)>(p, w);
    __builtin_memcpy(x, w, sizeof(w));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i].put(p[2 * i], p[2 * i + 1]);
  }
}

template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void store_pairs(T* p, const Pair<T> (&x)[N]) {
  if constexpr (ALIGNED) {
    uint32_t w[N * sizeof(T) / 2];
    __builtin_memcpy(w, x, sizeof(w));
    store_words<N * 2 * sizeof(T)>(p, w);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (__is_same(T, float)) p[2 * i] = x[i].a, p[2 * i + 1] = x[i].b;
      else p[2 * i] = x[i].both()[0], p[2 * i + 1] = x[i].both()[1];
    }
  }
}

// The four codes of w at a scale 1/factor times as large: decoded, multiplied, rounded.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float factor) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  int x = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * factor, a[1] * factor, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * factor, b[1] * factor, x, true);
}

// V's part of a tile in one lane: kPairs pairs of channels from channel() on, and the tokens of kWords words of four:
// all 32, or (head dim 64) those of the lane's half.
template <int D>
struct VPart {
  static constexpr int kPairs = D == 256 ? 2 : 1, kWords = D == 64 ? 4 : 8;
  int lane;
  __device__ __forceinline__ int channel() const { return D == 64 ? 2 * (lane & 31) : lane * 2 * kPairs; }
  __device__ __forceinline__ int word(int k) const { return D == 64 ? 4 * (lane >> 5) + k : k; }
  // the first token of word k; tokens 8 (word & 3) + 4 (word >> 2) + 0..3
  __device__ __forceinline__ int token(int k) const { return 8 * (word(k) & 3) + 4 * (word(k) >> 2); }
};

// Bytes of word w4 (tokens t .. t + 3) that belong to the tokens of the mask.
__device__ __forceinline__ uint32_t bytes_of(uint32_t mask, int t) {
  uint32_t b = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) b |= (mask >> (t + r) & 1u) ? 0xffu << (8 * r) : 0u;
  return b;
}

template <typename T, int D, bool ALIGNED>
__global__ __launch_bounds__(64 * kWaves) void kv_write_kernel(KvMove a) {
  const int lane = threadIdx.x & 63;
  Tile t;
  if (!kv_tile_of(a, blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), &t)) return;
  if (t.page < 0) return;
  const int64_t at = kv_tile(t.page, a.c.Hkv, t.h, D);
  const bool keeps = t.lo > 0 && t.q.first > 0;  // the block holds earlier tokens: places [0, lo)
  uint8_t* scale = (t.is_v ? a.c.v_scale : a.c.k_scale) + (int64_t)t.page * a.c.Hkv + t.h;
  const int held = min((int)*scale, 254), old = keeps ? held : 0;
  // The page's exponent: of the largest magnitude among the new tokens (over all of them first; where that is no
  // number, over the finite ones), and not below the one it has.
  const auto exponent = [&](auto most) {
    uint32_t m = wave_max(Pair<T>::f32_bits(most(false)));
    if (m >= 0x7f800000u) m = wave_max(Pair<T>::f32_bits(most(true)));
    return max(kv_exponent(m), old);
  };
  if (!t.is_v) {
    // 16 codes per lane and step: a token's 16 channels, D/16 lanes across its row
    constexpr int N = D / 32, R = D / 16;
    Pair<T> x[N][8];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * 64 + lane, tok = id / R, d = id % R * 16;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j].put((T)0.f, (T)0.f);
      if (tok >= t.lo && tok < t.hi) load_pairs<T, 8, ALIGNED>(reinterpret_cast<const T*>(a.k + (int64_t)(t.row + tok) * a.ldk) + t.h * D + d, x[i]);
    }
    const int e = exponent([&](bool finite) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) Pair<T>::most(m, x[i][j], finite);
      return m;
    });
    const float step = __uint_as_float((uint32_t)e << 23);  // 2^(e - 127), as the conversions read it: exponent bits alone
    const bool grows = keeps && e > old;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * 64 + lane, tok = id / R, d = id % R * 16;
      uint8_t* p = a.c.k + at + kv_k_place(tok, d);
      uint32_t w[4];
      if (tok >= t.lo && tok < t.hi) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = codes4(x[i][2 * j], x[i][2 * j + 1], step);
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
    // A lane's tokens of its own channels: the transposed tile needs no exchange between lanes.
    using Part = VPart<D>;
    const Part part{lane};
    constexpr int E = Part::kPairs, K = Part::kWords;
    uint8_t* base = a.c.v + at + part.channel() * 32 + 4 * part.word(0);
    const bool whole = t.lo == 0 && t.hi == 32;
    uint32_t had[2 * E][K];
    Pair<T> x[K][4][E];
    const T* rows = reinterpret_cast<const T*>(a.v + (int64_t)t.row * a.ldv) + t.h * D + part.channel();
    const int64_t ld = a.ldv / (int64_t)sizeof(T);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = part.token(k) + r;
#pragma unroll
        for (int j = 0; j < E; ++j) x[k][r][j].put((T)0.f, (T)0.f);
        if (tok >= t.lo && tok < t.hi) load_pairs<T, E, ALIGNED>(rows + tok * ld, x[k][r]);
      }
    const int e = exponent([&](bool finite) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < E; ++j) Pair<T>::most(m, x[k][r][j], finite);
      return m;
    });
    const float step = __uint_as_float((uint32_t)e << 23);
    const bool grows = keeps && e > old;
    const float f = __uint_as_float(kv_pow2_bits(old - e));
    if (!whole) {
#pragma unroll
      for (int c = 0; c < 2 * E; ++c) load_words<4 * K>(base + 32 * c, had[c]);
    }
    const uint32_t olds = (1u << t.lo) - 1u, news = (t.hi == 32 ? 0xffffffffu : (1u << t.hi) - 1u) & ~olds;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      uint32_t w[2][K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const uint32_t lo = codes4(x[k][0][j], x[k][1][j], step), hi = codes4(x[k][2][j], x[k][3][j], step);
        w[0][k] = __builtin_amdgcn_perm(hi, lo, 0x06040200u);  // four tokens of the pair's first channel
        w[1][k] = __builtin_amdgcn_perm(hi, lo, 0x07050301u);
        if (!whole) {
          const uint32_t mn = bytes_of(news, part.token(k)), mo = bytes_of(olds, part.token(k));
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t was = had[2 * j + c][k];
            uint32_t moved = was;
            if (grows) moved = rescale4(was, f);
            w[c][k] = (w[c][k] & mn) | (moved & mo) | (was & ~(mn | mo));
          }
        }
      }
      store_words<4 * K>(base + 64 * j, w[0]);
      store_words<4 * K>(base + 64 * j + 32, w[1]);
    }
    if (lane == 0) *scale = (uint8_t)e;
  }
}

template <typename T, int D, bool ALIGNED>
__global__ __launch_bounds__(64 * kWaves) void kv_read_kernel(KvMove a) {
  const int lane = threadIdx.x & 63;
  Tile t;
  if (!kv_tile_of(a, blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), &t)) return;
  const bool none = t.page < 0;  // its codes are taken as zeros
  const int64_t page = none ? 0 : t.page, at = kv_tile(page, a.c.Hkv, t.h, D);
  const int e = (t.is_v ? a.c.v_scale : a.c.k_scale)[page * a.c.Hkv + t.h];
  const float step = __uint_as_float((uint32_t)min(e, 254) << 23);  // 2^(e - 127), as the conversions read it
  if (!t.is_v) {
    constexpr int N = D / 32, R = D / 16;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * 64 + lane, tok = id / R, d = id % R * 16;
      if (tok < t.lo || tok >= t.hi) continue;
      uint32_t w[4] = {0, 0, 0, 0};
      if (!none) load_words<16>(a.c.k + at + kv_k_place(tok, d), w);
      Pair<T> x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = values2<false, T>(w[j], step);
        x[2 * j + 1] = values2<true, T>(w[j], step);
      }
      store_pairs<T, 8, ALIGNED>(reinterpret_cast<T*>(a.k + (int64_t)(t.row + tok) * a.ldk) + t.h * D + d, x);
    }
  } else {
    using Part = VPart<D>;
    const Part part{lane};
    constexpr int E = Part::kPairs, K = Part::kWords;
    uint32_t w[2 * E][K];
#pragma unroll
    for (int c = 0; c < 2 * E; ++c) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[c][k] = 0;
      if (!none) load_words<4 * K>(a.c.v + at + (part.channel() + c) * 32 + 4 * part.word(0), w[c]);
    }
    T* rows = reinterpret_cast<T*>(a.v + (int64_t)t.row * a.ldv) + t.h * D + part.channel();
    const int64_t ld = a.ldv / (int64_t)sizeof(T);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Pair<T> x[4][E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        // tokens 0, 1 and 2, 3 of the word, a channel pair of each in a half
        const uint32_t lo = __builtin_amdgcn_perm(w[2 * j + 1][k], w[2 * j][k], 0x05010400u),
                       hi = __builtin_amdgcn_perm(w[2 * j + 1][k], w[2 * j][k], 0x07030602u);
        x[0][j] = values2<false, T>(lo, step);
        x[1][j] = values2<true, T>(lo, step);
        x[2][j] = values2<false, T>(hi, step);
        x[3][j] = values2<true, T>(hi, step);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = part.token(k) + r;
        if (tok >= t.lo && tok < t.hi) store_pairs<T, E, ALIGNED>(rows + tok * ld, x[r]);
      }
    }
  }
}

template <typename T, int D>
hipError_t launch_d(const KvMove& a, bool write, bool aligned, hipStream_t stream) {
  const dim3 grid((a.tiles + kWaves - 1) / kWaves), block(64 * kWaves);
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
  int64_t tiles = 0;  // 32-bit in the kernel: divisions of 64 bits took longer there than the tile itself
  if (__builtin_mul_overflow(a->seqs.B * blocks, (int64_t)a->cache.Hkv * 2, &tiles) || tiles > kKvMaxThreads / 64 - kWaves)
    return fail(SA_ERR_UNSUPPORTED, "2 * Hkv tiles of each 32 rows of each sequence: more than 2^26 in one call");
  m.tiles = (uint32_t)tiles;
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
