// Attention over the 8-bit key/value cache (include/supra_kv.h).
//
// A row is one token's query head: the rows t * G + g of one key head share its K and V, whatever token they are of. A
// workgroup takes a group of such rows and a share of the sequence's pages. S^T = K Q^T leaves a row's scores in the
// lanes that need them as the second operand of O^T += V^T P^T, and the cache's V codes lie in that order: neither K, V
// nor P changes lanes, and a page's K and V come as 16-byte loads of 1 KiB per wave. The maximum and sum of the softmax
// run along in float32. Two kernels, chosen by the call's rows (kv_attn_plan):
//
// kv_attn_split_kernel, few rows: 16 or 32 rows to a workgroup, whose four or eight waves take the pages in turn and
//   are merged at the end. Bound by the cache's bytes: 64 sequences of 333 .. 8191 tokens, 8 key heads x 128, 117 us or
//   4.8 TB/s of codes (a copy of 4 GiB reaches 4.6); 2 of 131000 tokens at 4 x 128, 54 us with their merge. Where there
//   are too few workgroups the pages are split over several, whose records kv_attn_merge_kernel joins.
// kv_attn_rows_kernel, rows for some 512 workgroups of 128 and more: 128 to a workgroup, 32 to a wave, the pages through LDS for all four. Bound by the issue
//   of the matrix and vector instructions together: 4 x 2048 rows over 4096 keys, 32 heads x 128, bfloat16, 565 us or
//   0.97 PFLOP/s, with vector instructions in 59% of the cycles and matrix ones in 40% (an 8192^3 product of the
//   library: 1.2). Short calls of it are bound by q and o instead: 64 x 256 rows over up to 128 keys, 9 heads x 64,
//   float32, 25 us for 75 MB.
//
// Numbers. K and V codes are exact in float16 (v_cvt_scalef32_pk_f16_fp8), V's with its page's scale relative to the
// largest one so far (2^m_v; a growing one rescales the sums like the running maximum). Q is brought to float16 by a
// power of two of each row, its largest magnitude in [2^14, 2^15): float16 and bfloat16 rows in one term, exactly down
// to 2^-28 of the row's largest element; float32 rows in two terms, 22 bits of each element. (The kernel of many rows
// takes bfloat16 rows in two e4m3 terms: QCodes.) The probabilities, at 2^kPBias for the running maximum, are one
// float16 term (11 bits: half a step of it is a sixteenth of a bfloat16 output's, and half a float16 one's, before the
// sum averages them) or two for float32 rows. Sums, maxima and products are float32.
//
// V relative to the largest scale: codes times 2^(e - m_v + 6) stay exact for pages down to 2^-21 of the largest
// page of the head, and below that are off by at most 2^-40 of its largest value.

#include <hip/hip_runtime.h>

#include <math.h>

#include "common.h"
#include "kv_check.h"
#include "kv_layout.h"
#include "row_types.h"

namespace sa {

namespace {

constexpr int kCUs = 256;      // of an MI355X: what the splits are planned for
constexpr int kRows = 32;      // rows of a workgroup
constexpr int kPBias = 10;     // log2 of a probability's scale at the running maximum
constexpr float kLazy = 4.f;   // the maximum moves when a score passes it by more than this (log2): P stays below 2^14
constexpr int kVBias = 6;      // log2 of V's scale at the largest page

struct KvAttnParams {
  sa_kv_cache c;
  sa_kv_seqs s;
  const char* q;  // offset included; strides in bytes
  char* o;
  int64_t ldq, ldo;
  float* ws;      // records of the splits, or null
  float scale_log2;
  int H, G;       // query heads, and of one key head
  int causal;
  int groups;     // row groups of a sequence (of max_rows)
  int splits;
  int aligned_q, aligned_o;  // rows of 16-byte aligned heads
  int ordered;    // many rows: the workgroups with most pages first
  int len_blocks; // pages of the longest sequence, as the caller has it
};

template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;

__device__ __forceinline__ f16x8 half8(uint32_t a, uint32_t b, float scale) {
  const f16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true),
              x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true);
  return f16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

__device__ __forceinline__ f16x8 round8(const float* x) {
  f16x8 y;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const f16x2 p = __builtin_convertvector((f32x2{x[i], x[i + 1]}), f16x2);
    y[i] = p[0], y[i + 1] = p[1];
  }
  return y;
}

// hi[0..NT): x in NT float16 terms.
template <int NT>
__device__ __forceinline__ void split8(const float* x, f16x8 (&y)[NT]) {
  y[0] = round8(x);
  if constexpr (NT == 2) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i] - (float)y[0][i];
    y[1] = round8(r);
  }
}

__device__ __forceinline__ f32x16 mfma(const f16x8& a, const f16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// What a workgroup works on.
struct Work {
  KvSeq q;
  int b, hk, row0, rows;  // packed rows from row0 on, of `rows` in all (tokens * G)
  int blocks;             // pages that any of its rows attends to
};

__device__ __forceinline__ bool kv_work(const KvAttnParams& a, int rows, int group, int hk, int b, Work* w) {
  w->q = kv_seq(a.s, b);
  w->b = b;
  w->hk = hk;
  w->row0 = group * rows;
  w->rows = w->q.rows * a.G;
  if (w->row0 >= w->rows) return false;
  int keys = w->q.len;
  if (a.causal) {
    const int t = (min(w->row0 + rows, w->rows) - 1) / a.G;  // the last row's token
    keys = max(0, min(keys, w->q.first + t + 1));
  }
  w->blocks = (keys + kKvBlock - 1) / kKvBlock;
  return true;
}

// Factor that brings a row whose largest magnitude has the bits m to float16: 2^(14 - its exponent), with the scale's
// sign; the row is 2^exponent times that. A row with an infinity or NaN has infinite or NaN scores alone, and so NaN
// where it attends to anything, also where they are all -infinity, which the running maximum would pass over: NaN.
__device__ __forceinline__ float q_factor(const KvAttnParams& a, uint32_t m, int& exponent) {
  const int f = min(127 + 14 + 127 - (int)(m >> 23), 253);
  exponent = 127 - f;
  return m >= 0x7f800000u ? NAN : copysignf(__uint_as_float((uint32_t)f << 23), a.scale_log2);
}

// Q's operand for one 32-row group. float16 terms, one for float16 rows and two for float32: lane (row = lane & 31, half) has elements 32 c +
// 16 half .. + 16 of each chunk c.
template <typename T, int D>
struct QTile {
  f16x8 t[D / 32][2][kTerms<T>];
  int exponent;  // the row's elements are 2^exponent times the operand's
};

// bfloat16 rows, e4m3 terms for the scaled 32x32x64 products, in the same places: word 0..3 of operand i chunk 2 i, 4..7 chunk
// 2 i + 1, each with the scale of the row's 32 elements of that chunk, which lanes of half 0 and half 1 give (the
// instruction takes the scale of both halves' first 16 bytes from the one and of their last 16 from the other). K's codes
// are the other operand as they are, its page's exponent their scale. A bfloat16 element has 8 bits, two terms of 4:
// against one float16 term K needs no conversion (4 x 2048 rows over 4096 keys at 32 heads x 128: 598 us -> 560). A
// float16 element would take three (16 heads x 64: 130 -> 132) and keeps the float16 products.
typedef int i32x8 __attribute__((ext_vector_type(8)));
constexpr int kTerms8 = 2;
template <typename T>
constexpr bool kCodes = __is_same(T, __bf16);  // rows that the kernel of many rows takes in e4m3 terms

template <typename T, int D>
struct QCodes {
  i32x8 t[D / 64][kTerms8];
  int e[D / 64];  // exponent byte of the first term's chunk 2 i + half; the second's is 4 less
};

// Rows of 32 in one wave, as memory has them and as the operands want them. Memory: a chunk of 32 channels of a row is
// 16-byte parts in neighbouring lanes; operands: lane (row = lane & 31, half) has the chunk's 16 channels of its half.
// Loading or storing the operands' form directly touches another row in every lane, which costs the address unit four
// times as long; so the rows go through LDS, each wave in its own kRowsLds bytes, in order (64-image cross-attention in
// float32 26.2 -> 25.4 us, in bfloat16 21.2 -> 18.8).
constexpr int kRowsLds = 32 * 144;

// The row's place in q or o, in bytes; negative for rows past the last.
__device__ __forceinline__ int64_t row_place(const KvAttnParams& a, const Work& w, int row, int64_t ld, int head_bytes) {
  return row < w.rows ? (int64_t)(w.q.row0 + row / a.G) * ld + (int64_t)(w.hk * a.G + row % a.G) * head_bytes : -1;
}
__device__ __forceinline__ int64_t of_lane(int64_t x, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__shfl((int)(x >> 32), lane) << 32 | (uint32_t)__shfl((int)x, lane));
}

// A wave's 32 rows of q in float32: lane (row, half): channels 32 c + 16 half on.
template <typename T, int D>
__device__ __forceinline__ void load_rows32(const KvAttnParams& a, const Work& w, int lane, char* lds, float (&x)[D / 32][16]) {
  constexpr int C = D / 32;
  const int half = lane >> 5;
  const int64_t place = row_place(a, w, w.row0 + (lane & 31), a.ldq, D * (int)sizeof(T));
  if (a.aligned_q) {
    constexpr int PARTS = 2 * (int)sizeof(T), STEPS = PARTS / 2, STRIDE = 16 * PARTS + 16;  // of a chunk's row; wave steps of 64
    static_assert(32 * STRIDE <= kRowsLds, "the chunk fits");
    u32x4 raw[C][STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int id = 64 * i + lane;
      const int64_t from = of_lane(place, id / PARTS);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        raw[c][i] = u32x4{0, 0, 0, 0};
        if (from >= 0) raw[c][i] = *reinterpret_cast<const u32x4*>(a.q + from + 32 * c * (int)sizeof(T) + id % PARTS * 16);
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int id = 64 * i + lane;
        *reinterpret_cast<u32x4*>(lds + id / PARTS * STRIDE + id % PARTS * 16) = raw[c][i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      load_row<T, 16, true>(reinterpret_cast<const T*>(lds + (lane & 31) * STRIDE + half * 8 * PARTS), x[c]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[c][j] = 0.f;
      if (place >= 0) load_row<T, 16, false>(reinterpret_cast<const T*>(a.q + place) + 32 * c + 16 * half, x[c]);
    }
  }
}

template <typename T, int D>
__device__ __forceinline__ void load_q(const KvAttnParams& a, const Work& w, int lane, QTile<T, D>& q, char* lds) {
  float x[D / 32][16];
  load_rows32<T, D>(a, w, lane, lds, x);
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(x[c][i]) & 0x7fffffffu);
  auto sw = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = max(sw[0], sw[1]);
  const float factor = q_factor(a, m, q.exponent);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[c][i] *= factor;
    split8<kTerms<T>>(x[c], q.t[c][0]);
    split8<kTerms<T>>(x[c] + 8, q.t[c][1]);
  }
}

// The second term is the rest of the first, at a 16th of its scale: with the first scale the smallest that keeps the
// largest element within 448, the rest is at most half a step of 32, 16 = 256 sixteenths. Elements down to 2^-14 of the
// largest of their 32 are exact, smaller ones within 2^-22 of it.
template <typename T, int D>
__device__ __forceinline__ void load_q(const KvAttnParams& a, const Work& w, int lane, QCodes<T, D>& q, char* lds) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  float x[D / 32][16];
  load_rows32<T, D>(a, w, lane, lds, x);
  const uint32_t sign = __float_as_uint(a.scale_log2) & 0x80000000u;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[c][j] = __uint_as_float(__float_as_uint(x[c][j]) ^ sign);
      m = max(m, __float_as_uint(x[c][j]) & 0x7fffffffu);
    }
    auto sw = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    const int e = max(kv_exponent(max(sw[0], sw[1])), 4 * (kTerms8 - 1));
    if ((c & 1) == lane >> 5) q.e[c / 2] = e;
#pragma unroll
    for (int t = 0; t < kTerms8; ++t) {
      const float step = __uint_as_float((uint32_t)(e - 4 * t) << 23);
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        i16x2 w2 = {0, 0};
        w2 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w2, x[c][j], x[c][j + 1], step, false);
        w2 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w2, x[c][j + 2], x[c][j + 3], step, true);
        const int word = __builtin_bit_cast(int, w2);
        q.t[c / 2][t][4 * (c & 1) + j / 4] = word;
        if (t + 1 < kTerms8) {
          const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, step, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, step, true);
          x[c][j] -= lo[0], x[c][j + 1] -= lo[1], x[c][j + 2] -= hi[0], x[c][j + 3] -= hi[1];
        }
      }
    }
  }
}

// The running state of 32 rows in one wave: O^T (chunk c, register 4 g + r of half h: element 32 c + 8 g + 4 h + r of
// row lane & 31), the maximum (log2 units, one for both halves of a row) and this half's sum.
template <int D>
struct State {
  f32x16 o[D / 32];
  float m, l;
  int mv;  // exponent byte of V's reference scale
};

// Codes 0x7f and 0xff are NaN: bit 7 of their bytes.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
  const uint32_t n = nan_bytes(w);
  return w & ~(n | (n - (n >> 7)));
}
__device__ __forceinline__ uint32_t ones_at_nan(uint32_t w) { return (nan_bytes(w) >> 7) * 0x38u; }  // 0x38: the code of 1

// S^T of a page, and the factor that makes it log2 units. k(c): the lane's 16 bytes of KiB c of the K tile.
template <typename T, int D, typename K>
__device__ __forceinline__ f32x16 scores(const QTile<T, D>& q, const K& k, int ke, float scale_log2, float& f) {
  f32x16 s = zero16();
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const u32x4 x = k(c);
    const f16x8 k0 = half8(x[0], x[1], 1.f), k1 = half8(x[2], x[3], 1.f);
#pragma unroll
    for (int t = kTerms<T> - 1; t >= 0; --t) {
      s = mfma(k0, q.t[c][0][t], s);
      s = mfma(k1, q.t[c][1][t], s);
    }
  }
  f = ldexpf(scale_log2, q.exponent + ke - 127);  // >= 0
  return s;
}

template <typename T, int D, typename K>
__device__ __forceinline__ f32x16 scores(const QCodes<T, D>& q, const K& k, int ke, float scale_log2, float& f) {
  f32x16 s = zero16();
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const u32x4 lo = k(2 * i), hi = k(2 * i + 1);
    const i32x8 x = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
#pragma unroll
    for (int t = kTerms8 - 1; t >= 0; --t) s = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, q.t[i][t], s, 0, 0, 0, ke, 0, q.e[i] - 4 * t);
  }
  f = scale_log2;
  return s;
}

// One page of 32 keys. k(c), v(c): the lane's 16 bytes of KiB c of its K and V tiles. MASKED: of the page's keys each row
// attends to the first `limit` (its own).
template <typename T, int D, bool MASKED, typename Q, typename LoadK, typename LoadV>
__device__ __forceinline__ void step(const Q& q, State<D>& st, const LoadK& k, const LoadV& v, int ke, int ve, float scale_log2,
                                     int lane, int limit) {
  constexpr int NT = kTerms<T>;
  // Where registers allow, the whole page is on its way before the first product (the compiler would fetch V's part
  // after the exponentials: 571 us against 565 for 4 x 2048 rows over 4096 keys at 32 heads x 128).
  constexpr bool EARLY = D == 128 || (D == 64 && sizeof(T) == 4);
  u32x4 kr[D / 32], vr[D / 32];
  if constexpr (EARLY) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) kr[c] = k(c);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) vr[c] = v(c);
    __builtin_amdgcn_sched_barrier(0);
  }
  float f;
  f32x16 s = scores(q, [&](int c) { return EARLY ? kr[c] : k(c); }, ke, scale_log2, f);
  const int half = lane >> 5;
  float top;
  if constexpr (MASKED) {
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = 8 * (i >> 2) + 4 * half + (i & 3) < limit ? s[i] * f : -INFINITY;
      top = max_nan(top, s[i]);
    }
  } else {
    top = max_nan(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) top = max_nan(top, s[i]);
    top *= f;
  }
  top = max_with_partner(top);
  const bool grows = !(top <= st.m + kLazy), v_grows = ve > st.mv;
  if (__any(grows) || v_grows) {
    const float m = grows ? max_nan(st.m, top) : st.m;
    float r = fast_exp2(st.m - m);
    st.l *= r;
    if (v_grows) {
      r *= __uint_as_float(kv_pow2_bits(st.mv - ve));
      st.mv = ve;
    }
    st.m = m;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[c][i] *= r;
  }
  const float base = (float)kPBias - st.m;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = fast_exp2(MASKED ? s[i] + base : fmaf(s[i], f, base));
  f16x8 p0[NT], p1[NT];
  {
    float p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = s[i];
    split8<NT>(p, p0);
    split8<NT>(p + 8, p1);
    if constexpr (NT == 1) {
      // the sum of the probabilities as they enter the product: two of them in one instruction, exact products
      const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        st.l = __builtin_amdgcn_fdot2(f16x2{p0[0][i], p0[0][i + 1]}, one, st.l, false);
        st.l = __builtin_amdgcn_fdot2(f16x2{p1[0][i], p1[0][i + 1]}, one, st.l, false);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) st.l += p[i];
    }
  }
  const float vs = __uint_as_float((uint32_t)max(ve - st.mv + kVBias + 127, 1) << 23);
  bool nan_v = false;
  if constexpr (MASKED) {
    // A key that a row does not attend to may hold NaN in V, and 0 * NaN is not 0.
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const u32x4 x = v(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= nan_bytes(x[i]);
    }
    nan_v = __any(any != 0);
  }
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    u32x4 x = EARLY ? vr[c] : v(c);
    if (MASKED && nan_v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = without_nan(x[i]);
    }
    const f16x8 v0 = half8(x[0], x[1], vs), v1 = half8(x[2], x[3], vs);
#pragma unroll
    for (int t = NT - 1; t >= 0; --t) {
      st.o[c] = mfma(v0, p0[t], st.o[c]);
      st.o[c] = mfma(v1, p1[t], st.o[c]);
    }
  }
  if (MASKED && nan_v) {
    // The places of the NaN codes, which left the tile, times the attended keys: whose sums they turn into NaN.
    float seen[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) seen[i] = 8 * (i >> 2) + 4 * half + (i & 3) < limit ? 1.f : 0.f;
    const f16x8 s0 = round8(seen), s1 = round8(seen + 8);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      u32x4 x = v(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = ones_at_nan(x[i]);
      const f32x16 hits = mfma(half8(x[2], x[3], 1.f), s1, mfma(half8(x[0], x[1], 1.f), s0, zero16()));
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[c][i] = hits[i] > 0.f ? NAN : st.o[c][i];
    }
  }
}

// A split's record of a group of `rows` rows: rows x D floats, then their log2-sums.
__host__ __device__ constexpr int64_t record_floats(int rows, int D) { return (int64_t)rows * (D + 1); }
__device__ __forceinline__ int64_t record_at(const KvAttnParams& a, int b, int hk, int group, int split, int rows, int D) {
  return ((((int64_t)b * a.c.Hkv + hk) * a.groups + group) * a.splits + split) * record_floats(rows, D);
}

template <typename T, int D>
__device__ __forceinline__ void store_o4(const KvAttnParams& a, const Work& w, int row, int d, f32x4 x) {
  T* p = reinterpret_cast<T*>(a.o + (int64_t)(w.q.row0 + row / a.G) * a.ldo) + (int64_t)(w.hk * a.G + row % a.G) * D + d;
  const float y[4] = {x[0], x[1], x[2], x[3]};
  if (a.aligned_o) store_row<T, 4, true>(p, y);
  else store_row<T, 4, false>(p, y);
}

// ---- few rows: 16 or 32 of them to a workgroup, whose waves take the pages in turn and are merged at the end. Tiles of
// 16x16x32 instructions: S^T of 16 keys x 16 rows leaves the keys 4 kq + i of a tile in lane (row, kq = lane >> 4), and the
// two tiles of a page take its tokens in the order that makes those of one lane eight neighbouring codes of V:
// tile u, place p: token 16 ((p >> 2) & 1) + 8 u + 4 (p >> 3) + (p & 3).

__device__ __forceinline__ f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ int token16(int u, int p) { return 16 * (p >> 2 & 1) + 8 * u + 4 * (p >> 3) + (p & 3); }

// One page's codes as a lane needs them: K: of pair i of 32-channel chunks and tile u, 16 channels of one token
// (channels 64 i + 16 kq on); V: of channel 16 e + (lane & 15), eight tokens.
template <int D>
struct Page16 {
  u32x4 k[D / 64][2];
  uint2 v[D / 16];
  int ke, ve;
  bool ok;
};

template <int D>
__device__ __forceinline__ void load_page(const KvAttnParams& a, int hk, int32_t id, int lane, Page16<D>& p) {
  p.ok = kv_page_ok(id, a.c.pages);
  const int64_t head = (int64_t)(p.ok ? id : 0) * a.c.Hkv + hk, at = head * (kKvBlock * D);
  const int kq = lane >> 4;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u)
      p.k[i][u] = *reinterpret_cast<const u32x4*>(a.c.k + at + (2 * i + (kq >> 1)) * 1024 + token16(u, lane & 15) * 32 + (kq & 1) * 16);
#pragma unroll
  for (int e = 0; e < D / 16; ++e) p.v[e] = *reinterpret_cast<const uint2*>(a.c.v + at + (16 * e + (lane & 15)) * 32 + 8 * kq);
  p.ke = a.c.k_scale[head];
  p.ve = a.c.v_scale[head];
}

// 16 rows: Q's operand, O^T (channel 16 e + 4 kq + i of row lane & 15), maximum and this lane's sum.
template <typename T, int D>
struct Rows16 {
  f16x8 q[D / 64][2][kTerms<T>];  // channels 64 i + 16 kq + 8 m on
  f32x4 o[D / 16];
  float m, l;
  int exponent, limit;
};

template <typename T, int D>
__device__ __forceinline__ void load_rows16(const KvAttnParams& a, const Work& w, int row, int lane, Rows16<T, D>& st) {
  const int r = row + (lane & 15), kq = lane >> 4;
  const bool on = r < w.rows;
  const T* p = nullptr;
  if (on) p = reinterpret_cast<const T*>(a.q + (int64_t)(w.q.row0 + r / a.G) * a.ldq) + (int64_t)(w.hk * a.G + r % a.G) * D + 16 * kq;
  float x[D / 64][16];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[i][j] = 0.f;
    if (on) {
      if (a.aligned_q) load_row<T, 16, true>(p + 64 * i, x[i]);
      else load_row<T, 16, false>(p + 64 * i, x[i]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7fffffffu);
  }
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  const float factor = q_factor(a, m, st.exponent);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[i][j] *= factor;
    split8<kTerms<T>>(x[i], st.q[i][0]);
    split8<kTerms<T>>(x[i] + 8, st.q[i][1]);
  }
  st.limit = w.q.len;
  if (a.causal) st.limit = min(st.limit, w.q.first + r / a.G + 1);
  st.m = kMaxSeed;
  st.l = 0.f;
#pragma unroll
  for (int e = 0; e < D / 16; ++e) st.o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// One page (number blk) for N groups of 16 rows; mv as in State.
template <typename T, int D, int N, bool MASKED>
__device__ __forceinline__ void step16(const Page16<D>& pg, Rows16<T, D> (&st)[N], int& mv, float scale_log2, int lane, int blk) {
  constexpr int NT = kTerms<T>;
  const int kq = lane >> 4, ke = __builtin_amdgcn_readfirstlane(pg.ke), ve = __builtin_amdgcn_readfirstlane(pg.ve);
  f32x4 s[N][2];
#pragma unroll
  for (int n = 0; n < N; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const u32x4 x = pg.k[i][u];
      const f16x8 k0 = half8(x[0], x[1], 1.f), k1 = half8(x[2], x[3], 1.f);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int t = NT - 1; t >= 0; --t) {
          s[n][u] = mfma16(k0, st[n].q[i][0][t], s[n][u]);
          s[n][u] = mfma16(k1, st[n].q[i][1][t], s[n][u]);
        }
    }
  const bool v_grows = ve > mv;
  const float v_factor = v_grows ? __uint_as_float(kv_pow2_bits(mv - ve)) : 1.f;
  if (v_grows) mv = ve;
  f16x8 p[N][NT];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float f = ldexpf(scale_log2, st[n].exponent + ke - 127);
    float z[8], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = s[n][u][i] * f;
        if constexpr (MASKED) x = blk * kKvBlock + token16(u, 4 * kq + i) < st[n].limit ? x : -INFINITY;
        z[4 * u + i] = x;
        top = max_nan(top, x);
      }
    top = max_over_rows4(top);
    const bool grows = !(top <= st[n].m + kLazy);
    if (__any(grows) || v_grows) {
      const float m = grows ? max_nan(st[n].m, top) : st[n].m;
      const float r = fast_exp2(st[n].m - m);
      st[n].l *= r;
      st[n].m = m;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) st[n].o[e] *= r * v_factor;
    }
    const float base = (float)kPBias - st[n].m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      z[i] = fast_exp2(z[i] + base);
      if constexpr (NT == 2) st[n].l += z[i];
    }
    split8<NT>(z, p[n]);
    if constexpr (NT == 1) {
      const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
      for (int i = 0; i < 8; i += 2) st[n].l = __builtin_amdgcn_fdot2(f16x2{p[n][0][i], p[n][0][i + 1]}, one, st[n].l, false);
    }
  }
  const float vs = __uint_as_float((uint32_t)max(ve - mv + kVBias + 127, 1) << 23);
  bool nan_v = false;
  if constexpr (MASKED) {
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) any |= nan_bytes(pg.v[e].x) | nan_bytes(pg.v[e].y);
    nan_v = __any(any != 0);
  }
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    uint32_t x = pg.v[e].x, y = pg.v[e].y;
    if (MASKED && nan_v) {
      x = without_nan(x);
      y = without_nan(y);
    }
    const f16x8 v = half8(x, y, vs);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int t = NT - 1; t >= 0; --t) st[n].o[e] = mfma16(v, p[n][t], st[n].o[e]);
  }
  if (MASKED && nan_v) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float seen[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) seen[i] = blk * kKvBlock + token16(i >> 2, 4 * kq + (i & 3)) < st[n].limit ? 1.f : 0.f;
      const f16x8 sn = round8(seen);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        const f32x4 hits = mfma16(half8(ones_at_nan(pg.v[e].x), ones_at_nan(pg.v[e].y), 1.f), sn, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int i = 0; i < 4; ++i) st[n].o[e][i] = hits[i] > 0.f ? NAN : st[n].o[e][i];
      }
    }
  }
}

template <typename T, int D, int N, int W>
__global__ __launch_bounds__(64 * W, D <= 128 ? 2 : 1) void kv_attn_split_kernel(KvAttnParams a) {
  // The merge goes CH channels at a time through two buffers (one where that is all): as many as leave room for other
  // workgroups (16 at a time: 8.5 us against 7.7 for a call over 200 tokens).
  constexpr int ROWS = 16 * N, CH = 4096 / (W * ROWS) > 64 ? 64 : 4096 / (W * ROWS);
  static_assert(D % CH == 0 && CH % 16 == 0 && ROWS * CH / 4 <= 64 * W, "a thread for four channels of each row");
  __shared__ __attribute__((aligned(16))) float lo[D > CH ? 2 : 1][W][ROWS][CH + 4];
  __shared__ float lm[W][ROWS], ll[W][ROWS];
  __shared__ int lv[W];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Splits first, so that long sequences spread over the XCDs; with several groups of rows, which read the same pages,
  // key heads first and the groups next: where Hkv is a multiple of 8, a head's groups share an XCD's L2.
  int id = blockIdx.x, split = 0, group = 0;
  if (a.groups == 1) {
    split = id % a.splits;
    id /= a.splits;
  }
  const int hk = id % a.c.Hkv;
  id /= a.c.Hkv;
  if (a.groups > 1) {
    group = id % a.groups;
    id /= a.groups;
    split = id % a.splits;
    id /= a.splits;
  }
  const int b = id;
  // With all pages of a sequence in one workgroup, the first ones' ids need not wait for its length.
  const int32_t* table = a.s.block_table + (int64_t)b * a.s.max_blocks;
  int32_t first = -1, next = -1;  // ids of the wave's first page, and of the page after the one being loaded
  if (a.splits == 1) {
    if (wave < a.s.max_blocks) first = table[wave];
    if (wave + W < a.s.max_blocks) next = table[wave + W];
  }
  Work w;
  if (!kv_work(a, ROWS, group, hk, b, &w)) return;
  const int lo_block = (int)((int64_t)w.blocks * split / a.splits), hi_block = (int)((int64_t)w.blocks * (split + 1) / a.splits);

  int blk = lo_block + wave;
  constexpr bool AHEAD = D <= 128;  // registers for two pages
  Page16<D> pg[AHEAD ? 2 : 1];
  if (a.splits > 1) {
    first = blk < hi_block ? table[blk] : -1;
    next = blk + W < hi_block ? table[blk + W] : -1;
  }
  load_page<D>(a, w.hk, first, lane, pg[0]);
  Rows16<T, D> st[N];
#pragma unroll
  for (int n = 0; n < N; ++n) load_rows16<T, D>(a, w, w.row0 + 16 * n, lane, st[n]);
  int mv = 0;
  const float scale = fabsf(a.scale_log2);
  // Pages that every row attends to as a whole, two at a time, each loaded while the one before is worked on; what is
  // left (a whole one perhaps, then the cut ones) follows with the masks.
  int least = w.q.len;
  if (a.causal) least = max(0, min(least, w.q.first + w.row0 / a.G + 1));
  const int whole = min(hi_block, least / kKvBlock);
  const auto load_next = [&](int at, Page16<D>& p) {
    const int32_t now = next;
    next = at + W < hi_block ? table[at + W] : -1;
    load_page<D>(a, w.hk, now, lane, p);
  };
  if constexpr (!AHEAD) {
    for (; blk < whole; blk += W) {
      if (pg[0].ok) step16<T, D, N, false>(pg[0], st, mv, scale, lane, blk);
      load_next(blk + W, pg[0]);
    }
    for (; blk < hi_block; blk += W) {
      if (pg[0].ok) step16<T, D, N, true>(pg[0], st, mv, scale, lane, blk);
      load_next(blk + W, pg[0]);
    }
  }
  if constexpr (AHEAD) {
    while (blk + W < whole) {
      load_next(blk + W, pg[1]);
      if (pg[0].ok) step16<T, D, N, false>(pg[0], st, mv, scale, lane, blk);
      blk += W;
      load_next(blk + W, pg[0]);  // past the last page: page 0, not used
      if (pg[1].ok) step16<T, D, N, false>(pg[1], st, mv, scale, lane, blk);
      blk += W;
    }
    while (blk < hi_block) {
      const bool more = blk + W < hi_block;
      if (more) load_next(blk + W, pg[1]);
      if (pg[0].ok) step16<T, D, N, true>(pg[0], st, mv, scale, lane, blk);
      pg[0] = pg[1];
      blk += W;
    }
  }

  // ---- merge of the waves
  const int r = lane & 15, kq = lane >> 4;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float l = sum_over_rows4(st[n].l);
    if (lane < 16) {
      lm[wave][16 * n + lane] = st[n].m;
      ll[wave][16 * n + lane] = l;
    }
  }
  if (lane == 0) lv[wave] = mv;
  __syncthreads();
  float* rec = a.splits > 1 ? a.ws + record_at(a, w.b, w.hk, group, split, ROWS, D) : nullptr;
  int top_v = lv[0];
#pragma unroll
  for (int i = 1; i < W; ++i) top_v = max(top_v, lv[i]);
  float mine[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float m = lm[0][16 * n + r], total = 0.f;
#pragma unroll
    for (int i = 1; i < W; ++i) m = max_nan(m, lm[i][16 * n + r]);
#pragma unroll
    for (int i = 0; i < W; ++i) total += ll[i][16 * n + r] * fast_exp2(lm[i][16 * n + r] - m);
    // rows that attended to nothing: sum 0, and zeros
    mine[n] = total == 0.f ? 0.f : fast_exp2(st[n].m - m) * __uint_as_float(kv_pow2_bits(mv - top_v)) / total;
    if (rec && wave == 0 && lane < 16) rec[ROWS * D + 16 * n + lane] = total == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(total);
  }
#pragma unroll
  for (int c = 0; c < D / CH; ++c) {
    float(&part)[W][ROWS][CH + 4] = lo[c % (D > CH ? 2 : 1)];
#pragma unroll
    for (int e = 0; e < CH / 16; ++e)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ldexpf(st[n].o[c * (CH / 16) + e][i] * mine[n], top_v - 127 - kVBias);
        *reinterpret_cast<f32x4*>(&part[wave][16 * n + r][16 * e + 4 * kq]) = x;
      }
    __syncthreads();
    // thread: row, four channels; the other buffer takes the next channels meanwhile
    const int rr = threadIdx.x / (CH / 4), d = threadIdx.x % (CH / 4) * 4;
    if (rr < ROWS) {
      f32x4 x = *reinterpret_cast<const f32x4*>(&part[0][rr][d]);
#pragma unroll
      for (int i = 1; i < W; ++i) x += *reinterpret_cast<const f32x4*>(&part[i][rr][d]);
      if (rec) *reinterpret_cast<f32x4*>(rec + rr * D + CH * c + d) = x;
      else if (w.row0 + rr < w.rows) store_o4<T, D>(a, w, w.row0 + rr, CH * c + d, x);
    }
  }
}

// ---- many rows: 128 of them to a workgroup, 32 to a wave, and the pages of all through LDS. A page is loaded to
// registers while the one before is worked on and then left in one of two LDS buffers, so it costs one barrier (two pages
// to a barrier: 4 x 1024 rows over 4096 keys at 16 heads x 256 365 us against 334, 4 x 2048 at 32 x 128 573 against 567);
// in LDS a lane's 16 bytes of a KiB lie at 16 * lane, which neither its write nor its read conflicts on. Four waves to a
// SIMD for 16-bit rows of 64 channels (4 x 2048 rows over 4096 keys at 16 heads 178 us, in three 200), three for float32
// ones, two and one for the wider heads: what the registers allow without spills.
constexpr int kRowWaves = 4;

// Workgroup number `rank` of one key head when those of all sequences (at most 64, one to a lane) stand in the order
// of their pages, most first: its sequence and its place there; false past the last. Ragged prompts end with their
// short workgroups instead of whichever come last: 8 of up to 2048 rows over 4096 keys, 32 heads on 8 x 128, 527 us ->
// 332, 64 of up to 512 over 2048 459 -> 412, 16 of up to 1024 at 8 x 64 in float32 42.5 -> 39; 64 x 256 rows over
// contexts of up to 512 keys, 9 x 64 in float32, 49 -> 43.5. Equal sequences pay for it: 4 x 2048 rows over 4096 keys
// 437 -> 441, and short ones: 64 prompts of up to 512 tokens at 8 x 64 29 -> 30.3. So from 16 pages on, 32 where causal.
// Pages grow with the place in a sequence, so the workgroups of a sequence with at least c pages are its last ones,
// and their number follows from c alone; the c of this rank is searched for by halves.
__device__ __forceinline__ bool longest_first(const KvAttnParams& a, int rank, int* b, int* place) {
  constexpr int ROWS = kRows * kRowWaves;
  const int lane = threadIdx.x & 63, lanes = min(a.s.B, 64);
  KvSeq q{0, 0, 0, 0};
  if (lane < lanes) q = kv_seq(a.s, lane);
  const int all = (q.rows * a.G + ROWS - 1) / ROWS;
  const auto sum = [](int x) {  // over the rows of 16 lanes by rotations (0x120 + n: by n lanes), then of the four rows
    x += __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);
    return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48);
  };
  const auto at_least = [&](int c) {  // of this lane's workgroups
    const int keys = kKvBlock * (c - 1);  // with more of them: those from token t on
    if (c == 0) return all;
    if (q.len <= keys) return 0;
    const int t = a.causal ? keys - q.first : 0;
    return t >= q.rows ? 0 : t <= 0 ? all : all - t * a.G / ROWS;
  };
  if (rank >= sum(all)) return false;
  int c = 0, end = a.s.max_blocks + 1;  // sum(at_least(c)) > rank >= sum(at_least(end))
  if (a.len_blocks + 1 < end && sum(at_least(a.len_blocks + 1)) <= rank) end = a.len_blocks + 1;
  while (end - c > 1) {
    const int mid = (c + end) / 2;
    if (sum(at_least(mid)) > rank) c = mid;
    else end = mid;
  }
  const int more = at_least(c + 1), mine = at_least(c) - more;  // with more than c pages; with c
  int before = mine;  // those of the lanes before, then without this one's
  for (int m = 1; m < lanes; m <<= 1) {
    const int x = __shfl_up(before, m);
    if (lane >= m) before += x;
  }
  before -= mine;
  const int here = rank - sum(more) - before;  // within this lane's, if it is one of them
  const uint64_t found = __ballot(here >= 0 && here < mine);
  const int from = __builtin_ctzll(found);
  *b = from;
  *place = __builtin_amdgcn_readlane(all - more - 1 - here, from);
  return true;
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kRowWaves, D <= 64 ? (sizeof(T) == 2 ? 4 : 3) : D <= 128 ? 2 : 1) void kv_attn_rows_kernel(KvAttnParams a) {
  constexpr int C = D / 32, ITEMS = 2 * C, MINE = ITEMS / kRowWaves;  // KiB of a page, and a wave's
  static_assert(ITEMS % kRowWaves == 0, "whole KiB per wave");
  constexpr int BYTES = 2 * ITEMS * 1024 > kRowWaves * kRowsLds ? 2 * ITEMS * 1024 : kRowWaves * kRowsLds;
  __shared__ __attribute__((aligned(16))) char shared[BYTES];  // the pages; before and after them, the waves' rows
  u32x4(&tiles)[2][ITEMS][64] = *reinterpret_cast<u32x4(*)[2][ITEMS][64]>(shared);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int hk = id % a.c.Hkv;
  id /= a.c.Hkv;
  int b = id % a.s.B, block4 = (a.groups + kRowWaves - 1) / kRowWaves - 1 - id / a.s.B;  // of a sequence's rows, the last first
  if (a.ordered && !longest_first(a, id, &b, &block4)) return;
  Work all, w;
  if (!kv_work(a, kRows, block4 * kRowWaves, hk, b, &all)) return;
  w = all;
  // pages of the workgroup: those of its last rows
  {
    const int last = min(block4 * kRowWaves + kRowWaves, (all.rows + kRows - 1) / kRows) - 1;
    kv_work(a, kRows, last, all.hk, all.b, &all);
  }
  const bool on = kv_work(a, kRows, block4 * kRowWaves + wave, w.hk, w.b, &w);  // waves past the last rows only load
  const int lo_block = (int)((int64_t)all.blocks * split / a.splits), hi_block = (int)((int64_t)all.blocks * (split + 1) / a.splits);

  std::conditional_t<kCodes<T>, QCodes<T, D>, QTile<T, D>> q;
  State<D> st;
  char* mine = shared + wave * kRowsLds;
  if (on) load_q<T, D>(a, w, lane, q, mine);
#pragma unroll
  for (int c = 0; c < C; ++c) st.o[c] = zero16();
  st.m = kMaxSeed;
  st.l = 0.f;
  st.mv = 0;
  const int row = w.row0 + (lane & 31);
  int limit = w.q.len;
  if (a.causal) limit = min(limit, w.q.first + row / a.G + 1);

  const int32_t* table = a.s.block_table + (int64_t)w.b * a.s.max_blocks;
  const int place = (lane & 31) * 32 + (lane >> 5) * 16;
  u32x4 part[MINE];
  int page, ke, ve;  // of the page being loaded; one that holds nothing: -1
  int32_t id_next;   // of the page after that: a page's loads wait for its id, so it comes a page earlier
  const auto look = [&](int blk) { id_next = blk < hi_block ? table[blk] : -1; };
  const auto fetch = [&](int blk) {
    page = kv_page_ok(id_next, a.c.pages) ? id_next : -1;
    const int64_t at = (int64_t)max(page, 0) * a.c.Hkv + w.hk;
    ke = a.c.k_scale[at];
    ve = a.c.v_scale[at];
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int item = wave + kRowWaves * j, c = item % C;
      const bool is_v = item / C & 1;  // (as a comparison of item with C it compiles to 395 us for 335 at 4 x 1024 rows, 16 heads x 256)
      const uint8_t* base = (is_v ? a.c.v : a.c.k) + kv_tile(max(page, 0), a.c.Hkv, w.hk, D);
      part[j] = *reinterpret_cast<const u32x4*>(base + c * 1024 + place);
    }
    look(blk + 1);
  };
  const auto leave = [&](int buf) {
#pragma unroll
    for (int j = 0; j < MINE; ++j) tiles[buf][wave + kRowWaves * j][lane] = part[j];
  };

  if (lo_block < hi_block) {
    look(lo_block);
    fetch(lo_block);
    __syncthreads();  // every wave has its rows
    leave(0);
  }
  // Pages that every row of the workgroup attends to as a whole, then the others.
  const float scale = fabsf(a.scale_log2);
  int buf = 0;
  const auto steps = [&](int begin, int end, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    for (int blk = begin; blk < end; ++blk, buf ^= 1) {
      const int now = page, kn = ke, vn = ve;
      __syncthreads();
      const bool more = blk + 1 < hi_block;
      if (more) fetch(blk + 1);
      if (on && now >= 0 && !(MASKED && blk >= w.blocks)) {
        const auto k = [&](int c) { return tiles[buf][c][lane]; };
        const auto v = [&](int c) { return tiles[buf][C + c][lane]; };
        const int kk = __builtin_amdgcn_readfirstlane(kn), vv = __builtin_amdgcn_readfirstlane(vn);
        step<T, D, MASKED>(q, st, k, v, kk, vv, scale, lane, limit - blk * kKvBlock);
      }
      if (more) leave(buf ^ 1);
    }
  };
  int least = w.q.len;  // keys that the workgroup's first row attends to
  if (a.causal) least = max(0, min(least, w.q.first + block4 * kRowWaves * kRows / a.G + 1));
  const int whole = max(lo_block, min(hi_block, least / kKvBlock));
  steps(lo_block, whole, std::false_type{});
  steps(whole, hi_block, std::true_type{});
  __syncthreads();  // the last page is done with
  if (!on) return;

  const float total = sum_with_partner(st.l);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int half = lane >> 5;
  float* rec = nullptr;  // narrower heads come here only with more workgroups than their keys would be split for
  if constexpr (D == 256) rec = a.splits > 1 ? a.ws + record_at(a, w.b, w.hk, w.row0 / kRows, split, kRows, D) : nullptr;
  if (rec && half == 0) rec[(int64_t)kRows * D + lane] = total == 0.f ? -INFINITY : st.m + __builtin_amdgcn_logf(total);
  const int64_t at = row_place(a, w, row, a.ldo, D * (int)sizeof(T));
  // Through LDS, as Q came: E elements of a row in a lane, 16 bytes of a record or an output row.
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = ldexpf(st.o[c][4 * g + i] * inv, st.mv - 127 - kVBias);
      *reinterpret_cast<f32x4*>(mine + (lane & 31) * 144 + (8 * g + 4 * half) * 4) = x;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (rec) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int id = 64 * i + lane;
        *reinterpret_cast<f32x4*>(rec + (int64_t)(id / 8) * D + 32 * c + id % 8 * 4) = *reinterpret_cast<const f32x4*>(mine + id / 8 * 144 + id % 8 * 16);
      }
    } else {
      constexpr int E = 16 / (int)sizeof(T), PARTS = 32 / E;
#pragma unroll
      for (int i = 0; i < PARTS / 2; ++i) {
        const int id = 64 * i + lane;
        float x[E];
        load_row<float, E, true>(reinterpret_cast<const float*>(mine + id / PARTS * 144) + id % PARTS * E, x);
        const int64_t to = of_lane(at, id / PARTS);
        T* p = reinterpret_cast<T*>(a.o + to) + 32 * c + id % PARTS * E;
        if (to >= 0) {
          if (a.aligned_o) store_row<T, E, true>(p, x);
          else store_row<T, E, false>(p, x);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// The records of a row's splits into the row, a workgroup for each row: the weights of its splits in LDS, then D/4
// threads to a record and 1024 / D records at a time, joined through LDS. Latency: 3.9 us of 11 for 32 rows x 4 splits.
constexpr int kMaxSplits = 512;

template <typename T, int D>
__global__ __launch_bounds__(256) void kv_attn_merge_kernel(KvAttnParams a, int group_rows, int rows) {
  constexpr int W = D / 4, SIDE = 256 / W;
  __shared__ float weight[kMaxSplits];
  __shared__ float wave_m[4], wave_l[4];
  __shared__ __attribute__((aligned(16))) f32x4 parts[SIDE][W];
  int id = blockIdx.x;
  const int r = id % rows;
  id /= rows;
  const int group = id % a.groups;
  const int bh = id / a.groups;
  Work w;
  if (!kv_work(a, group_rows, group, bh % a.c.Hkv, bh / a.c.Hkv, &w)) return;
  if (w.row0 + r >= w.rows) return;
  const float* rec = a.ws + record_at(a, bh / a.c.Hkv, bh % a.c.Hkv, group, 0, group_rows, D);
  const int64_t next = record_floats(group_rows, D);
  const int tid = threadIdx.x, lane = tid & 63;
  const float* sums = rec + (int64_t)group_rows * D + r;
  float m = kMaxSeed;
  for (int s = tid; s < a.splits; s += 256) m = max_nan(m, weight[s] = sums[s * next]);
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) m = max_nan(m, __shfl_xor(m, i));
  if (lane == 0) wave_m[tid >> 6] = m;
  __syncthreads();
  m = max_nan(max_nan(wave_m[0], wave_m[1]), max_nan(wave_m[2], wave_m[3]));
  float l = 0.f;
  for (int s = tid; s < a.splits; s += 256) l += weight[s] = fast_exp2(weight[s] - m);
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) l += __shfl_xor(l, i);
  if (lane == 0) wave_l[tid >> 6] = l;
  __syncthreads();
  l = wave_l[0] + wave_l[1] + wave_l[2] + wave_l[3];
  const int side = tid / W, d = tid % W * 4;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = side; s < a.splits; s += SIDE) x += *reinterpret_cast<const f32x4*>(rec + s * next + (int64_t)r * D + d) * weight[s];
  parts[side][d / 4] = x;
  __syncthreads();
  if (side > 0) return;
#pragma unroll
  for (int i = 1; i < SIDE; ++i) x += parts[i][d / 4];
  store_o4<T, D>(a, w, w.row0 + r, d, x * (l == 0.f ? 0.f : 1.f / l));
}

struct KvAttnPlan {
  int waves;                       // of a workgroup
  int group_rows, groups, splits;  // of a row group; row groups of a sequence and key head; workgroups that share their keys
  bool many;                       // the kernel of many rows
  bool ordered;                    // its workgroups by their pages
  int64_t blocks;                  // pages of the longest sequence, as the caller has it
  int64_t workgroups, ws_bytes;
};

KvAttnPlan kv_attn_plan(const sa_kv_attn_args* a) {
  KvAttnPlan p;
  const int G = a->H / a->cache.Hkv;
  const int64_t rows = (int64_t)a->seqs.max_rows * G;
  const int64_t heads = (int64_t)a->seqs.B * a->cache.Hkv;
  // The kernel of many rows where it has two workgroups for each CU (one and a half of 16-bit rows of 128 channels), from
  // 128 rows on: a lone workgroup waits for each page in turn. In it / in groups of 32: one prompt of 1000 tokens over 1000
  // keys at 32 heads on 8 x 64 60 us / 17, on 8 x 128 64 / 29; 4 of 300 over 8000 (320 workgroups) at 8 x 64 200 / 126, on
  // 8 x 128 247 / 198, one of 2000 (504) on 8 x 64 183 / 175, on 8 x 128 249 / 281, in float32 439 / 411; 32 of 64 over
  // 1000 (512) on 8 x 128 52 / 87, 32 of 32 (rows of 128) 76 / 49. At 256 channels, whose groups are of 16 rows, from 64
  // rows on: 32 of 24 tokens over 1000 keys 103 / 122, of 16 89 / 86.
  const int64_t full = a->cache.D == 128 && a->dtype != SA_DT_F32 ? kCUs * 3 / 2 : 2 * kCUs;
  p.many = a->cache.D == 256 ? rows > 64 : rows > 128 && heads * ((rows + 127) / 128) > full;
  // Groups of 16 rows while a workgroup for each fits the CUs: 4 sequences of 12 rows x 8 heads over 2000 keys at 8 x 64
  // in float32 12.0 us, in groups of 32 17.8; with more, 32 of 16 rows over 1000 keys (128) 43.5 / 28.6.
  const bool narrow = a->cache.D == 256 || rows <= 16 || heads * ((rows + 15) / 16) <= kCUs;
  p.group_rows = p.many ? kRows : narrow ? 16 : 32;
  p.groups = (int)((rows + p.group_rows - 1) / p.group_rows);
  const int64_t base = heads * (p.many ? (p.groups + kRowWaves - 1) / kRowWaves : p.groups);
  const int64_t cap = (int64_t)a->seqs.max_blocks * kKvBlock;
  const int64_t len = a->max_len > 0 && a->max_len < cap ? a->max_len : cap;
  const int64_t blocks = (len + kKvBlock - 1) / kKvBlock;
  // Few rows and more than eight pages: eight waves to a workgroup instead of four and splits of eight pages (which cost
  // the second launch):
  // - with a workgroup for at least a quarter of the CUs; their keys are split from 64 pages on. 16 sequences of 2000
  //   tokens at 8 key heads x 128 18.4 us (20.9), 32 of them 31.5 (35.5), 16 of 500 11.4 (13.0); at 8 x 256 in float16 32
  //   of 777 27.2 (33.6), 16 of 2000 41.0 (38.0), 32 of 2000 56.5 (60.7);
  // - with fewer, while eight waves have few pages each: one sequence of 777 tokens at 8 x 128 9.6 us (11.2), 1000 10.2
  //   (11.2), 1400 11.3 (11.1), 2000 13.5 (11.4); at 8 x 64 in float32, 1400 8.9 (10.4), 2000 10.6 (10.7); at 8 x 256
  //   777 14.8 (13.2).
  // Eight pages or fewer are done in four waves, without a split: 16 of 200 tokens at 8 x 256 11.2 us (12.7).
  const bool wide = base >= kCUs / 4 || (a->cache.D <= 128 && blocks * a->cache.D <= 4096);
  p.waves = !p.many && base <= kCUs && blocks > 8 && wide ? 8 : 4;
  // Splits fill two workgroups of four waves to a CU or one of eight, and no more (one too many is a round of its own:
  // 20 sequences of 8000 tokens at 8 x 128 82 us for 65); few rows of one group in four waves are quicker past that.
  // Many rows pay for splits with a record of each (1200 rows x 8 heads over 1000 keys at 64 channels, two splits 28.7
  // us, one 13), worth it only where the last round would be nearly empty: 12 x 80 tokens over 8000 keys at 32 heads on
  // 8 x 256 807 us, in one 986.
  int64_t splits = 1;
  if (p.waves == 4) {
    splits = (2 * kCUs + (p.groups > 1 ? 0 : base - 1)) / base;
    if (p.many && base > kCUs && base <= kCUs + kCUs / 4 && a->cache.D == 256 && blocks >= 128) splits = 2;
    if (splits > (blocks + 7) / 8) splits = (blocks + 7) / 8;
  } else if (blocks > 64) {
    splits = kCUs / base;
    if (splits > (blocks + 31) / 32) splits = (blocks + 31) / 32;
  }
  if (splits < 1) splits = 1;
  p.splits = (int)splits;
  p.blocks = blocks;
  p.ordered = p.many && p.groups > kRowWaves && a->seqs.B > 1 && a->seqs.B <= 64 && blocks >= (a->causal ? 32 : 16);  // longest_first
  p.workgroups = base * splits;
  p.ws_bytes = splits > 1 ? (int64_t)a->seqs.B * a->cache.Hkv * p.groups * splits * record_floats(p.group_rows, a->cache.D) * 4 : 0;
  return p;
}

template <typename T, int D>
hipError_t launch_kv_attn(const KvAttnParams& a, const KvAttnPlan& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.workgroups);
  if (p.many) hipLaunchKernelGGL((kv_attn_rows_kernel<T, D>), grid, dim3(64 * kRowWaves), 0, stream, a);
  else if (p.group_rows == 16 && p.waves == 8) hipLaunchKernelGGL((kv_attn_split_kernel<T, D, 1, 8>), grid, dim3(64 * 8), 0, stream, a);
  else if (p.group_rows == 16) hipLaunchKernelGGL((kv_attn_split_kernel<T, D, 1, 4>), grid, dim3(64 * 4), 0, stream, a);
  else if constexpr (D <= 128) {
    if (p.waves == 8) hipLaunchKernelGGL((kv_attn_split_kernel<T, D, 2, 8>), grid, dim3(64 * 8), 0, stream, a);
    else hipLaunchKernelGGL((kv_attn_split_kernel<T, D, 2, 4>), grid, dim3(64 * 4), 0, stream, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t most = (int64_t)a.s.max_rows * a.G;
  const int rows = (int)(most < p.group_rows ? most : p.group_rows);
  const int64_t merges = (int64_t)a.s.B * a.c.Hkv * p.groups * rows;  // below 2^31: splits > 1 bounds the groups
  hipLaunchKernelGGL((kv_attn_merge_kernel<T, D>), dim3((unsigned)merges), dim3(256), 0, stream, a, p.group_rows, rows);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_kv_attn_t(const KvAttnParams& a, const KvAttnPlan& p, hipStream_t stream) {
  return a.c.D == 64 ? launch_kv_attn<T, 64>(a, p, stream) : a.c.D == 128 ? launch_kv_attn<T, 128>(a, p, stream) : launch_kv_attn<T, 256>(a, p, stream);
}

// Checks; SA_OK with p->s.B == 0 for a call with nothing to do.
int resolve_kv_attn(const sa_kv_attn_args* a, KvAttnParams* p, KvAttnPlan* plan) {
  if (a == nullptr) return fail(SA_ERR_INVALID, "args is NULL");
  if (a->struct_size != sizeof(sa_kv_attn_args))
    return fail(SA_ERR_INVALID, "struct_size %u does not match sizeof(sa_kv_attn_args) = %zu", a->struct_size, sizeof(sa_kv_attn_args));
  int rc = kv_check_dtype(a->dtype);
  if (rc == SA_OK) rc = kv_check_cache(a->cache);
  if (rc == SA_OK) rc = kv_check_seqs(a->seqs);
  if (rc != SA_OK) return rc;
  if (a->H <= 0 || a->H % a->cache.Hkv) return fail(SA_ERR_INVALID, "H = %d must be a positive multiple of Hkv = %d", a->H, a->cache.Hkv);
  if (a->H > (1 << 16)) return fail(SA_ERR_UNSUPPORTED, "%d heads (at most 65536)", a->H);
  if (a->causal != 0 && a->causal != 1) return fail(SA_ERR_INVALID, "causal must be 0 or 1 (got %d)", a->causal);
  if (!isfinite(a->scale * kLog2e)) return fail(SA_ERR_INVALID, "scale must be finite, and of magnitude below 2^127");
  if (a->max_len < 0) return fail(SA_ERR_INVALID, "max_len must be >= 0");
  *p = KvAttnParams{};
  *plan = KvAttnPlan{4, kRows, 0, 1, false, false, 0, 0, 0};
  if (kv_nothing(a->seqs)) return SA_OK;
  const int size = kv_type_bytes(a->dtype);
  const int64_t width = (int64_t)a->H * a->cache.D;
  KvRows q, o;
  rc = kv_rows(a->q, a->q_off, a->ldq, width, a->seqs.T, size, "q", &q);
  if (rc == SA_OK) rc = kv_rows(a->o, a->o_off, a->ldo, width, a->seqs.T, size, "o", &o);
  if (rc != SA_OK) return rc;
  if (kv_overlap(q, o)) return fail(SA_ERR_ALIAS, "o overlaps q");
  if (kv_overlap_cache(o, a->cache)) return fail(SA_ERR_ALIAS, "o overlaps the cache");
  if (kv_overlap_seqs(o, a->seqs)) return fail(SA_ERR_ALIAS, "o overlaps the sequences' arrays");
  const int G = a->H / a->cache.Hkv;
  if ((int64_t)a->seqs.max_rows * G > (1 << 30)) return fail(SA_ERR_UNSUPPORTED, "%d rows of %d heads in one sequence", a->seqs.max_rows, G);
  *plan = kv_attn_plan(a);
  if (plan->workgroups > kKvMaxThreads / (64 * plan->waves))
    return fail(SA_ERR_UNSUPPORTED, "%lld workgroups: more than one launch takes", (long long)plan->workgroups);
  p->c = a->cache;
  p->s = a->seqs;
  p->q = q.lo;
  p->o = const_cast<char*>(o.lo);
  p->ldq = q.ld;
  p->ldo = o.ld;
  p->scale_log2 = a->scale * kLog2e;
  p->H = a->H;
  p->G = G;
  p->causal = a->causal;
  p->groups = plan->groups;
  p->splits = plan->splits;
  p->ordered = plan->ordered;
  p->len_blocks = (int)plan->blocks;
  p->aligned_q = (((uintptr_t)q.lo | (uintptr_t)q.ld) & 15) == 0;
  p->aligned_o = (((uintptr_t)o.lo | (uintptr_t)o.ld) & 15) == 0;
  return SA_OK;
}

}  // namespace

}  // namespace sa

using sa::fail;
using sa::ok;

extern "C" {

int sa_kv_attention(const sa_kv_attn_args* args, void* stream) {
  sa::KvAttnParams p;
  sa::KvAttnPlan plan;
  const int rc = sa::resolve_kv_attn(args, &p, &plan);
  if (rc != SA_OK) return rc;
  if (plan.workgroups == 0) return ok();
  if (plan.ws_bytes > 0) {
    if (!args->workspace || args->workspace_bytes < plan.ws_bytes)
      return fail(SA_ERR_INVALID, "this call needs a device workspace of %lld bytes (sa_kv_attention_workspace_bytes)", (long long)plan.ws_bytes);
    if ((uintptr_t)args->workspace & 15) return fail(SA_ERR_INVALID, "workspace must be 16-byte aligned");
    const sa::KvRows q = {p.q, p.ldq, (int64_t)p.H * p.c.D * sa::kv_type_bytes(args->dtype), p.s.T};
    const sa::KvRows o = {p.o, p.ldo, q.width, p.s.T}, ws = {(const char*)args->workspace, plan.ws_bytes, plan.ws_bytes, 1};
    if (sa::kv_overlap(q, ws.lo, plan.ws_bytes) || sa::kv_overlap(o, ws.lo, plan.ws_bytes) || sa::kv_overlap_cache(ws, p.c) || sa::kv_overlap_seqs(ws, p.s))
      return fail(SA_ERR_ALIAS, "the workspace overlaps q, o, the cache or the sequences' arrays");
    p.ws = (float*)args->workspace;
  }
  const hipError_t e = args->dtype == SA_DT_F32   ? sa::launch_kv_attn_t<float>(p, plan, (hipStream_t)stream)
                       : args->dtype == SA_DT_F16 ? sa::launch_kv_attn_t<_Float16>(p, plan, (hipStream_t)stream)
                                                  : sa::launch_kv_attn_t<__bf16>(p, plan, (hipStream_t)stream);
  return e == hipSuccess ? ok() : sa::hip_fail(e, "kv_attention");
}

int64_t sa_kv_attention_workspace_bytes(const sa_kv_attn_args* args) {
  sa::KvAttnParams p;
  sa::KvAttnPlan plan;
  const int rc = sa::resolve_kv_attn(args, &p, &plan);
  if (rc != SA_OK) return rc;
  ok();
  return plan.ws_bytes;
}

int sa_kv_attention_shape(const sa_kv_attn_args* args, int32_t* rows, int32_t* splits) {
  if (!rows || !splits) return fail(SA_ERR_INVALID, "rows and splits must be non-NULL");
  sa::KvAttnParams p;
  sa::KvAttnPlan plan;
  const int rc = sa::resolve_kv_attn(args, &p, &plan);
  if (rc != SA_OK) return rc;
  *rows = plan.many ? sa::kRows * sa::kRowWaves : plan.group_rows;
  *splits = plan.splits;
  return ok();
}

}  // extern "C"
