// Norms of queries and keys for each head, with the position rotation in the same pass (include/supra_kv.h).
//
// One wave takes one token and a run of its heads; the D elements of a head lie across a power-of-two group of
// lanes, so a wave works on several heads at once and the sum of squares is a few exchanges inside the group. A
// lane's chunk is P pairs of the rotation: P elements and their P partners (or 2P neighbours), both in its own
// registers, so the rotation exchanges nothing; the elements past rotary_dim are cut into pairs the same way and
// turned by no angle. A lane keeps the same pairs for every head, so a token's sines and cosines are formed once, one
// pair to a lane, and handed out through LDS (every lane forming its own: 48.5 us against 39.1 at 8191 tokens x 40 heads
// x 128 in bfloat16, 14.8 against 7.5 at 777 x 9 x 256). The next step's rows are loaded before this one's are worked on.
//
// Angles: position * inv_freq in float64, in turns, less the nearest whole turn (exact); what is left is at most half a
// turn and goes on in float32, so position 2^20 is as good as position 1. sincospif of twice that.
//
// Bound: HBM traffic, every element read and written once: 168 MB in 39.6 us, 4.2 TB/s (8191 x 40 x 128, bfloat16);
// 151 MB in 33.3 us, 4.5 TB/s (16384 x 18 x 64, float32), where a copy of 4 GiB reaches 4.6. Down to some hundred
// tokens, latency: 6.6 us at 777 x 9 x 256, 4.2 us of kernel at one token.

#include <hip/hip_runtime.h>

#include <math.h>

#include "common.h"
#include "kv_check.h"
#include "row_types.h"

namespace sa {

namespace {

constexpr int kRopeWaves = 4;
constexpr int kRopeMaxPairs = 256;  // D is at most 512
constexpr int kRopePairs = 4;       // pairs of a lane: 16 bytes of float32, 8 of a 16-bit type (8 pairs, 16 bytes of one, take
                                    // twice the registers: 16384 x 18 heads x 64 in bfloat16 23.5 us against 20.7)

struct RopeParams {
  const char* q;  // rows, offsets included; strides in bytes
  const char* k;
  char* qo;
  char* ko;
  int64_t ldq, ldk, ldqo, ldko;
  const float* wq;
  const float* wk;
  const double* inv_freq;
  const int32_t* positions;
  int T, H, heads;  // heads: query and key heads together
  int D, half;      // half: rotary_dim / 2 pairs are rotated
  int group;        // lanes of a head (a power of two)
  int shift;        // its log2
  int per_wave;     // heads of a wave's run, a multiple of 64 / group
  int runs;         // runs of a token
  int norm;
  float eps, inv_d, rope_scale;
};

// P pairs of chunk c: the places of their first elements (contiguous from a) and of their partners (HALF: contiguous
// from b; NEAR: interleaved with them from a on).
template <typename T, int P, bool NEAR, bool ALIGNED>
__device__ __forceinline__ void load_pairs(const T* x, int a, int b, float (&u)[P], float (&v)[P]) {
  if constexpr (NEAR) {
    float z[2 * P];
    load_row<T, 2 * P, ALIGNED>(x + a, z);
#pragma unroll
    for (int i = 0; i < P; ++i) u[i] = z[2 * i], v[i] = z[2 * i + 1];
  } else {
    load_row<T, P, ALIGNED>(x + a, u);
    load_row<T, P, ALIGNED>(x + b, v);
  }
}

template <typename T, int P, bool NEAR, bool ALIGNED>
__device__ __forceinline__ void store_pairs(T* x, int a, int b, const float (&u)[P], const float (&v)[P]) {
  if constexpr (NEAR) {
    float z[2 * P];
#pragma unroll
    for (int i = 0; i < P; ++i) z[2 * i] = u[i], z[2 * i + 1] = v[i];
    store_row<T, 2 * P, ALIGNED>(x + a, z);
  } else {
    store_row<T, P, ALIGNED>(x + a, u);
    store_row<T, P, ALIGNED>(x + b, v);
  }
}

// N chunks of P pairs per lane. ALIGNED: P pairs are whole vector accesses (P > 1) on both sides of the rotated part.
template <typename T, int P, int N, bool NEAR>
__global__ __launch_bounds__(64 * kRopeWaves) void qk_rope_kernel(RopeParams a) {
  constexpr bool ALIGNED = P > 1;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * kRopeWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = item / a.runs;
  if (t >= a.T) return;
  const int run = (int)(item % a.runs);
  const int first = run * a.per_wave, last = min(first + a.per_wave, a.heads);

  const int in_group = lane & (a.group - 1), sub = lane >> a.shift, step = 64 >> a.shift;
  int pa[N], pb[N];
  bool has[N], turned[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int p = (n * a.group + in_group) * P;  // the chunk's first pair
    has[n] = 2 * p < a.D;
    turned[n] = p < a.half;
    if constexpr (NEAR) {
      pa[n] = 2 * p;
      pb[n] = 2 * p + 1;
    } else {
      pa[n] = turned[n] ? p : p + a.half;
      pb[n] = pa[n] + (turned[n] ? a.half : a.D / 2 - a.half);
    }
  }

  // The rows of one step: a head for each group of lanes. Groups past the last head run along (the exchanges need
  // all lanes) with zeros.
  const auto load = [&](int h0, float (&u)[N][P], float (&v)[N][P]) {
    const int h = h0 + sub;
    const bool is_k = h >= a.H;
    const T* x = reinterpret_cast<const T*>((is_k ? a.k : a.q) + t * (is_k ? a.ldk : a.ldq)) + (int64_t)(is_k ? h - a.H : h) * a.D;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int i = 0; i < P; ++i) u[n][i] = v[n][i] = 0.f;
      if (h < last && has[n]) load_pairs<T, P, NEAR, ALIGNED>(x, pa[n], pb[n], u[n], v[n]);
    }
  };
  float u[N][P], v[N][P];
  load(first, u, v);

  // Weights of the lane's places, and the token's sines and cosines: lane i forms those of pairs i, i + 64, ... once
  // for the wave, and each lane takes its own from LDS (the wave's own part of it: its accesses are in order).
  float wq[N][2][P], wk[N][2][P], cs[N][P], sn[N][P];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int i = 0; i < P; ++i) wq[n][0][i] = wq[n][1][i] = wk[n][0][i] = wk[n][1][i] = 1.f;
    if (has[n] && a.wq) load_pairs<float, P, NEAR, ALIGNED>(a.wq, pa[n], pb[n], wq[n][0], wq[n][1]);
    if (has[n] && a.wk) load_pairs<float, P, NEAR, ALIGNED>(a.wk, pa[n], pb[n], wk[n][0], wk[n][1]);
  }
  __shared__ __attribute__((aligned(16))) float turns[kRopeWaves][2][kRopeMaxPairs];
  float(&mine)[2][kRopeMaxPairs] = turns[threadIdx.x >> 6];
  if (a.half > 0) {
    const double at = (double)a.positions[t];
    for (int p = lane; p < a.half; p += 64) {
      double f = at * a.inv_freq[p] * 0.15915494309189533576888;  // turns: 1 / (2 pi)
      f -= rint(f);
      float s, c;
      sincospif(2.f * (float)f, &s, &c);
      mine[0][p] = c * a.rope_scale;
      mine[1][p] = s * a.rope_scale;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int p = (n * a.group + in_group) * P;
#pragma unroll
    for (int i = 0; i < P; ++i) cs[n][i] = 1.f, sn[n][i] = 0.f;
    if (turned[n]) {
      load_row<float, P, ALIGNED>(&mine[0][p], cs[n]);
      load_row<float, P, ALIGNED>(&mine[1][p], sn[n]);
    }
  }

  for (int h0 = first; h0 < last; h0 += step) {
    float nu[N][P], nv[N][P];
    load(h0 + step, nu, nv);  // past the last head: zeros
    const int h = h0 + sub;
    const bool is_k = h >= a.H;
    T* y = reinterpret_cast<T*>((is_k ? a.ko : a.qo) + t * (is_k ? a.ldko : a.ldqo)) + (int64_t)(is_k ? h - a.H : h) * a.D;
    float r = 1.f;
    if (a.norm == SA_NORM_RMS) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < P; ++i) ss = fmaf(u[n][i], u[n][i], fmaf(v[n][i], v[n][i], ss));
      for (int m = 1; m < a.group; m <<= 1) ss += __shfl_xor(ss, m);
      r = 1.f / sqrtf(ss * a.inv_d + a.eps);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float p = u[n][i] * r * (is_k ? wk[n][0][i] : wq[n][0][i]), q = v[n][i] * r * (is_k ? wk[n][1][i] : wq[n][1][i]);
        u[n][i] = p * cs[n][i] - q * sn[n][i];
        v[n][i] = q * cs[n][i] + p * sn[n][i];
      }
      if (h < last && has[n]) store_pairs<T, P, NEAR, ALIGNED>(y, pa[n], pb[n], u[n], v[n]);
#pragma unroll
      for (int i = 0; i < P; ++i) u[n][i] = nu[n][i], v[n][i] = nv[n][i];
    }
  }
}

template <typename T, bool NEAR>
hipError_t launch_rope(const RopeParams& a, bool vec, unsigned grid, hipStream_t stream) {
  if (vec) hipLaunchKernelGGL((qk_rope_kernel<T, kRopePairs, 1, NEAR>), dim3(grid), dim3(64 * kRopeWaves), 0, stream, a);
  else hipLaunchKernelGGL((qk_rope_kernel<T, 1, 4, NEAR>), dim3(grid), dim3(64 * kRopeWaves), 0, stream, a);
  return hipGetLastError();
}

int resolve_rope(const sa_qk_rope_args* a, RopeParams* p, bool* vector) {
  if (a == nullptr) return fail(SA_ERR_INVALID, "args is NULL");
  if (a->struct_size != sizeof(sa_qk_rope_args))
    return fail(SA_ERR_INVALID, "struct_size %u does not match sizeof(sa_qk_rope_args) = %zu", a->struct_size, sizeof(sa_qk_rope_args));
  int rc = kv_check_dtype(a->dtype);
  if (rc != SA_OK) return rc;
  if (a->T < 0 || a->H < 0 || a->Hkv < 0) return fail(SA_ERR_INVALID, "T, H and Hkv must be >= 0 (got %d, %d, %d)", a->T, a->H, a->Hkv);
  if (a->D <= 0 || a->D % 2) return fail(SA_ERR_INVALID, "head dim %d must be even and positive", a->D);
  if (a->D > 512) return fail(SA_ERR_UNSUPPORTED, "head dim %d exceeds the supported maximum 512", a->D);
  if (a->H > (1 << 16) || a->Hkv > (1 << 16)) return fail(SA_ERR_UNSUPPORTED, "%d and %d heads (at most 65536)", a->H, a->Hkv);
  if (a->rotary_dim < 0 || a->rotary_dim > a->D || a->rotary_dim % 2)
    return fail(SA_ERR_INVALID, "rotary_dim %d must be even and within the head dim %d", a->rotary_dim, a->D);
  if (a->pairs != SA_ROPE_HALF && a->pairs != SA_ROPE_NEAR) return fail(SA_ERR_INVALID, "unknown pairs %d", a->pairs);
  if (a->norm != SA_NORM_NONE && a->norm != SA_NORM_RMS) return fail(SA_ERR_INVALID, "unknown norm %d", a->norm);
  if (!isfinite(a->eps) || a->eps < 0) return fail(SA_ERR_INVALID, "eps must be finite and >= 0");
  if (!isfinite(a->rope_scale)) return fail(SA_ERR_INVALID, "rope_scale must be finite");
  *p = RopeParams{};
  p->T = a->T;
  p->H = a->H;
  p->heads = a->H + a->Hkv;
  if (a->T == 0 || p->heads == 0) return SA_OK;
  if (a->rotary_dim > 0 && (!a->inv_freq || !a->positions)) return fail(SA_ERR_INVALID, "inv_freq and positions must be non-NULL device pointers");
  if ((uintptr_t)a->inv_freq & 7 || (uintptr_t)a->positions & 3 || ((uintptr_t)a->q_weight | (uintptr_t)a->k_weight) & 3)
    return fail(SA_ERR_INVALID, "inv_freq, positions and the weights must be aligned to their types");
  const int size = kv_type_bytes(a->dtype);
  KvRows q{}, k{}, qo{}, ko{};
  const int64_t nq = (int64_t)a->H * a->D, nk = (int64_t)a->Hkv * a->D;
  if (a->H > 0) {
    rc = kv_rows(a->q, a->q_off, a->ldq, nq, a->T, size, "q", &q);
    if (rc == SA_OK) rc = kv_rows(a->q_out, a->qo_off, a->ldqo, nq, a->T, size, "q_out", &qo);
  }
  if (rc == SA_OK && a->Hkv > 0) {
    rc = kv_rows(a->k, a->k_off, a->ldk, nk, a->T, size, "k", &k);
    if (rc == SA_OK) rc = kv_rows(a->k_out, a->ko_off, a->ldko, nk, a->T, size, "k_out", &ko);
  }
  if (rc != SA_OK) return rc;
  const auto same = [](const KvRows& x, const KvRows& y) { return x.lo == y.lo && x.ld == y.ld; };
  for (const KvRows* o : {&qo, &ko}) {
    if (o->width == 0) continue;
    const bool for_q = o == &qo;
    if ((q.width && !(for_q && same(q, *o)) && kv_overlap(q, *o)) || (k.width && !(!for_q && same(k, *o)) && kv_overlap(k, *o)))
      return fail(SA_ERR_ALIAS, "%s overlaps q or k (an output may only be its own input, rows and all)", for_q ? "q_out" : "k_out");
    if (kv_overlap(*o, a->q_weight, a->q_weight ? 4LL * a->D : 0) || kv_overlap(*o, a->k_weight, a->k_weight ? 4LL * a->D : 0) ||
        (a->rotary_dim > 0 && (kv_overlap(*o, a->inv_freq, 4LL * a->rotary_dim) || kv_overlap(*o, a->positions, 4LL * a->T))))
      return fail(SA_ERR_ALIAS, "%s overlaps the weights, inv_freq or positions", for_q ? "q_out" : "k_out");
  }
  if (qo.width && ko.width && kv_overlap(qo, ko)) return fail(SA_ERR_ALIAS, "q_out overlaps k_out");
  p->q = q.lo;
  p->k = k.lo;
  p->qo = const_cast<char*>(qo.lo);
  p->ko = const_cast<char*>(ko.lo);
  p->ldq = q.ld;
  p->ldk = k.ld;
  p->ldqo = qo.ld;
  p->ldko = ko.ld;
  p->wq = a->q_weight;
  p->wk = a->k_weight;
  p->inv_freq = a->inv_freq;
  p->positions = a->positions;
  p->D = a->D;
  p->half = a->rotary_dim / 2;
  p->norm = a->norm;
  p->eps = a->eps;
  p->inv_d = 1.f / (float)a->D;
  p->rope_scale = a->rope_scale == 0.f ? 1.f : a->rope_scale;

  // Vector accesses where every chunk of pairs stays on one side of the rotated part and every access is aligned;
  // single elements otherwise (any even D, any alignment).
  const uintptr_t bits = (uintptr_t)q.lo | (uintptr_t)k.lo | (uintptr_t)qo.lo | (uintptr_t)ko.lo | (uintptr_t)q.ld | (uintptr_t)k.ld |
                         (uintptr_t)qo.ld | (uintptr_t)ko.ld | (uintptr_t)a->q_weight | (uintptr_t)a->k_weight;
  const bool vec = bits % 16 == 0 && p->half % kRopePairs == 0 && a->D % (2 * kRopePairs) == 0;
  const int chunks = a->D / 2 / (vec ? kRopePairs : 1), most = vec ? 1 : 4;  // of a head, and of a lane
  p->group = 1;
  while (p->group * most < chunks || (!vec && p->group < 64 && p->group < chunks)) {
    p->group *= 2;
    p->shift++;
  }
  *vector = vec;
  return SA_OK;
}

}  // namespace

}  // namespace sa

using sa::fail;
using sa::ok;

extern "C" int sa_qk_norm_rope(const sa_qk_rope_args* args, void* stream) {
  sa::RopeParams p;
  bool vec = false;
  const int rc = sa::resolve_rope(args, &p, &vec);
  if (rc != SA_OK) return rc;
  if (p.T == 0 || p.heads == 0) return ok();
  // A wave takes all heads of a token (its angles and weights are fetched once) unless the tokens alone leave the
  // device short of waves: then a token's heads are cut into runs, down to one step of the wave. Enough is one
  // wave per SIMD and then some for 16-bit rows (8191 tokens x 40 heads x 128, whole tokens / runs of one step:
  // 39.6 / 42.5 us), many more for float32 rows, whose steps move twice the bytes (73.5 / 63.6 us).
  const int step = 64 / p.group, steps = (p.heads + step - 1) / step;
  const int64_t want = args->dtype == SA_DT_F32 ? 40000 : 4096;
  int64_t runs = p.T >= want ? 1 : (want + p.T - 1) / p.T;
  if (runs > steps) runs = steps;
  const int per = (int)((steps + runs - 1) / runs);
  p.per_wave = per * step;
  p.runs = (steps + per - 1) / per;
  const int64_t groups = ((int64_t)p.T * p.runs + sa::kRopeWaves - 1) / sa::kRopeWaves;
  if (groups > sa::kKvMaxThreads / (64 * sa::kRopeWaves)) return fail(SA_ERR_UNSUPPORTED, "T = %d tokens: more than one launch takes", p.T);
  const bool near = args->pairs == SA_ROPE_NEAR;
  const hipStream_t s = (hipStream_t)stream;
  const unsigned grid = (unsigned)groups;
  hipError_t e;
  if (args->dtype == SA_DT_F32) e = near ? sa::launch_rope<float, true>(p, vec, grid, s) : sa::launch_rope<float, false>(p, vec, grid, s);
  else if (args->dtype == SA_DT_F16) e = near ? sa::launch_rope<_Float16, true>(p, vec, grid, s) : sa::launch_rope<_Float16, false>(p, vec, grid, s);
  else e = near ? sa::launch_rope<__bf16, true>(p, vec, grid, s) : sa::launch_rope<__bf16, false>(p, vec, grid, s);
  return e == hipSuccess ? ok() : sa::hip_fail(e, "qk_norm_rope");
}
