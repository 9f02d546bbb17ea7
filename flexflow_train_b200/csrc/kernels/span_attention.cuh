// span_attention.cuh -- what the forward and the backward kernels of attention over spans of keys share.
//
//   x[q, k] = f(scale * Q_q . K_k) - slope_h * |q - k|,   f(u) = cap * tanh(u / cap) with a cap, u without
//   P[q, .] = softmax of x[q, k] over low_q <= k <= high_q,   O = P V
//
// per batch row and query head h, with the keys and values of head h / (H / KH).  A query whose span is empty sees nothing: O = 0, and it
// gives no gradient.  All matrices are bf16 [batch * S, ld] with head h in the D columns from h * D on; D is a multiple of 8 up to 128
// (TMA fills a tile's columns beyond D with zeros); statistics and accumulators are fp32, scores are kept in units of log 2.
//
// Rows of Q, K, V and dO that no pair of the tile at hand needs may hold anything: a masked score is replaced, not multiplied, and rows
// that nothing in the block sees are cleared in shared memory before a product sums over them (0 * NaN is not 0).
#pragma once
#include "tcgen05.cuh"

struct FfkSpanAttnDesc {
  int B, H, KH, S, D;
  float scale, cap;
  const void *spans;               // [B, S] pairs of int32: first and last visible key
  const float *slopes;             // [H] or null
  const void *Q; long long ldq;
  const void *K; long long ldk;
  const void *V; long long ldv;
  void *O; long long ldo;
  float *lse;                      // [B, H, S], base 2; 0 for a query that sees nothing
  const void *dO; long long lddo;
  void *dQ; long long lddq;
  void *dK; long long lddk;
  void *dV; long long lddv;
  float *scratch;                  // backward: delta [B, H, S], then one summary of four ints per batch row and 128 queries
};

namespace {

constexpr float SA_LOG2E = 1.4426950408889634f;
constexpr int SA_T = 128;          // rows of a tile of queries or keys
constexpr int SA_PANEL = SA_T * 128;   // bytes of 64 columns of a tile

struct SpanArgs {
  int B, H, KH, S, D;
  const int2 *spans;
  const float *slopes;
  float mul;                       // to the log-2 domain: scale * log2(e), or with a cap scale / cap
  float cap2;                      // cap * log2(e)
  float scale;
  bf16 *O;
  long long ldo;
  float *lse;
  const float *delta;
  const int4 *summary;
  bf16 *dQ, *dK, *dV;
  long long lddq, lddk, lddv;
  int tiles;                       // forward: 128-query tiles of a CTA, 1 or 2
  int *err;
};

__host__ __device__ constexpr uint32_t sa_idesc(int M, int N, int a_mn, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// ---- pairs of fp32: one instruction of the FMA pipe for two elements
typedef unsigned long long pair32;
__device__ __forceinline__ pair32 pair_of(float a, float b) {
  pair32 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void pair_to(pair32 p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ pair32 pair_fma(pair32 a, pair32 b, pair32 c) {
  pair32 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair32 pair_mul(pair32 a, pair32 b) {
  pair32 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair32 pair_add(pair32 a, pair32 b) {
  pair32 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair32 pair_get(const uint32_t *r) { return pair_of(__uint_as_float(r[0]), __uint_as_float(r[1])); }
__device__ __forceinline__ void pair_set(uint32_t *r, pair32 p) {
  float a, b;
  pair_to(p, a, b);
  r[0] = __float_as_uint(a);
  r[1] = __float_as_uint(b);
}

// 2^x, the special-function unit's (results below the normal range are 0)
__device__ __forceinline__ float sa_exp2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x of a pair on the FMA pipe: x = n + f, |f| <= 1/2, a polynomial of degree 4 for 2^f (least squares on the relative error, 2.6e-6),
// n added to the exponent.  x below -126 counts as -126.
__device__ __forceinline__ void sa_exp2_pair(float &a, float &b) {
  const float magic = 12582912.f;                        // 1.5 * 2^23: the sum holds round(x) in its low bits
  const pair32 x = pair_of(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const pair32 t = pair_add(x, pair_of(magic, magic));
  const pair32 n = pair_add(t, pair_of(-magic, -magic));
  const pair32 f = pair_fma(n, pair_of(-1.f, -1.f), x);
  pair32 p = pair_fma(f, pair_of(0.009570101276f, 0.009570101276f), pair_of(0.05591785908f, 0.05591785908f));
  p = pair_fma(p, f, pair_of(0.2402474433f, 0.2402474433f));
  p = pair_fma(p, f, pair_of(0.6931217909f, 0.6931217909f));
  p = pair_fma(p, f, pair_of(0.9999992847f, 0.9999992847f));
  float p0, p1, t0, t1;
  pair_to(p, p0, p1);
  pair_to(t, t0, t1);
  a = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  b = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

// tanh(z) for |z| <= SA_TANH_SMALL: z times a polynomial of degree 4 in z^2 (least squares on the relative error, 1.1e-7)
constexpr float SA_TANH_SMALL = 0.625f;
__device__ __forceinline__ pair32 sa_tanh_small(pair32 z) {
  const pair32 w = pair_mul(z, z);
  pair32 p = pair_fma(w, pair_of(0.01505094394f, 0.01505094394f), pair_of(-0.05182186514f, -0.05182186514f));
  p = pair_fma(p, w, pair_of(0.1330452561f, 0.1330452561f));
  p = pair_fma(p, w, pair_of(-0.3333195448f, -0.3333195448f));
  p = pair_fma(p, w, pair_of(0.9999998808f, 0.9999998808f));
  return pair_mul(z, p);
}
// tanh(z) = 1 - 2 / (1 + e^2z), everywhere, to 2e-7 of 1
__device__ __forceinline__ float sa_tanh_any(float z) { return 1.f - __fdividef(2.f, 1.f + sa_exp2(fminf(z * (2.f * SA_LOG2E), 120.f))); }

// `x` (N raw scores of one row) becomes tanh(mul * x) with a cap; the score in log-2 units is x times what is returned.  All lanes of the
// warp; a row that does not `count` has no say in the way tanh is taken.
template <int N, bool CAP>
__device__ __forceinline__ float sa_capped(uint32_t (&x)[N], const SpanArgs &p, bool count) {
  if constexpr (!CAP) return p.mul;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(x[i])), fabsf(__uint_as_float(x[i + 1]))));
  if (__all_sync(0xffffffffu, !count || most * p.mul <= SA_TANH_SMALL)) {
    const pair32 a = pair_of(p.mul, p.mul);
#pragma unroll
    for (int i = 0; i < N; i += 2) pair_set(&x[i], sa_tanh_small(pair_mul(pair_get(&x[i]), a)));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __float_as_uint(sa_tanh_any(__uint_as_float(x[i]) * p.mul));
  }
  return p.cap2;
}

__device__ __forceinline__ void sa_warp_arrive(uint64_t *bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
__device__ __forceinline__ bool sa_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, const SpanArgs &p, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err, code));
}

// span of query q of batch row b, cut to the sequence; empty: first > last
__device__ __forceinline__ int2 sa_span(const SpanArgs &p, int b, int q) {
  int2 s = p.spans[(long long)b * p.S + q];
  s.x = max(s.x, 0);
  s.y = min(s.y, p.S - 1);
  return s;
}

// Clears the rows of a tile (panels of 64 columns, 128 bytes a row) whose bit in `keep` (four words, 32 rows each) is not set.  One warp.
__device__ __forceinline__ void sa_clear_rows(uint8_t *tile, int panels, const uint32_t (&keep)[4], int lane) {
  const int per_row = panels * 8;                        // 16-byte pieces
  const int at_once = 32 / per_row;                      // rows a warp clears at once
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t drop = ~keep[w];
    while (drop) {
      // the rows of the `at_once` lowest bits
      int mine = -1;
      for (int i = 0; i < at_once && drop; ++i) {
        const int r = __ffs(drop) - 1;
        drop &= drop - 1;
        if (lane / per_row == i) mine = w * 32 + r;
      }
      if (mine >= 0) {
        const int c = lane % per_row;
        *reinterpret_cast<uint4 *>(tile + (c >> 3) * SA_PANEL + mine * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
    }
  }
}

// bits [from, to] of the four words of a 128-row mask
__device__ __forceinline__ void sa_add_bits(uint32_t (&m)[4], int from, int to) {
  from = max(from, 0);
  to = min(to, 127);
  if (from > to) return;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int a = max(from - 32 * w, 0), b = min(to - 32 * w, 31);
    if (a <= b) m[w] |= (0xffffffffu >> (31 - b)) & (0xffffffffu << a);
  }
}

// 4-D map {column, row, head, batch row} of a [B * S, ld] matrix; box = 64 columns x 128 rows
inline int sa_head_map(CUtensorMap *map, const void *ptr, int D, int S, long long ld, int heads, int B) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return -1;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)heads, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)(ld * 2), (cuuint64_t)(D * 2), (cuuint64_t)((long long)S * ld * 2)};
  cuuint32_t box[4] = {64, SA_T, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void *)ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

inline bool sa_aligned(const void *p, long long ld) { return (((uintptr_t)p) & 15) == 0 && (ld * 2) % 16 == 0; }
inline bool sa_shape_ok(const FfkSpanAttnDesc *d) {
  return d->KH > 0 && d->H % d->KH == 0 && d->D >= 8 && d->D <= 128 && d->D % 8 == 0 && d->scale > 0.f && d->cap >= 0.f && (((uintptr_t)d->spans) & 7) == 0;
}
inline void sa_args(const FfkSpanAttnDesc *d, SpanArgs &a, int *err) {
  a.B = d->B; a.H = d->H; a.KH = d->KH; a.S = d->S; a.D = d->D;
  a.spans = (const int2 *)d->spans; a.slopes = d->slopes;
  a.mul = d->cap > 0.f ? d->scale / d->cap : d->scale * SA_LOG2E;
  a.cap2 = d->cap * SA_LOG2E;
  a.scale = d->scale;
  a.O = (bf16 *)d->O; a.ldo = d->ldo; a.lse = d->lse;
  a.err = err;
}

}  // namespace

// one error word for both directions (span_attention_fwd.cu)
extern "C" __attribute__((visibility("hidden"))) int *ffk_span_attention_err();
