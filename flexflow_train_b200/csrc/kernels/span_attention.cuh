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

static_assert(sizeof(FfkSpanAttnDesc) == 192, "packed field by field by the Python side");

namespace {

constexpr float SA_LOG2E = 1.4426950408889634f;
constexpr float SA_MOST_CAP = 1073741824.f;   // cap / scale at most: beyond, the cap is no cap
constexpr int SA_T = 128;          // rows of a tile of queries or keys
constexpr int SA_PANEL = SA_T * 128;   // bytes of 64 columns of a tile

struct SpanArgs {
  int B, H, KH, S, D;
  const int2 *spans;
  const float *slopes;
  float scale, factor;             // factor = scale * log2(e): a score in log-2 units is factor * y, see sa_cap
  float to_z, from_z;              // with a cap: scale / cap and cap / scale
  float lim2, lim4;                // |raw score| up to which tanh is a polynomial of degree 2 or 4 in its square; negative: nowhere
  float t2[3], t4[5];              // the polynomials' coefficients, for raw scores
  float *lse;
  const float *delta;
  const int4 *summary;
  bf16 *dK, *dV;
  long long lddk, lddv;
  const bf16 *Q, *K, *V;           // of the kernels that do not go through tensor maps
  long long ldq, ldk, ldv;
  int wide;                        // results' rows lie on 32-byte boundaries
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
// tanh(z) = 1 - 2 / (1 + e^2z), everywhere, to 2e-7 of 1
__device__ __forceinline__ float sa_tanh_any(float z) { return 1.f - __fdividef(2.f, 1.f + sa_exp2(fminf(z * (2.f * SA_LOG2E), 120.f))); }

// Scores of N columns of a row, in place: raw products s become y with  (score in log-2 units) = factor * y:
//   y = s, with a cap tanh(a s) / a (a = scale / cap), with a bias less slope / scale * |distance|.
// The special-function unit has its hands full with the exponentials (8 cycles a warp instruction), and the FMA pipe takes one element a
// cycle whether packed or not, so tanh(a s) / a = s T((a s)^2) is a polynomial as short as the warp's largest |s| allows: degree 2 up to |a s| =
// 1/4, degree 4 up to 5/8 (least squares on the relative error: 4e-7 and 1.1e-7), the exponential form beyond.
//
// sa_cap: false where a score of the warp is beyond the polynomials (x is unchanged: sa_cap_any).  `count`: whether the row has a say in
// that (one that sees nothing may hold anything).  All lanes of the warp.
template <int N>
__device__ __forceinline__ bool sa_cap(uint32_t (&x)[N], const SpanArgs &p, bool count) {
  float most[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    most[0] = fmaxf(most[0], fabsf(__uint_as_float(x[i])));
    most[1] = fmaxf(most[1], fabsf(__uint_as_float(x[i + 1])));
  }
  const float top = fmaxf(most[0], most[1]);
  if (__all_sync(0xffffffffu, !count || top <= p.lim2)) {
    const pair32 c0 = pair_of(p.t2[0], p.t2[0]), c1 = pair_of(p.t2[1], p.t2[1]), c2 = pair_of(p.t2[2], p.t2[2]);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const pair32 s = pair_get(&x[i]), w = pair_mul(s, s);
      pair_set(&x[i], pair_mul(s, pair_fma(pair_fma(w, c2, c1), w, c0)));
    }
    return true;
  }
  if (__all_sync(0xffffffffu, !count || top <= p.lim4)) {
    const pair32 c0 = pair_of(p.t4[0], p.t4[0]), c1 = pair_of(p.t4[1], p.t4[1]), c2 = pair_of(p.t4[2], p.t4[2]), c3 = pair_of(p.t4[3], p.t4[3]),
                 c4 = pair_of(p.t4[4], p.t4[4]);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const pair32 s = pair_get(&x[i]), w = pair_mul(s, s);
      pair_set(&x[i], pair_mul(s, pair_fma(pair_fma(pair_fma(pair_fma(w, c4, c3), w, c2), w, c1), w, c0)));
    }
    return true;
  }
  return false;
}
__device__ __forceinline__ void sa_cap_any(uint32_t (&x)[32], const SpanArgs &p) {
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(sa_tanh_any(__uint_as_float(x[i]) * p.to_z) * p.from_z);
}
// one score, the same way
__device__ __forceinline__ float sa_cap_one(float s, const SpanArgs &p) {
  const float w = s * s;
  if (fabsf(s) <= p.lim2) return s * fmaf(fmaf(w, p.t2[2], p.t2[1]), w, p.t2[0]);
  if (fabsf(s) <= p.lim4) return s * fmaf(fmaf(fmaf(fmaf(w, p.t4[4], p.t4[3]), w, p.t4[2]), w, p.t4[1]), w, p.t4[0]);
  return sa_tanh_any(s * p.to_z) * p.from_z;
}
// The bias: d0 = position of the first column less the row's (distances are whole numbers: exact), side: -1 / 1 where no column of the warp
// lies right / left of its row, 0 otherwise; slope: the head's, over the scale
template <int N>
__device__ __forceinline__ void sa_bias(uint32_t (&x)[N], float slope, float d0, int side) {
  pair32 d = pair_of(d0, d0 + 1.f);
  const pair32 two = pair_of(2.f, 2.f);
  const float k = side < 0 ? slope : -slope;
  const pair32 kk = pair_of(k, k);
  if (side != 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      pair_set(&x[i], pair_fma(kk, d, pair_get(&x[i])));
      d = pair_add(d, two);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      pair_set(&x[i], pair_fma(kk, d & 0x7fffffff7fffffffull, pair_get(&x[i])));
      d = pair_add(d, two);
    }
  }
}
// The distance bias of successive pairs of columns in log-2 units, added to `to` (backward: the cap's derivative needs the score without it)
struct SaBias {
  pair32 d, k, bits;
  __device__ __forceinline__ SaBias(float slope, float d0, int side) {
    const float kk = side < 0 ? slope : -slope;
    d = pair_of(d0, d0 + 1.f);
    k = pair_of(kk * SA_LOG2E, kk * SA_LOG2E);
    bits = side != 0 ? ~0ull : 0x7fffffff7fffffffull;
  }
  __device__ __forceinline__ pair32 next(pair32 to) {
    const pair32 r = pair_fma(k, d & bits, to);
    d = pair_add(d, pair_of(2.f, 2.f));
    return r;
  }
};
// 32 of a thread's registers
template <int N>
__device__ __forceinline__ uint32_t (&sa_group(uint32_t (&x)[N], int g))[32] { return *reinterpret_cast<uint32_t(*)[32]>(&x[g * 32]); }

// the first load through a tensor map waits for the map itself: asked for ahead
__device__ __forceinline__ void sa_prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory"); }

// 16 columns of a warp's 32 lanes into tensor memory
__device__ __forceinline__ void sa_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
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

// columns before `a` and behind `z` (of 32) become `v`
__device__ __forceinline__ void sa_mask(uint32_t (&x)[32], int a, int z, uint32_t v) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < a || i > z) x[i] = v;
}

// Clears the rows of a tile (panels of 64 columns, 128 bytes a row) whose bit in `keep` (four words, 32 rows each) is not set.  One warp, a
// lane per row; lanes begin at different pieces of their rows, so that four and not 32 of them share a bank.
template <int PANELS>
__device__ __forceinline__ void sa_clear_rows(uint8_t *tile, const uint32_t (&keep)[4], int lane) {
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (!(keep[w] >> lane & 1u)) {
#pragma unroll
      for (int c = 0; c < PANELS * 8; ++c)
        *reinterpret_cast<uint4 *>(tile + (c >> 3) * SA_PANEL + (w * 32 + lane) * 128 + ((c + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
}

// ---- Blocks of a grid taken over by the ones that run.  A CTA of these kernels fills an SM (tensor memory, shared memory), so that the set-up of
// one (barriers, tensor memory, first loads: about 5000 cycles) and the read-out of its results run with the tensor core idle; a CTA here
// is a few tiles long.  So a running CTA asks for the next block that has not been launched, gets its index (or learns that there is none) while
// it works, and goes on with that block, its rings and barriers running through.
__device__ __forceinline__ void sa_ask_next(uint64_t *answer, uint64_t *bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// the answer's block, or -1
__device__ __forceinline__ int sa_next_block(const uint64_t *answer) {
  uint32_t x, got;
  asm volatile(
      "{\n.reg .pred p;\n.reg .b128 c;\nld.shared.b128 c, [%2];\nclusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, c;\n"
      "selp.u32 %1, 1, 0, p;\nmov.u32 %0, 0;\n@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, _, _, _}, c;\n}"
      : "=r"(x), "=r"(got)
      : "r"(smem_u32(answer))
      : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // read before the next answer is written there
  return got ? (int)x : -1;
}

// 32 columns of a row of results, `left` of which exist, as bf16 to global memory: whole sectors where addresses allow it (`wide`)
__device__ __forceinline__ void sa_store_row(bf16 *out, const uint32_t (&o)[32], float f, int left, bool wide) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = pack_bf162(__uint_as_float(o[16 * u + 2 * j]) * f, __uint_as_float(o[16 * u + 2 * j + 1]) * f);
    if (wide && 16 * u + 16 <= left) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + 16 * u), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                   "r"(v[5]), "r"(v[6]), "r"(v[7])
                   : "memory");
    } else {
      if (16 * u < left) *reinterpret_cast<uint4 *>(out + 16 * u) = make_uint4(v[0], v[1], v[2], v[3]);
      if (16 * u + 8 < left) *reinterpret_cast<uint4 *>(out + 16 * u + 8) = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}

// 32 columns of a row (from column `col` on, a multiple of 32) into a tile in shared memory as TMA reads it: 16-byte piece XOR (row % 8)
__device__ __forceinline__ void sa_tile_row(uint8_t *tile, int row, int col, const uint32_t (&o)[32], float f) {
  uint8_t *base = tile + (col >> 6) * SA_PANEL + row * 128;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    *reinterpret_cast<uint4 *>(base + ((((col & 63) >> 3) + u) ^ (row & 7)) * 16) =
        make_uint4(pack_bf162(__uint_as_float(o[8 * u]) * f, __uint_as_float(o[8 * u + 1]) * f),
                   pack_bf162(__uint_as_float(o[8 * u + 2]) * f, __uint_as_float(o[8 * u + 3]) * f),
                   pack_bf162(__uint_as_float(o[8 * u + 4]) * f, __uint_as_float(o[8 * u + 5]) * f),
                   pack_bf162(__uint_as_float(o[8 * u + 6]) * f, __uint_as_float(o[8 * u + 7]) * f));
}
// The tile that `threads` threads (named barrier `id`) have written goes out by TMA, which leaves out what lies behind the sequence or the
// head's columns; thread `first` issues and waits until the tile has been read.
template <int PANELS>
__device__ __forceinline__ void sa_tile_out(uint8_t *tile, const CUtensorMap *map, int row, int head, int b, int id, int threads, bool first) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
  if (first) {
#pragma unroll
    for (int c = 0; c < PANELS; ++c) tma_store_4d(smem_u32(tile + c * SA_PANEL), map, c * 64, row, head, b);
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the tile has been read; it is written by the kernel's end
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

inline bool sa_wide(const void *p, long long ld, int D) { return (((uintptr_t)p) & 31) == 0 && ld % 16 == 0 && D % 16 == 0; }
inline bool sa_aligned(const void *p, long long ld) { return (((uintptr_t)p) & 15) == 0 && (ld * 2) % 16 == 0; }
inline bool sa_shape_ok(const FfkSpanAttnDesc *d) {
  return d->KH > 0 && d->H % d->KH == 0 && d->D >= 8 && d->D <= 128 && d->D % 8 == 0 && d->scale > 0.f && d->cap >= 0.f &&
         d->cap <= d->scale * SA_MOST_CAP && d->S <= (1 << 30) && (((uintptr_t)d->spans) & 7) == 0;
}
inline void sa_args(const FfkSpanAttnDesc *d, SpanArgs &a, int *err) {
  a.B = d->B; a.H = d->H; a.KH = d->KH; a.S = d->S; a.D = d->D;
  a.spans = (const int2 *)d->spans; a.slopes = d->slopes;
  a.scale = d->scale;
  a.factor = d->scale * SA_LOG2E;
  a.lim2 = a.lim4 = -1.f;
  if (d->cap > 0.f) {
    const float z = d->scale / d->cap, w = z * z;
    a.to_z = z;
    a.from_z = d->cap / d->scale;
    const float t2[3] = {0.9999996043f, -0.3332190822f, 0.1284161341f};
    const float t4[5] = {0.9999998808f, -0.3333195448f, 0.1330452561f, -0.05182186514f, 0.01505094394f};
    float f = 1.f;
    for (int i = 0; i < 5; ++i, f *= w) {
      if (i < 3) a.t2[i] = t2[i] * f;
      a.t4[i] = t4[i] * f;
    }
    // z^4 and z^8 have to be within the range of 32 bits (z is at least 2^-30: sa_shape_ok); the exponential form, which is exact to 2e-7 of the
    // cap, is then taken only where a score is a fair part of the cap, or the cap itself is next to nothing
    if (z <= 1024.f) {
      a.lim2 = 0.25f / z;
      if (z >= 1.f / 16384) a.lim4 = 0.625f / z;
    }
  }
  a.lse = d->lse;
  a.err = err;
}

}  // namespace

// one error word for both directions (span_attention_fwd.cu)
extern "C" __attribute__((visibility("hidden"))) int *ffk_span_attention_err();
