// span_attention_bwd.cu -- backward pass of attention over spans of keys (span_attention.cuh has the forward mathematics).
//
//   P = exp(x - lse),  delta_q = dO_q . O_q,  dS = P o (dO V^T - delta) o f'(u),  f'(u) = 1 - tanh(u / cap)^2 (1 without a cap)
//   dV = P^T dO,   dK = scale dS^T Q  (both summed over the query heads of the key head),   dQ = scale dS K
//
// Two kernels recompute the scores, one per accumulator that has to stay on chip: seven products a tile pair where one kernel with all three
// gradients needs five, but no gradient is added to in global memory, so there are no atomics, no 32-bit copy of dQ to clear and convert, and
// the same inputs give the same bits.
//   span_attn_prep_kernel  delta, and what each 128 queries of a batch row see together
//   span_attn_dkv_kernel   CTA = 128 keys of one key head, over the query tiles that see them, of all its query heads.  Scores are produced
//                          transposed (lanes = keys), so that P^T and dS^T, written back to tensor memory as bf16, are the A operands of
//                          dV += P^T dO and dK += dS^T Q where they lie.
//   span_attn_dq_kernel    CTA = 128 queries of one head, over the key tiles that they see; lanes = queries, dS is the A operand of dQ += dS K.
// Roles in both (640 threads): warp 0 TMA producer, warp 1 MMA issuer, warp 2 clears rows that nothing sees, warps 4-19 the element-wise
// part (thread = one row and 32 of the columns); in the first kernel warp 3 brings each query tile's lse, delta and spans.
//
// Rounded to bf16: P and dS (the type that the products take), and dQ, dK, dV once, when they are stored.  delta is taken of the O that
// forward stored, but for queries that see few keys; its rounding and that of dS are what sets the gradients' error (2.5e-3 to 2.7e-3 of their
// norm, 1.7e-3 with both in fp32).
// dS as the sum of two bf16 operands (16 bits of it, 1.8e-3) costs a fourth of the pass: 8 x 2048 packed 510 -> 648 us, 8192 causal 1046 -> 1301.
//
// What bounds it: a tile pair of a long sequence takes about 8300 cycles in both kernels together (8192 causal, cap), of which the seven
// products fill 3584 at the tensor core's rate; the rest is the element-wise chain (tensor-memory load, cap, exponential, mask, dS, store,
// barrier), which the 16 warps that registers allow issue in 41 to 45 % of the cycles.  8192 causal, 16 heads of 128, 4 key heads, cap: 1040 us
// (660 TFLOP/s of the formula's five products), without a cap 860 (800).  8 x 2048 in documents of about 700, 16 heads of 128, cap: delta 45,
// dK / dV 237, dQ 199; without a cap 450 in all.  Tried and slower: dQ as two CTAs an SM with tiles of 64 keys (8192 causal: 1180), or
// going on with the next block of the grid as dK / dV does (its registers do not suffice).
//
// Every wait is bounded (tcgen05.cuh).
#include "span_attention.cuh"

namespace {

constexpr int SAB_THREADS = 640;
constexpr int SAB_WARPS = 16;           // element-wise warps: 32 columns of a tile each

// y[c], y[c + 1] (scores, see sa_cap) become e0, e1 times the cap's derivative 1 - (a y)^2
__device__ __forceinline__ void sa_times_slope(uint32_t (&y)[32], int c, float e0, float e1, float a) {
  const pair32 e = pair_of(e0, e1), z = pair_mul(pair_get(&y[c]), pair_of(a, a));
  pair_set(&y[c], pair_fma(pair_mul(z, pair_of(-e0, -e1)), z, e));
}

// ---------------------------------------------------------------------------------------------- delta and summaries
// The delta of a query that sees few keys is sum_k P dP over them, from Q, K, V and dO, instead of dO . O: its gradients are differences of a few
// products, and the rounding of O to bf16 would be a fair part of them (one head, a sequence of 2 tokens: dQ off by up to its own size; of 3:
// 2.6e-2; of 8: 5e-3, as much as the other roundings).  It costs two dot products a key: backward of 8 x 2048, 16 heads of 128, documents of
// about 700: 524 -> 538 us, of 60: 293 -> 318, of 5: 260 -> 341; with up to 16 keys, a warp per 128 queries: 574, 556, 734 (documents of 12).
constexpr int SAB_FEW = 8;

__device__ __forceinline__ bool sa_few(int2 s) { return s.x <= s.y && s.y - s.x < SAB_FEW; }

__device__ __forceinline__ float sa_dot8(uint4 a, uint4 b) {
  const uint32_t aa[4] = {a.x, a.y, a.z, a.w}, bb[4] = {b.x, b.y, b.z, b.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack_bf162(aa[i]), y = unpack_bf162(bb[i]);
    s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
  }
  return s;
}

// L lanes (the group at `peers` of their warp), 16 bytes of the head from column c on each
template <int L>
__device__ __forceinline__ float span_attn_few(uint4 ov, const SpanArgs &p, unsigned row, int h, int c, int2 span, uint32_t peers) {
  const int b = (int)(row / (unsigned)p.S), q = (int)(row - (unsigned)b * p.S);
  const int kh = h / (p.H / p.KH);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const long long first = (long long)b * p.S;
  const uint4 qv = c < p.D ? *reinterpret_cast<const uint4 *>(p.Q + (first + q) * p.ldq + (long long)h * p.D + c) : zero;
  const float lse = p.lse[((long long)b * p.H + h) * p.S + q], slope = p.slopes ? p.slopes[h] * SA_LOG2E : 0.f;
  const bf16 *K = p.K + (first + span.x) * p.ldk + (long long)kh * p.D + c, *V = p.V + (first + span.x) * p.ldv + (long long)kh * p.D + c;
  float sum = 0.f, total = 0.f;
#pragma unroll 1
  for (int k = span.x; k <= span.y; ++k, K += p.ldk, V += p.ldv) {
    uint4 kv = zero, vv = zero;
    if (c < p.D) {
      kv = *reinterpret_cast<const uint4 *>(K);
      vv = *reinterpret_cast<const uint4 *>(V);
    }
    float x = sa_dot8(qv, kv), dp = sa_dot8(ov, vv);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      x += __shfl_xor_sync(peers, x, o);
      dp += __shfl_xor_sync(peers, dp, o);
    }
    if (p.to_z > 0.f) x = sa_cap_one(x, p);
    const float e = sa_exp2(fmaf(x, p.factor, -slope * (float)abs(q - k)) - lse);
    sum = fmaf(e, dp, sum);
    total += e;
  }
  return total > 0.f ? sum / total : 0.f;
}

// Blocks up to `delta_blocks`: delta, L lanes (16 bytes each) per (row, head).  From there on a warp per 128 queries, their summary: smallest first
// key and largest last key of the queries that see any, largest first key and smallest last key of all (an empty span among them: nothing is
// seen by all).
template <int L>
__global__ void __launch_bounds__(256, 6) span_attn_prep_kernel(const bf16 *dO, long long lddo, const bf16 *O, long long ldo, float *__restrict__ delta,
                                                             int4 *__restrict__ summary, int delta_blocks, const SpanArgs p) {
  pdl_entry();
  const int lane = threadIdx.x & 31;
  if ((int)blockIdx.x < delta_blocks) {
    // (row, head) pairs are counted in 32 bits (checked at the launch): 64-bit divisions had bounded this kernel
    const unsigned at = blockIdx.x * (256 / L) + threadIdx.x / L, total = (unsigned)p.B * p.S * p.H;
    const int c = (threadIdx.x % L) * 8;
    if (at >= total) return;               // whole groups
    const unsigned row32 = at / (unsigned)p.H;
    const int h = (int)(at - row32 * p.H);
    const long long row = row32;
    const uint32_t peers = ((1u << L) - 1u) << (lane / L * L);
    uint4 u = make_uint4(0, 0, 0, 0), w = u;
    if (c < p.D) {
      u = *reinterpret_cast<const uint4 *>(dO + row * lddo + (long long)h * p.D + c);
      w = *reinterpret_cast<const uint4 *>(O + row * ldo + (long long)h * p.D + c);
    }
    int2 span = p.spans[row];
    span.x = max(span.x, 0);
    span.y = min(span.y, p.S - 1);
    float s = sa_dot8(u, w);               // for all: O's load does not wait for the span's
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(peers, s, o);
    if (sa_few(span)) s = span_attn_few<L>(u, p, row32, h, c, span, peers);
    if (c == 0) {
      const unsigned b = row32 / (unsigned)p.S, q = row32 - b * p.S;
      delta[((long long)b * p.H + h) * p.S + q] = s;
    }
    return;
  }
  const int nqt = (p.S + SA_T - 1) / SA_T;
  const long long w = (long long)(blockIdx.x - delta_blocks) * 8 + (threadIdx.x >> 5);
  if (w >= (long long)p.B * nqt) return;
  const int b = (int)(w / nqt), i = (int)(w % nqt);
  int lo = 0x7fffffff, hi = -1, lo_all = -1, hi_all = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int q = i * SA_T + r * 32 + lane;
    if (q < p.S) {
      const int2 s = sa_span(p, b, q);
      if (s.x <= s.y) {
        lo = min(lo, s.x); hi = max(hi, s.y); lo_all = max(lo_all, s.x); hi_all = min(hi_all, s.y);
      } else {
        lo_all = 0x7fffffff;
      }
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo); hi = __reduce_max_sync(0xffffffffu, hi);
  lo_all = __reduce_max_sync(0xffffffffu, lo_all); hi_all = __reduce_min_sync(0xffffffffu, hi_all);
  if (lane == 0) summary[w] = make_int4(lo, hi, lo_all, hi_all);
}

// ---------------------------------------------------------------------------------------------- dK, dV
template <int DT>
struct DkvCfg {
  static constexpr int PANELS = DT / 64;
  static constexpr int TILE = SA_T * DT * 2;
  static constexpr int NQ = 2;                                     // stages of (Q, dO)
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + TILE;
  static constexpr int OFF_Q = OFF_V + TILE;                       // [NQ]
  static constexpr int OFF_DO = OFF_Q + NQ * TILE;                 // [NQ]
  static constexpr int OFF_LSE = OFF_DO + NQ * TILE;               // [NQ][128] float
  static constexpr int OFF_DELTA = OFF_LSE + NQ * 512;             // [NQ][128] float
  static constexpr int OFF_SPAN = OFF_DELTA + NQ * 512;            // [NQ][128] int2
  static constexpr int OFF_GROUP = OFF_SPAN + NQ * 1024;           // [NQ][4] int4: summary of each 32 queries
  static constexpr int OFF_INFO = OFF_GROUP + NQ * 64;             // [2] int4: block, first query tile, query tiles
  static constexpr int OFF_ANSWER = OFF_INFO + 32;                 // 16 bytes
  static constexpr int OFF_BAR = OFF_ANSWER + 16;
  static constexpr int SLACK = 1024;
  static constexpr int SMEM = OFF_BAR + 256 + SLACK;
  static constexpr int TM_S = 0, TM_DP = 128, TM_DK = 256, TM_DV = 256 + DT;
  static_assert(SMEM <= 232448, "tiles exceed the shared memory of a CTA");
};

// A block: 128 keys of one key head.  Block numbers: the first keys, which most queries see under a causal mask, first.
struct DkvBlock {
  int b, kh, k0, k1;
  __device__ __forceinline__ DkvBlock(const SpanArgs &p, int block) {
    const int heads = p.B * p.KH, kb = block / heads, bh = block - kb * heads;
    b = bh / p.KH;
    kh = bh - b * p.KH;
    k0 = kb * SA_T;
    k1 = min(k0 + SA_T, p.S) - 1;
  }
};

template <int DT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(SAB_THREADS, 1)
span_attn_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ CUtensorMap tmDO, const SpanArgs p) {
  using C = DkvCfg<DT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int4 *info = (int4 *)(smem + C::OFF_INFO);
  uint64_t *answer = (uint64_t *)(smem + C::OFF_ANSWER);
  uint64_t *bars = (uint64_t *)(smem + C::OFF_BAR);
  uint64_t *kv_full = bars;
  uint64_t *kv_empty = bars + 1;
  uint64_t *qd_full = bars + 2;       // [2]
  uint64_t *qd_ready = bars + 4;      // [2]
  uint64_t *qd_empty = bars + 6;      // [2]
  uint64_t *st_full = bars + 8;       // [2]
  uint64_t *st_empty = bars + 10;     // [2] SAB_WARPS
  uint64_t *s_full = bars + 12;
  uint64_t *dp_full = bars + 13;
  uint64_t *p_full = bars + 14;       // SAB_WARPS
  uint64_t *ds_full = bars + 15;      // SAB_WARPS
  uint64_t *dkv_full = bars + 16;
  uint64_t *info_full = bars + 17;    // [2]
  uint64_t *info_empty = bars + 19;   // [2] all warps but the first
  uint64_t *answered = bars + 21;
  uint32_t *tmem_slot = (uint32_t *)(bars + 22);
  volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((uintptr_t)(smem - smem_raw) > (uintptr_t)C::SLACK) {
    pdl_entry();
    if (threadIdx.x == 0 && p.err) atomicCAS(p.err, 0, (int)FFK_ERR_BAD_ARG);
    return;
  }
  const int group = p.H / p.KH;
  const int nqt = (p.S + SA_T - 1) / SA_T;

  if (warp == 0) {
    if (lane == 0) {
      sa_prefetch_map(&tmK); sa_prefetch_map(&tmV); sa_prefetch_map(&tmQ); sa_prefetch_map(&tmDO);
      mbar_init(kv_full, 1);
      mbar_init(kv_empty, 1);
      for (int s = 0; s < 2; ++s) {
        mbar_init(&qd_full[s], 1); mbar_init(&qd_ready[s], 1); mbar_init(&qd_empty[s], 1); mbar_init(&st_full[s], 1); mbar_init(&st_empty[s], SAB_WARPS);
        mbar_init(&info_full[s], 1); mbar_init(&info_empty[s], SAB_THREADS / 32 - 1);
      }
      mbar_init(s_full, 1); mbar_init(dp_full, 1); mbar_init(p_full, SAB_WARPS); mbar_init(ds_full, SAB_WARPS); mbar_init(dkv_full, 1);
      mbar_init(answered, 1);
      *abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_entry();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // The next block's (number, first query tile, query tiles), for the warps that follow the first one: false at the end
  int turn = 0;
  auto next_block = [&](int4 &t) -> bool {
    const int s = turn & 1;
    if (!sa_wait(&info_full[s], (uint32_t)(turn >> 1) & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE)) return false;
    t = info[s];
    sa_warp_arrive(&info_empty[s], lane);
    ++turn;
    return t.x >= 0;
  };

  // registers go from the warps that move data to the element-wise ones (128 x 64 + 512 x 104 = 640 x 96)
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer; finds the next block while this one is worked on
    int block = blockIdx.x, steps = 0, blocks = 0;        // steps: of all blocks so far; blocks: those with steps
    bool ok = true;
    while (true) {
      int i0 = 0x7fffffff, i1 = -1;
      const int s = turn & 1;
      if (block >= 0) {                   // first and last query tile that see a key of the block
        const DkvBlock k(p, block);
        const int4 *summary = p.summary + (long long)k.b * nqt;
        for (int i = lane; i < nqt; i += 32) {
          const int4 t = summary[i];
          if (t.x <= k.k1 && t.y >= k.k0) { i0 = min(i0, i); i1 = i; }
        }
        i0 = __reduce_min_sync(0xffffffffu, i0);
        i1 = __reduce_max_sync(0xffffffffu, i1);
      }
      const int ni = i1 < 0 ? 0 : i1 - i0 + 1;
      ok = sa_wait(&info_empty[s], ((uint32_t)(turn >> 1) & 1u) ^ 1u, abort_flag, p, FFK_ERR_TIMEOUT_PRODUCER);
      if (!ok) break;
      if (lane == 0) {
        info[s] = make_int4(block, i0, ni, 0);
        mbar_arrive(&info_full[s]);
      }
      if (block < 0) break;
      if (lane == 0) {
        const DkvBlock k(p, block);
        if (ni > 0) {
          ok = mbar_wait(kv_empty, ((uint32_t)blocks & 1u) ^ 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_PRODUCER);
          if (ok) {
            mbar_expect_tx(kv_full, 2 * C::TILE);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c) {
              tma_load_4d(smem_u32(smem + C::OFF_K + c * SA_PANEL), &tmK, kv_full, c * 64, k.k0, k.kh, k.b);
              tma_load_4d(smem_u32(smem + C::OFF_V + c * SA_PANEL), &tmV, kv_full, c * 64, k.k0, k.kh, k.b);
            }
          }
        }
        int at = steps;
        for (int g = 0; g < group && ok; ++g)
          for (int i = i0; i < i0 + ni; ++i, ++at) {
            ok = mbar_wait(&qd_empty[at & 1], ((uint32_t)(at >> 1) & 1u) ^ 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_PRODUCER);
            if (!ok) break;
            uint64_t *full = &qd_full[at & 1];
            const uint32_t off = (uint32_t)((at & 1) * C::TILE);
            mbar_expect_tx(full, 2 * C::TILE);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c) {
              tma_load_4d(smem_u32(smem + C::OFF_Q + off + c * SA_PANEL), &tmQ, full, c * 64, i * SA_T, k.kh * group + g, k.b);
              tma_load_4d(smem_u32(smem + C::OFF_DO + off + c * SA_PANEL), &tmDO, full, c * 64, i * SA_T, k.kh * group + g, k.b);
            }
          }
        // asked for when the block's last tiles are on their way, two steps before its end: early enough to hide, and late enough that a
        // CTA with a long block does not hold another one back (prompts, heads of 64: 79 us when asked for at the block's start, 58 without)
        sa_ask_next(answer, answered);
      }
      // the answer is waited for even when a wait ran out: a write under way does not outlive its CTA
      ok = sa_wait(answered, (uint32_t)turn & 1u, abort_flag, p, FFK_ERR_TIMEOUT_PRODUCER) && __all_sync(0xffffffffu, ok);
      if (!ok) break;
      steps += ni * group;
      blocks += ni > 0;
      block = sa_next_block(answer);
      ++turn;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer: the whole warp runs, one lane issues
    const bool leader = elect_one();
    const uint64_t dk = make_smem_desc(smem_u32(smem + C::OFF_K), 16, 1024), dv = make_smem_desc(smem_u32(smem + C::OFF_V), 16, 1024);
    const uint64_t q_k0 = make_smem_desc(smem_u32(smem + C::OFF_Q), 16, 1024), q_n0 = make_smem_desc(smem_u32(smem + C::OFF_Q), SA_PANEL, 1024);
    const uint64_t o_k0 = make_smem_desc(smem_u32(smem + C::OFF_DO), 16, 1024), o_n0 = make_smem_desc(smem_u32(smem + C::OFF_DO), SA_PANEL, 1024);
    const int ksteps = (p.D + 15) / 16;
    const uint32_t id_s = sa_idesc(128, SA_T, 0, 0), id_g = sa_idesc(128, ksteps * 16, 0, 1);
    // [keys x queries] = A (keys x D) B (queries x D)^T
    auto issue_t = [&](uint32_t d, uint64_t a, uint64_t bq, uint64_t *bar) {
      if (leader) {
        tc_mma_bf16<false>(d, a, bq, id_s);
#pragma unroll
        for (int s = 1; s < DT / 16; ++s) {
          if (s >= ksteps) break;
          const uint32_t off = (uint32_t)((s >> 2) * SA_PANEL + (s & 3) * 32);
          tc_mma_bf16<true>(d, desc_advance(a, off), desc_advance(bq, off), id_s);
        }
        tc_commit(bar);
      }
      __syncwarp();
    };
    // [keys x D] += A (bf16 in tensor memory: keys x queries, 32 queries in the first 16 of each 32 columns) B (queries x D)
    auto issue_g = [&](uint32_t d, uint32_t a, uint64_t bn, bool first) {
      if (leader) {
        if (first) tc_mma_ts_bf16<false>(d, a, bn, id_g);
        else tc_mma_ts_bf16<true>(d, a, bn, id_g);
#pragma unroll
        for (int s = 1; s < SA_T / 16; ++s)
          tc_mma_ts_bf16<true>(d, a + (uint32_t)((s >> 1) * 32 + (s & 1) * 8), desc_advance(bn, (uint32_t)(s * 2048)), id_g);
      }
      __syncwarp();
    };
    auto wait_qd = [&](int at) -> bool {
      return mbar_wait_warp(&qd_full[at & 1], (uint32_t)(at >> 1) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) &&
             mbar_wait_warp(&qd_ready[at & 1], (uint32_t)(at >> 1) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
    };
    bool ok = true;
    int at = 0, blocks = 0;               // at: steps so far
    int4 t;
    while (ok && next_block(t)) {
      const int n = t.z * group;
      if (n == 0) continue;
      ok = mbar_wait_warp(kv_full, (uint32_t)blocks & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) && wait_qd(at);
      if (!ok) break;
      tc_fence_after();
      const uint32_t off0 = (uint32_t)((at & 1) * C::TILE);
      issue_t(tmem_base + C::TM_S, dk, desc_advance(q_k0, off0), s_full);
      issue_t(tmem_base + C::TM_DP, dv, desc_advance(o_k0, off0), dp_full);
      if (n == 1 && leader) tc_commit(kv_empty);
      for (int it = 0; it < n; ++it, ++at) {
        const uint32_t ph = (uint32_t)at & 1u, off = (uint32_t)((at & 1) * C::TILE), next = (uint32_t)(((at + 1) & 1) * C::TILE);
        // the block before has been read out by the warps that now bring their probabilities
        ok = mbar_wait_warp(p_full, ph, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        issue_g(tmem_base + C::TM_DV, tmem_base + C::TM_S, desc_advance(o_n0, off), it == 0);
        if (it + 1 < n) {                 // the next scores take the columns that P^T is read from: products run in issue order
          ok = wait_qd(at + 1);
          if (!ok) break;
          tc_fence_after();
          issue_t(tmem_base + C::TM_S, dk, desc_advance(q_k0, next), s_full);
        }
        ok = mbar_wait_warp(ds_full, ph, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        issue_g(tmem_base + C::TM_DK, tmem_base + C::TM_DP, desc_advance(q_n0, off), it == 0);
        if (leader) tc_commit(&qd_empty[at & 1]);
        __syncwarp();
        if (it + 1 < n) issue_t(tmem_base + C::TM_DP, dv, desc_advance(o_k0, next), dp_full);
        if (it + 2 == n && leader) tc_commit(kv_empty);
      }
      if (!ok) break;
      if (leader) tc_commit(dkv_full);
      __syncwarp();
      ++blocks;
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ rows of Q and dO that see none of these keys
    bool ok = true;
    int at = 0;
    int4 t;
    while (ok && next_block(t)) {
      const DkvBlock k(p, t.x);
      const int4 *summary = p.summary + (long long)k.b * nqt;
      for (int g = 0; g < group && ok; ++g)
        for (int i = t.y; i < t.y + t.z; ++i, ++at) {
          const int s = at & 1;
          const int4 all = summary[i];
          uint32_t keep[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
          if (all.z > k.k0 || all.w < k.k1) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int q = i * SA_T + w * 32 + lane;
              bool sees = true;                                   // rows behind the sequence arrive as zeros
              if (q < p.S) {
                const int2 sp = sa_span(p, k.b, q);
                sees = sp.x <= sp.y && sp.x <= k.k1 && sp.y >= k.k0;
              }
              keep[w] = __ballot_sync(0xffffffffu, sees);
            }
          }
          ok = sa_wait(&qd_full[s], (uint32_t)(at >> 1) & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
          if (!ok) break;
          if ((keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu) {
            sa_clear_rows<C::PANELS>(smem + C::OFF_Q + s * C::TILE, keep, lane);
            sa_clear_rows<C::PANELS>(smem + C::OFF_DO + s * C::TILE, keep, lane);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          sa_warp_arrive(&qd_ready[s], lane);
        }
    }
  } else {
    // ------------------------------------------------------------------ statistics of each query tile
    bool ok = true;
    int at = 0;
    int4 t;
    while (ok && next_block(t)) {
      const DkvBlock k(p, t.x);
      for (int g = 0; g < group && ok; ++g)
        for (int i = t.y; i < t.y + t.z; ++i, ++at) {
          const int s = at & 1;
          float *lse = (float *)(smem + C::OFF_LSE) + s * SA_T, *dlt = (float *)(smem + C::OFF_DELTA) + s * SA_T;
          int2 *sp = (int2 *)(smem + C::OFF_SPAN) + s * SA_T;
          const long long base = ((long long)k.b * p.H + k.kh * group + g) * p.S;
          float vl[4], vd[4];
          int2 vs[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int q = i * SA_T + r * 32 + lane;
            // a query that sees nothing, or does not exist: probabilities of 0
            vl[r] = INFINITY; vd[r] = 0.f; vs[r] = make_int2(1, 0);
            if (q < p.S) {
              const int2 u = sa_span(p, k.b, q);
              if (u.x <= u.y) {
                vs[r] = u;
                vl[r] = p.lse[base + q];
                vd[r] = p.delta[base + q];
              }
            }
          }
          ok = sa_wait(&st_empty[s], ((uint32_t)(at >> 1) & 1u) ^ 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
          if (!ok) break;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            lse[r * 32 + lane] = vl[r];
            dlt[r * 32 + lane] = vd[r];
            sp[r * 32 + lane] = vs[r];
            // rows behind the sequence count as seeing all: their probabilities are zeros
            const bool there = i * SA_T + r * 32 + lane < p.S, sees = vs[r].x <= vs[r].y;
            int4 u;
            u.x = __reduce_min_sync(0xffffffffu, sees ? vs[r].x : 0x7fffffff);
            u.y = __reduce_max_sync(0xffffffffu, sees ? vs[r].y : -1);
            u.z = __reduce_max_sync(0xffffffffu, sees ? vs[r].x : there ? 0x7fffffff : -1);
            u.w = __reduce_min_sync(0xffffffffu, sees ? vs[r].y : there ? -1 : 0x7fffffff);
            if (lane == 0) *(int4 *)(smem + C::OFF_GROUP + (s * 4 + r) * 16) = u;
          }
          sa_warp_arrive(&st_full[s], lane);
        }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ------------------------------------------------------------------ P^T and dS^T: thread = key x 32 of the tile's queries
    const int quarter = warp & 3, cols = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(cols * 32);
    const pair32 ff = pair_of(p.factor, p.factor);
    bool ok = true;
    int at = 0, blocks = 0;
    int4 t;
    while (ok && next_block(t)) {
      const DkvBlock k(p, t.x);
      const int key = k.k0 + r, kw = k.k0 + quarter * 32;
      for (int g = 0; g < group && ok; ++g) {
        const float slope = BIAS ? p.slopes[k.kh * group + g] : 0.f;
        for (int i = t.y; i < t.y + t.z; ++i, ++at) {
          const int s = at & 1;
          const uint32_t ph = (uint32_t)at & 1u;
          const float *lse = (const float *)(smem + C::OFF_LSE) + s * SA_T + cols * 32, *dlt = (const float *)(smem + C::OFF_DELTA) + s * SA_T + cols * 32;
          const int4 *sp = (const int4 *)(smem + C::OFF_SPAN) + (s * SA_T + cols * 32) / 2;       // two spans each
          ok = sa_wait(&st_full[s], (uint32_t)(at >> 1) & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE) &&
               sa_wait(s_full, ph, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
          if (!ok) break;
          tc_fence_after();
          // how this warp's 32 keys are seen by its 32 queries
          const int4 seen = *(const int4 *)(smem + C::OFF_GROUP + (s * 4 + cols) * 16);
          const bool none = seen.x > kw + 31 || seen.y < kw, masked = seen.z > kw || seen.w < kw + 31;
          uint32_t y[32], pk[16];
          if (none) {
#pragma unroll
            for (int c = 0; c < 16; ++c) pk[c] = 0u;
          } else {
            tmem_ld32(lane_base + C::TM_S, y);
            tmem_ld_wait();
            if (CAP && masked) {              // masked scores do not choose the way tanh is taken
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                const int4 t = sp[c / 2];
                if (key < t.x || key > t.y) y[c] = 0u;
                if (key < t.z || key > t.w) y[c + 1] = 0u;
              }
            }
            if constexpr (CAP) {
              if (!sa_cap(y, p, true)) sa_cap_any(y, p);
            }
            const int qg = i * SA_T + cols * 32;
            SaBias bias(slope, (float)(qg - key), qg >= kw + 31 ? 1 : qg + 31 <= kw ? -1 : 0);
#pragma unroll
            for (int c = 0; c < 32; c += 16) {
              float e[16];
#pragma unroll
              for (int u = 0; u < 16; u += 4) {
                const float4 w = *reinterpret_cast<const float4 *>(lse + c + u);
                pair32 w0 = pair_of(-w.x, -w.y), w1 = pair_of(-w.z, -w.w);
                if constexpr (BIAS) { w0 = bias.next(w0); w1 = bias.next(w1); }
                pair_to(pair_fma(pair_get(&y[c + u]), ff, w0), e[u], e[u + 1]);
                pair_to(pair_fma(pair_get(&y[c + u + 2]), ff, w1), e[u + 2], e[u + 3]);
              }
              if (masked) {
#pragma unroll
                for (int u = 0; u < 16; u += 2) {
                  const int4 t = sp[(c + u) / 2];
                  if (key < t.x || key > t.y) e[u] = -INFINITY;
                  if (key < t.z || key > t.w) e[u + 1] = -INFINITY;
                }
              }
#pragma unroll
              for (int u = 0; u < 16; ++u) e[u] = sa_exp2(e[u]);
#pragma unroll
              for (int u = 0; u < 16; u += 2) pk[(c + u) >> 1] = pack_bf162(e[u], e[u + 1]);
              // what dS needs of P: times the cap's derivative
#pragma unroll
              for (int u = 0; u < 16; u += 2) {
                if constexpr (CAP) {
                  sa_times_slope(y, c + u, e[u], e[u + 1], p.to_z);
                } else {
                  y[c + u] = __float_as_uint(e[u]);
                  y[c + u + 1] = __float_as_uint(e[u + 1]);
                }
              }
            }
          }
          sa_tmem_st16(lane_base + C::TM_S, pk);
          tmem_st_wait();
          tc_fence_before();
          sa_warp_arrive(p_full, lane);
          ok = sa_wait(dp_full, ph, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
          if (!ok) break;
          tc_fence_after();
          if (!none) {
            uint32_t z[32];
            tmem_ld32(lane_base + C::TM_DP, z);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 w = *reinterpret_cast<const float4 *>(dlt + c);
              float v[4];
              pair_to(pair_mul(pair_get(&y[c]), pair_add(pair_get(&z[c]), pair_of(-w.x, -w.y))), v[0], v[1]);
              pair_to(pair_mul(pair_get(&y[c + 2]), pair_add(pair_get(&z[c + 2]), pair_of(-w.z, -w.w))), v[2], v[3]);
              if (masked) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                  if (__uint_as_float(y[c + u]) == 0.f) v[u] = 0.f;                 // whatever dO and delta hold there
              }
              pk[c >> 1] = pack_bf162(v[0], v[1]);
              pk[(c >> 1) + 1] = pack_bf162(v[2], v[3]);
            }
          }
          sa_tmem_st16(lane_base + C::TM_DP, pk);
          tmem_st_wait();
          tc_fence_before();
          sa_warp_arrive(ds_full, lane);
          if (lane == 0) mbar_arrive(&st_empty[s]);
        }
      }
      if (!ok) break;
      // eight warps store dK, eight dV, a thread half of its key's columns
      if (t.z > 0) {
        ok = sa_wait(dkv_full, (uint32_t)blocks & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        ++blocks;
      }
      constexpr int DH = DT / 2;
      const int w = cols & 1, col = (cols >> 1) * DH;
      const long long row = (long long)k.b * p.S + key;
      bf16 *out = (w == 0 ? p.dK + row * p.lddk : p.dV + row * p.lddv) + (long long)k.kh * p.D + col;
#pragma unroll 1
      for (int c = 0; c < DH; c += 32) {
        uint32_t o[32];
        if (t.z > 0) {
          tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((w == 0 ? C::TM_DK : C::TM_DV) + col + c), o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] = 0u;
        }
        if (key < p.S) sa_store_row(out + c, o, w == 0 ? p.scale : 1.f, p.D - col - c, p.wide);
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------- dQ
template <int DT>
struct DqCfg {
  static constexpr int PANELS = DT / 64;
  static constexpr int TILE = SA_T * DT * 2;
  static constexpr int NK = 3, NV = 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_DO = OFF_Q + TILE;
  static constexpr int OFF_K = OFF_DO + TILE;
  static constexpr int OFF_V = OFF_K + NK * TILE;
  static constexpr int OFF_SPAN = OFF_V + NV * TILE;               // [128] int2
  static constexpr int OFF_RANGE = OFF_SPAN + 1024;                // [4] int2
  static constexpr int OFF_BAR = OFF_RANGE + 32;
  static constexpr int SLACK = 1024;
  static constexpr int SMEM = OFF_BAR + 256 + SLACK;
  static constexpr int TM_S = 0, TM_DP = 256, TM_DQ = 384;         // two score buffers
  static_assert(SMEM <= 232448, "tiles exceed the shared memory of a CTA");
};

template <int DT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(SAB_THREADS, 1)
span_attn_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ CUtensorMap tmDQ, const SpanArgs p) {
  using C = DqCfg<DT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int2 *span = (int2 *)(smem + C::OFF_SPAN);
  int2 *range = (int2 *)(smem + C::OFF_RANGE);
  uint64_t *bars = (uint64_t *)(smem + C::OFF_BAR);
  uint64_t *q_full = bars;
  uint64_t *k_full = bars + 1;        // [NK]
  uint64_t *k_ready = bars + 4;       // [NK]
  uint64_t *k_empty = bars + 7;       // [NK]
  uint64_t *v_full = bars + 10;       // [NV]
  uint64_t *v_empty = bars + 12;      // [NV]
  uint64_t *s_full = bars + 14;       // [2]
  uint64_t *dp_full = bars + 16;
  uint64_t *dp_free = bars + 17;      // SAB_WARPS
  // two, for the warps may be a tile apart (dP of the next one is there as soon as all have read this one's): an arrival for the next tile
  // must not count for this one
  uint64_t *ds_full = bars + 18;      // [2] SAB_WARPS
  uint64_t *dq_full = bars + 20;
  uint32_t *tmem_slot = (uint32_t *)(bars + 21);
  volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((uintptr_t)(smem - smem_raw) > (uintptr_t)C::SLACK) {
    pdl_entry();
    if (threadIdx.x == 0 && p.err) atomicCAS(p.err, 0, (int)FFK_ERR_BAD_ARG);
    return;
  }
  const int nqb = (p.S + SA_T - 1) / SA_T;
  const int bh = blockIdx.x % (p.B * p.H);
  const int qb = nqb - 1 - blockIdx.x / (p.B * p.H);
  const int h = bh % p.H, b = bh / p.H, kh = h / (p.H / p.KH);
  const int q0 = qb * SA_T;

  if (warp == 0) {
    if (lane == 0) {
      sa_prefetch_map(&tmQ); sa_prefetch_map(&tmDO); sa_prefetch_map(&tmK); sa_prefetch_map(&tmV);
      mbar_init(q_full, 1);
      for (int s = 0; s < C::NK; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_ready[s], 1); mbar_init(&k_empty[s], 1); }
      for (int s = 0; s < C::NV; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
      for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&ds_full[s], SAB_WARPS); }
      mbar_init(dp_full, 1); mbar_init(dp_free, SAB_WARPS); mbar_init(dq_full, 1);
      *abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_entry();
  if (warp == 0 && lane == 0) {           // before the others have met (see the forward kernel)
    mbar_expect_tx(q_full, 2 * C::TILE);
#pragma unroll
    for (int c = 0; c < C::PANELS; ++c) {
      tma_load_4d(smem_u32(smem + C::OFF_Q + c * SA_PANEL), &tmQ, q_full, c * 64, q0, h, b);
      tma_load_4d(smem_u32(smem + C::OFF_DO + c * SA_PANEL), &tmDO, q_full, c * 64, q0, h, b);
    }
  }
  __syncwarp();
  if (warp >= 4 && warp < 8) {
    const int r = (int)threadIdx.x - 128, q = q0 + r;
    const int2 s = q < p.S ? sa_span(p, b, q) : make_int2(1, 0);
    span[r] = s;
    const bool sees = s.x <= s.y;
    const int lo = __reduce_min_sync(0xffffffffu, sees ? s.x : 0x7fffffff), hi = __reduce_max_sync(0xffffffffu, sees ? s.y : -1);
    if (lane == 0) range[warp - 4] = make_int2(lo, hi);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int w = 0; w < 4; ++w) { first = min(first, range[w].x); last = max(last, range[w].y); }
  const int j0 = last < 0 ? 0 : first / SA_T;
  const int n = last < 0 ? 0 : last / SA_T - j0 + 1;

  // registers go from the warps that move data to the element-wise ones (128 x 64 + 512 x 104 = 640 x 96)
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      int ki = 0, vi = 0;
      uint64_t t0 = ffk_globaltimer();
      uint32_t spins = 0;
      while (ki < n || vi < n) {
        bool progress = false;
        if (ki < n) {
          const int s = ki % C::NK;
          if (mbar_try_wait(&k_empty[s], ((uint32_t)(ki / C::NK) & 1u) ^ 1u)) {
            mbar_expect_tx(&k_full[s], C::TILE);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
              tma_load_4d(smem_u32(smem + C::OFF_K + s * C::TILE + c * SA_PANEL), &tmK, &k_full[s], c * 64, (j0 + ki) * SA_T, kh, b);
            ++ki;
            progress = true;
          }
        }
        if (vi < n) {
          const int s = vi % C::NV;
          if (mbar_try_wait(&v_empty[s], ((uint32_t)(vi / C::NV) & 1u) ^ 1u)) {
            mbar_expect_tx(&v_full[s], C::TILE);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
              tma_load_4d(smem_u32(smem + C::OFF_V + s * C::TILE + c * SA_PANEL), &tmV, &v_full[s], c * 64, (j0 + vi) * SA_T, kh, b);
            ++vi;
            progress = true;
          }
        }
        if (progress) {
          t0 = ffk_globaltimer();
        } else if ((++spins & 63u) == 0) {
          if (*abort_flag) break;
          if (ffk_globaltimer() - t0 > WAIT_LIMIT_NS) {
            *abort_flag = 1;
            if (p.err) atomicCAS(p.err, 0, (int)FFK_ERR_TIMEOUT_PRODUCER);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    const uint64_t dq = make_smem_desc(smem_u32(smem + C::OFF_Q), 16, 1024), dd = make_smem_desc(smem_u32(smem + C::OFF_DO), 16, 1024);
    const uint64_t k_k0 = make_smem_desc(smem_u32(smem + C::OFF_K), 16, 1024), k_n0 = make_smem_desc(smem_u32(smem + C::OFF_K), SA_PANEL, 1024);
    const uint64_t v_k0 = make_smem_desc(smem_u32(smem + C::OFF_V), 16, 1024);
    const int ksteps = (p.D + 15) / 16;
    const uint32_t id_s = sa_idesc(128, SA_T, 0, 0), id_g = sa_idesc(128, ksteps * 16, 0, 1);
    auto issue_t = [&](uint32_t d, uint64_t a, uint64_t bk) {
      if (leader) {
        tc_mma_bf16<false>(d, a, bk, id_s);
#pragma unroll
        for (int s = 1; s < DT / 16; ++s) {
          if (s >= ksteps) break;
          const uint32_t off = (uint32_t)((s >> 2) * SA_PANEL + (s & 3) * 32);
          tc_mma_bf16<true>(d, desc_advance(a, off), desc_advance(bk, off), id_s);
        }
      }
    };
    auto issue_s = [&](int i) -> bool {
      const int s = i % C::NK;
      if (!mbar_wait_warp(&k_full[s], (uint32_t)(i / C::NK) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) ||
          !mbar_wait_warp(&k_ready[s], (uint32_t)(i / C::NK) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA))
        return false;
      tc_fence_after();
      issue_t(tmem_base + (uint32_t)(C::TM_S + (i & 1) * SA_T), dq, desc_advance(k_k0, (uint32_t)(s * C::TILE)));
      if (leader) tc_commit(&s_full[i & 1]);
      __syncwarp();
      return true;
    };
    auto issue_dp = [&](int i) -> bool {
      const int s = i % C::NV;
      if (!mbar_wait_warp(&v_full[s], (uint32_t)(i / C::NV) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA)) return false;
      tc_fence_after();
      issue_t(tmem_base + (uint32_t)C::TM_DP, dd, desc_advance(v_k0, (uint32_t)(s * C::TILE)));
      if (leader) {
        tc_commit(dp_full);
        tc_commit(&v_empty[s]);
      }
      __syncwarp();
      return true;
    };
    // also where the queries see nothing: a load under way does not outlive its CTA
    bool ok = mbar_wait_warp(q_full, 0, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) && n > 0 && issue_s(0) && issue_dp(0);
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t ph = (uint32_t)i & 1u;
      if (i + 1 < n) {
        ok = issue_s(i + 1) && mbar_wait_warp(dp_free, ph, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) && issue_dp(i + 1);
        if (!ok) break;
      }
      ok = mbar_wait_warp(&ds_full[i & 1], (uint32_t)(i >> 1) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        const uint32_t d = tmem_base + (uint32_t)C::TM_DQ, a = tmem_base + (uint32_t)(C::TM_S + (i & 1) * SA_T);
        const uint64_t bn = desc_advance(k_n0, (uint32_t)((i % C::NK) * C::TILE));
        if (i == 0) tc_mma_ts_bf16<false>(d, a, bn, id_g);
        else tc_mma_ts_bf16<true>(d, a, bn, id_g);
#pragma unroll
        for (int s = 1; s < SA_T / 16; ++s)
          tc_mma_ts_bf16<true>(d, a + (uint32_t)((s >> 1) * 32 + (s & 1) * 8), desc_advance(bn, (uint32_t)(s * 2048)), id_g);
        tc_commit(&k_empty[i % C::NK]);
        if (i + 1 == n) tc_commit(dq_full);
      }
      __syncwarp();
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ rows of K that no query of the block sees
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int k0 = (j0 + i) * SA_T, s = i % C::NK;
      uint32_t keep[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int2 t = span[r * 32 + lane];
        if (t.x <= t.y) sa_add_bits(keep, t.x - k0, t.y - k0);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) keep[w] = __reduce_or_sync(0xffffffffu, keep[w]);
      ok = sa_wait(&k_full[s], (uint32_t)(i / C::NK) & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
      if (!ok) break;
      if ((keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu) {
        sa_clear_rows<C::PANELS>(smem + C::OFF_K + s * C::TILE, keep, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      sa_warp_arrive(&k_ready[s], lane);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ------------------------------------------------------------------ dS: thread = query x 32 of the tile's keys
    const int quarter = warp & 3, cols = (warp - 4) >> 2;
    const int r = quarter * 32 + lane, q = q0 + r, q_low = q - lane;
    const int2 mine = span[r];
    const bool empty = mine.x > mine.y;
    const int lo = empty ? -1 : mine.x, hi = empty ? 0x7ffffff0 : mine.y;      // see the forward kernel
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(cols * 32);
    const float slope = BIAS ? p.slopes[h] : 0.f;
    const long long stat = ((long long)b * p.H + h) * p.S + q;
    const float neg_lse = empty ? -INFINITY : -p.lse[stat], neg_delta = empty ? 0.f : -p.delta[stat];
    const pair32 nl = pair_of(neg_lse, neg_lse), nd = pair_of(neg_delta, neg_delta), ff = pair_of(p.factor, p.factor);
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t ph = (uint32_t)i & 1u;
      const int kg = (j0 + i) * SA_T + cols * 32;
      const uint32_t t_s = lane_base + (uint32_t)(C::TM_S + (i & 1) * SA_T);
      const bool masked = !__all_sync(0xffffffffu, lo <= kg && hi >= kg + 31);
      const bool none = masked && !__any_sync(0xffffffffu, lo <= kg + 31 && hi >= kg);
      ok = sa_wait(&s_full[i & 1], (uint32_t)(i >> 1) & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
      if (!ok) break;
      tc_fence_after();
      uint32_t y[32], pk[16];
      if (!none) {
        tmem_ld32(t_s, y);
        tmem_ld_wait();
        if (CAP && masked) sa_mask(y, lo - kg, hi - kg, 0u);       // masked scores do not choose the way tanh is taken
        if constexpr (CAP) {
          if (!sa_cap(y, p, !empty)) sa_cap_any(y, p);
        }
        SaBias bias(slope, (float)(kg - q), kg + 31 <= q_low ? -1 : kg >= q_low + 31 ? 1 : 0);
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
          float e[16];
#pragma unroll
          for (int u = 0; u < 16; u += 2) pair_to(pair_fma(pair_get(&y[c + u]), ff, BIAS ? bias.next(nl) : nl), e[u], e[u + 1]);
          if (masked) {
#pragma unroll
            for (int u = 0; u < 16; ++u)
              if (c + u < lo - kg || c + u > hi - kg) e[u] = -INFINITY;
          }
#pragma unroll
          for (int u = 0; u < 16; ++u) e[u] = sa_exp2(e[u]);
#pragma unroll
          for (int u = 0; u < 16; u += 2) {
            if constexpr (CAP) {
              sa_times_slope(y, c + u, e[u], e[u + 1], p.to_z);
            } else {
              y[c + u] = __float_as_uint(e[u]);
              y[c + u + 1] = __float_as_uint(e[u + 1]);
            }
          }
        }
      }
      ok = sa_wait(dp_full, ph, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
      if (!ok) break;
      tc_fence_after();
      uint32_t z[32];
      if (!none) {
        tmem_ld32(lane_base + C::TM_DP, z);
        tmem_ld_wait();
      }
      tc_fence_before();
      sa_warp_arrive(dp_free, lane);
      if (none) {
#pragma unroll
        for (int c = 0; c < 16; ++c) pk[c] = 0u;
      } else {
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          float e0, e1;
          pair_to(pair_mul(pair_get(&y[c]), pair_add(pair_get(&z[c]), nd)), e0, e1);
          if (masked) {                   // whatever V and delta hold there
            if (__uint_as_float(y[c]) == 0.f) e0 = 0.f;
            if (__uint_as_float(y[c + 1]) == 0.f) e1 = 0.f;
          }
          pk[c >> 1] = pack_bf162(e0, e1);
        }
      }
      sa_tmem_st16(t_s, pk);
      tmem_st_wait();
      tc_fence_before();
      sa_warp_arrive(&ds_full[i & 1], lane);
    }
    if (ok) {                             // without a step, Q has to be there before its place is written
      ok = sa_wait(n > 0 ? dq_full : q_full, 0, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
      tc_fence_after();
    }
    if (ok) {
      if (cols * 32 < DT) {               // a thread 32 of its query's columns, through the place of Q
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(C::TM_DQ + cols * 32), o);
          tmem_ld_wait();
        }
        if (empty) {
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] = 0u;
        }
        sa_tile_row(smem + C::OFF_Q, r, cols * 32, o, p.scale);
        sa_tile_out<C::PANELS>(smem + C::OFF_Q, &tmDQ, q0, h, b, 1, DT * 4, warp == 4 && lane == 0);
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

struct SpanMaps { CUtensorMap q, k, v, dout, dq; };

template <int DT, bool CAP, bool BIAS>
int launch_bwd(const SpanMaps &m, const SpanArgs &a, cudaStream_t st) {
  static unsigned long long done_kv = 0, done_q = 0;
  cudaError_t e = ffk_allow_smem(span_attn_dkv_kernel<DT, CAP, BIAS>, DkvCfg<DT>::SMEM, done_kv);
  if (e != cudaSuccess) return (int)e;
  e = ffk_allow_smem(span_attn_dq_kernel<DT, CAP, BIAS>, DqCfg<DT>::SMEM, done_q);
  if (e != cudaSuccess) return (int)e;
  const long long tiles = (a.S + SA_T - 1) / SA_T;
  int r = ffk_launch(span_attn_dkv_kernel<DT, CAP, BIAS>, (unsigned)(tiles * a.B * a.KH), SAB_THREADS, DkvCfg<DT>::SMEM, st, m.q, m.k, m.v, m.dout, a);
  if (r) return r;
  return ffk_launch(span_attn_dq_kernel<DT, CAP, BIAS>, (unsigned)(tiles * a.B * a.H), SAB_THREADS, DqCfg<DT>::SMEM, st, m.q, m.k, m.v, m.dout, m.dq, a);
}

long long delta_floats(long long B, long long H, long long S) { return (B * H * S + 3) / 4 * 4; }

}  // namespace

FFK_API long long ffk_span_attention_bwd_scratch_floats(int B, int H, int S) {
  if (B <= 0 || H <= 0 || S <= 0) return 0;
  return delta_floats(B, H, S) + 4ll * B * ((S + SA_T - 1) / SA_T);
}

FFK_API int ffk_span_attention_bwd(const FfkSpanAttnDesc *d, cudaStream_t st) {
  if (d->B <= 0 || d->H <= 0 || d->S <= 0) return 0;
  if (!sa_shape_ok(d)) return -2;
  if (!sa_aligned(d->Q, d->ldq) || !sa_aligned(d->K, d->ldk) || !sa_aligned(d->V, d->ldv) || !sa_aligned(d->O, d->ldo) || !sa_aligned(d->dO, d->lddo) ||
      !sa_aligned(d->dQ, d->lddq) || !sa_aligned(d->dK, d->lddk) || !sa_aligned(d->dV, d->lddv) || (((uintptr_t)d->scratch) & 15) || !d->lse)
    return -2;
  const long long tiles = (d->S + SA_T - 1) / SA_T, rows = (long long)d->B * d->S * d->H;
  const int lanes = d->D <= 64 ? 8 : 16;
  const long long delta_blocks = (rows * lanes + 255) / 256, sum_blocks = (d->B * tiles + 7) / 8;
  if (tiles * d->B * d->H > 0x7fffffffll || rows > 0x7fffffffll || delta_blocks + sum_blocks > 0x7fffffffll) return -2;
  SpanMaps m;
  int r;
  if ((r = sa_head_map(&m.q, d->Q, d->D, d->S, d->ldq, d->H, d->B))) return r;
  if ((r = sa_head_map(&m.k, d->K, d->D, d->S, d->ldk, d->KH, d->B))) return r;
  if ((r = sa_head_map(&m.v, d->V, d->D, d->S, d->ldv, d->KH, d->B))) return r;
  if ((r = sa_head_map(&m.dout, d->dO, d->D, d->S, d->lddo, d->H, d->B))) return r;
  if ((r = sa_head_map(&m.dq, d->dQ, d->D, d->S, d->lddq, d->H, d->B))) return r;
  SpanArgs a = {};
  sa_args(d, a, ffk_span_attention_err());
  float *delta = d->scratch;
  int4 *summary = reinterpret_cast<int4 *>(d->scratch + delta_floats(d->B, d->H, d->S));
  a.delta = delta;
  a.summary = summary;
  a.dK = (bf16 *)d->dK; a.lddk = d->lddk; a.dV = (bf16 *)d->dV; a.lddv = d->lddv;
  a.wide = sa_wide(d->dK, d->lddk, d->D) && sa_wide(d->dV, d->lddv, d->D);
  FfkTraffic traffic((long long)d->B * d->S * d->D * 4 * (d->H + d->KH));
  a.Q = (const bf16 *)d->Q; a.ldq = d->ldq; a.K = (const bf16 *)d->K; a.ldk = d->ldk; a.V = (const bf16 *)d->V; a.ldv = d->ldv;
  const unsigned blocks = (unsigned)(delta_blocks + sum_blocks);
  r = lanes == 8 ? ffk_launch(span_attn_prep_kernel<8>, blocks, 256, 0, st, (const bf16 *)d->dO, d->lddo, (const bf16 *)d->O, d->ldo, delta, summary,
                              (int)delta_blocks, a)
                 : ffk_launch(span_attn_prep_kernel<16>, blocks, 256, 0, st, (const bf16 *)d->dO, d->lddo, (const bf16 *)d->O, d->ldo, delta, summary,
                              (int)delta_blocks, a);
  if (r) return r;
  const bool cap = d->cap > 0.f, bias = d->slopes != nullptr;
  if (d->D <= 64) {
    if (cap) return bias ? launch_bwd<64, true, true>(m, a, st) : launch_bwd<64, true, false>(m, a, st);
    return bias ? launch_bwd<64, false, true>(m, a, st) : launch_bwd<64, false, false>(m, a, st);
  }
  if (cap) return bias ? launch_bwd<128, true, true>(m, a, st) : launch_bwd<128, true, false>(m, a, st);
  return bias ? launch_bwd<128, false, true>(m, a, st) : launch_bwd<128, false, false>(m, a, st);
}
