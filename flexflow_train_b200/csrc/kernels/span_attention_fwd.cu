// span_attention_fwd.cu -- forward pass of attention over spans of keys (span_attention.cuh has the mathematics).
//
// A CTA (256 threads, two of them on an SM) takes 128 queries of one (batch row, head) and walks over the key tiles from the first to the
// last that any of them sees; scores and probabilities exist in tensor memory and registers only:
//   warp 0      TMA producer: Q once, then the K and V tiles
//   warp 1      MMA issuer: S = Q K_j^T, O += P V_j
//   warp 2      clears the rows of V_j that no query of the CTA sees (only where a tile holds such rows)
//   warps 4-7   softmax, thread = query row.  P overwrites the first columns of S as bf16 and is the A operand of the second product from
//               there.  The reference maximum of a row moves only when the true one has grown by 2^8, and then the thread rescales its row
//               of O in tensor memory: the common step has no correction pass.
// P is rounded to bf16, the type that the second product takes; its sum l is taken of the unrounded values in fp32, O is rounded once.
//
// What bounds it: per SM and pair of tiles (128 x 128 x 128 each) the tensor core takes 2048 cycles for both CTAs' products, the exponentials
// 2048 of the special-function unit, and within a tile the one waits for the other; a cap adds about as much of the FMA pipe.  Two CTAs an SM
// fill each other's waits, also where one sets up or writes its result, which a CTA of a few tiles spends a third of its time on, and balance
// spans of uneven lengths by 128 queries.  They hold half of the tensor memory and, with heads of 128, one K and one V tile each: K_j+1 arrives
// under the softmax of tile j, V_j+1 under that of j + 1.  Against one CTA with two query tiles and rings of two and three, K and V read
// once for both (both on the same device in turn): 8192 causal, 16 heads of 128, cap: 339 -> 329 us (835 TFLOP/s), without a cap 244 -> 255
// (1080); 8 x 2048 in documents of about 700, 16 heads of 128, cap: 189 -> 162; 8 x 1024 with prompts, heads of 64, bias: 49 -> 41; 4 x 1001
// causal, bias: 41 -> 35.
//
// Every wait is bounded (tcgen05.cuh).
#include "span_attention.cuh"

namespace {

constexpr int SAF_THREADS = 256;
constexpr float SAF_GAP = 8.f;          // log-2 units by which a row's maximum may exceed the reference in use

template <int DT>                       // columns of a tile: 64 or 128
struct SafCfg {
  static constexpr int PANELS = DT / 64;
  static constexpr int TILE = SA_T * DT * 2;
  static constexpr int NK = DT == 128 ? 1 : 2, NV = NK;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + TILE;
  static constexpr int OFF_V = OFF_K + NK * TILE;
  static constexpr int OFF_SPAN = OFF_V + NV * TILE;              // [128] int2
  static constexpr int OFF_RANGE = OFF_SPAN + SA_T * 8;           // [4] int2: smallest first and largest last of 32 rows
  static constexpr int OFF_BAR = OFF_RANGE + 32;
  static constexpr int SLACK = 1024;                              // the base is aligned to that (checked in the kernel)
  static constexpr int SMEM = OFF_BAR + 128 + SLACK;
  static_assert(SMEM <= 233472 / 2 - 1024, "two CTAs do not fit an SM");
  static constexpr int TM_S = 0, TM_O = 128, TM_COLS = 256;       // columns of tensor memory: half of the SM's
};

template <int DT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(SAF_THREADS, 2)
span_attn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ CUtensorMap tmO, const SpanArgs p) {
  using C = SafCfg<DT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int2 *span = (int2 *)(smem + C::OFF_SPAN);
  int2 *range = (int2 *)(smem + C::OFF_RANGE);
  uint64_t *bars = (uint64_t *)(smem + C::OFF_BAR);
  uint64_t *q_full = bars;
  uint64_t *s_full = bars + 1;
  uint64_t *p_full = bars + 2;        // four warps
  uint64_t *o_full = bars + 3;
  uint64_t *k_full = bars + 4;        // [NK]
  uint64_t *k_empty = bars + 6;       // [NK]
  uint64_t *v_full = bars + 8;        // [NV]
  uint64_t *v_ready = bars + 10;      // [NV]
  uint64_t *v_empty = bars + 12;      // [NV]
  uint32_t *tmem_slot = (uint32_t *)(bars + 14);
  volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((uintptr_t)(smem - smem_raw) > (uintptr_t)C::SLACK) {      // the launch did not leave room to align the tiles: refuse
    pdl_entry();
    if (threadIdx.x == 0 && p.err) atomicCAS(p.err, 0, (int)FFK_ERR_BAD_ARG);
    return;
  }
  // the query blocks of all heads in turn, the last ones (which see most keys under a causal mask) first
  const int nqb = (p.S + SA_T - 1) / SA_T;
  const int bh = blockIdx.x % (p.B * p.H);
  const int qb = nqb - 1 - blockIdx.x / (p.B * p.H);
  const int h = bh % p.H, b = bh / p.H, kh = h / (p.H / p.KH);
  const int q0 = qb * SA_T;

  // Set-up, as far as it does not touch global memory under the previous kernel's tail.  The warp that sets up the barriers asks for Q before
  // the others have met: a CTA is a few tiles long, and its first products wait for these loads.
  if (warp == 0) {
    if (lane == 0) {
      sa_prefetch_map(&tmQ); sa_prefetch_map(&tmK); sa_prefetch_map(&tmV);
      mbar_init(q_full, 1); mbar_init(s_full, 1); mbar_init(p_full, 4); mbar_init(o_full, 1);
      for (int s = 0; s < C::NK; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
      for (int s = 0; s < C::NV; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_ready[s], 1); mbar_init(&v_empty[s], 1); }
      *abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)C::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_entry();
  if (warp == 0 && lane == 0) {
    mbar_expect_tx(q_full, C::TILE);
#pragma unroll
    for (int c = 0; c < C::PANELS; ++c) tma_load_4d(smem_u32(smem + C::OFF_Q + c * SA_PANEL), &tmQ, q_full, c * 64, q0, h, b);
  }
  __syncwarp();
  // spans of the CTA's queries, and what each 32 of them see together
  if (warp >= 4) {
    const int r = (int)threadIdx.x - 128, q = q0 + r;
    int2 s = make_int2(1, 0);
    if (q < p.S) s = sa_span(p, b, q);
    span[r] = s;
    const bool sees = s.x <= s.y;
    const int lo = __reduce_min_sync(0xffffffffu, sees ? s.x : 0x7fffffff), hi = __reduce_max_sync(0xffffffffu, sees ? s.y : -1);
    if (lane == 0) range[warp - 4] = make_int2(lo, hi);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // key tiles that any of the queries sees: j0 to j0 + n - 1
  int j0 = 0x7fffffff, j1 = -1;
#pragma unroll
  for (int w = 0; w < 4; ++w) { j0 = min(j0, range[w].x); j1 = max(j1, range[w].y); }
  const int n = j1 < 0 ? 0 : j1 / SA_T - j0 / SA_T + 1;
  j0 = n > 0 ? j0 / SA_T : 0;

  // the softmax warps hold a row of scores each: registers go from the four warps that move data to them (128 x 72 + 128 x 184 = 256 x
  // 128; splits from 48 / 208 to this one take the same time within 2 %)
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      // the K and the V ring advance independently; the wait for progress on either is bounded
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
    // ------------------------------------------------------------------ MMA issuer: the whole warp runs, one lane issues
    const bool leader = elect_one();
    const uint64_t dq0 = make_smem_desc(smem_u32(smem + C::OFF_Q), 16, 1024);
    const uint64_t dk0 = make_smem_desc(smem_u32(smem + C::OFF_K), 16, 1024);
    const uint64_t dv0 = make_smem_desc(smem_u32(smem + C::OFF_V), SA_PANEL, 1024);
    const int ksteps = (p.D + 15) / 16;                                   // of Q K^T; the columns beyond D are zeros
    const uint32_t id_s = sa_idesc(128, SA_T, 0, 0), id_o = sa_idesc(128, ksteps * 16, 0, 1);
    bool ok = true;
    // S overwrites the columns that P was read from: products run in issue order
    auto issue_s = [&](int i) {
      if (leader) {
        const uint64_t k = desc_advance(dk0, (uint32_t)((i % C::NK) * C::TILE));
        const uint32_t d = tmem_base + (uint32_t)C::TM_S;
        tc_mma_bf16<false>(d, dq0, k, id_s);
#pragma unroll
        for (int s = 1; s < DT / 16; ++s) {
          if (s >= ksteps) break;         // unrolled: the one lane that issues bounds the tensor core otherwise
          const uint32_t off = (uint32_t)((s >> 2) * SA_PANEL + (s & 3) * 32);
          tc_mma_bf16<true>(d, desc_advance(dq0, off), desc_advance(k, off), id_s);
        }
        tc_commit(s_full);
        tc_commit(&k_empty[i % C::NK]);
      }
      __syncwarp();
    };
    // also where the queries see nothing: a load under way does not outlive its CTA
    ok = mbar_wait_warp(q_full, 0, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
    for (int i = 0; i <= n && ok; ++i) {
      if (i > 0) {
        const int at = (i - 1) % C::NV;
        const uint32_t phase = (uint32_t)((i - 1) / C::NV) & 1u;
        ok = mbar_wait_warp(&v_full[at], phase, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) &&
             mbar_wait_warp(&v_ready[at], phase, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA) &&
             mbar_wait_warp(p_full, (uint32_t)(i - 1) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint64_t v = desc_advance(dv0, (uint32_t)(at * C::TILE));
          const uint32_t d = tmem_base + (uint32_t)C::TM_O, a = tmem_base + (uint32_t)C::TM_S;
          if (i == 1) tc_mma_ts_bf16<false>(d, a, v, id_o);
          else tc_mma_ts_bf16<true>(d, a, v, id_o);
#pragma unroll
          for (int s = 1; s < SA_T / 16; ++s) tc_mma_ts_bf16<true>(d, a + (uint32_t)(s * 8), desc_advance(v, (uint32_t)(s * 2048)), id_o);
          tc_commit(&v_empty[at]);
          if (i == n) tc_commit(o_full);
        }
        __syncwarp();
      }
      if (i < n) {
        ok = mbar_wait_warp(&k_full[i % C::NK], (uint32_t)(i / C::NK) & 1u, abort_flag, p.err, FFK_ERR_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        issue_s(i);
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ rows of V that nothing sees
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int k0 = (j0 + i) * SA_T;
      uint32_t keep[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int2 s = span[r * 32 + lane];
        if (s.x <= s.y) sa_add_bits(keep, s.x - k0, s.y - k0);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) keep[w] = __reduce_or_sync(0xffffffffu, keep[w]);
      ok = sa_wait(&v_full[i % C::NV], (uint32_t)(i / C::NV) & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
      if (!ok) break;
      if ((keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu) {
        sa_clear_rows<C::PANELS>(smem + C::OFF_V + (i % C::NV) * C::TILE, keep, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      sa_warp_arrive(&v_ready[i % C::NV], lane);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ------------------------------------------------------------------ softmax: thread = query row
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int q = q0 + r;
    const int2 mine = span[r];
    const bool empty = mine.x > mine.y;
    // a row that sees nothing computes what it likes and stores zeros: it does not keep its warp from the unmasked path
    const int lo = empty ? -1 : mine.x, hi = empty ? 0x7ffffff0 : mine.y;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t t_s = lane_base + (uint32_t)C::TM_S, t_o = lane_base + (uint32_t)C::TM_O;
    const float slope = BIAS ? p.slopes[h] / p.scale : 0.f;
    const int q_low = q - lane;            // the warp's first row
    float m = -INFINITY, l = 0.f;          // m: what the row's exponentials are taken against; -infinity until the row has seen a key
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int k0 = (j0 + i) * SA_T;
      ok = sa_wait(s_full, (uint32_t)i & 1u, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);
      if (!ok) break;
      tc_fence_after();
      uint32_t x[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(t_s + (uint32_t)(c * 32), *reinterpret_cast<uint32_t(*)[32]>(&x[c * 32]));
      tmem_ld_wait();
      // a warp whose rows all see the whole tile takes no mask; masked scores do not choose the way tanh is taken
      const bool full = __all_sync(0xffffffffu, lo <= k0 && hi >= k0 + SA_T - 1);
      const int first = lo - k0, width = hi - lo;
      if (CAP && !full) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if ((unsigned)(c - first) > (unsigned)width) x[c] = 0u;
      }
      if constexpr (CAP) {
        if (!sa_cap(x, p, !empty)) {
          // scores near the cap, 32 columns at a time through tensor memory, where they still are: this path is rare and its code was as long
          // as the rest of the step's
#pragma unroll 1
          for (int g = 0; g < 4; ++g) {
            uint32_t y[32];
            tmem_ld32(t_s + (uint32_t)(g * 32), y);
            tmem_ld_wait();
            sa_cap_any(y, p);
            tmem_st32(t_s + (uint32_t)(g * 32), y);
          }
          tmem_st_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_s + (uint32_t)(c * 32), sa_group(x, c));
          tmem_ld_wait();
        }
      }
      if constexpr (BIAS) sa_bias(x, slope, (float)(k0 - q), k0 + SA_T - 1 <= q_low ? -1 : k0 >= q_low + 31 ? 1 : 0);
      if (!full) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if ((unsigned)(c - first) > (unsigned)width) x[c] = 0xff800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 128; c += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], fmaxf(__uint_as_float(x[c + u]), __uint_as_float(x[c + 4 + u])));
      }
      const float f = p.factor;
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * f;
      const bool need = top > m + SAF_GAP;
      if (i == 0) {
        m = top;
      } else if (__any_sync(0xffffffffu, need)) {
        // the scores were issued after P V of the tile before, and have arrived: O holds all earlier tiles and nothing is under way
        const float alpha = need ? (m == -INFINITY ? 0.f : sa_exp2(m - top)) : 1.f;
#pragma unroll 1
        for (int c = 0; c < DT / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + (uint32_t)(c * 32), o);
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * alpha);
          tmem_st32(t_o + (uint32_t)(c * 32), o);
        }
        l *= alpha;
        if (need) m = top;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      const pair32 ff = pair_of(f, f), neg = pair_of(-ref, -ref);
      pair32 sum0 = pair_of(l, 0.f), sum1 = pair_of(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 128; c += 16) {
        float e[16];
#pragma unroll
        for (int u = 0; u < 16; u += 2) pair_to(pair_fma(pair_get(&x[c + u]), ff, neg), e[u], e[u + 1]);
#pragma unroll
        for (int u = 0; u < 16; ++u) e[u] = sa_exp2(e[u]);
#pragma unroll
        for (int u = 0; u < 16; u += 4) {
          sum0 = pair_add(sum0, pair_of(e[u], e[u + 1]));
          sum1 = pair_add(sum1, pair_of(e[u + 2], e[u + 3]));
        }
#pragma unroll
        for (int u = 0; u < 16; u += 2) x[(c + u) >> 1] = pack_bf162(e[u], e[u + 1]);
      }
      float s0, s1, s2, s3;
      pair_to(sum0, s0, s1);
      pair_to(sum1, s2, s3);
      l = (s0 + s1) + (s2 + s3);
      tmem_st32(t_s, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
      tmem_st32(t_s + 32u, *reinterpret_cast<uint32_t(*)[32]>(&x[32]));
      tmem_st_wait();
      tc_fence_before();
      sa_warp_arrive(p_full, lane);
    }
    if (ok) ok = sa_wait(n > 0 ? o_full : q_full, 0, abort_flag, p, FFK_ERR_TIMEOUT_EPILOGUE);      // without a key, Q has to be there before its place is written
    tc_fence_after();
    if (ok) {
      const bool stored = q < p.S;
      const float inv = empty || !(l != 0.f) ? 0.f : 1.f / l;
      if (stored && p.lse) p.lse[((long long)b * p.H + h) * p.S + q] = empty ? 0.f : m + __log2f(l);
      // O goes out through the queries' place: the last product has read that
      uint8_t *tile = smem + C::OFF_Q;
#pragma unroll 1
      for (int c = 0; c < DT / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(t_o + (uint32_t)(c * 32), o);
          tmem_ld_wait();
        }
        if (empty) {
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] = 0u;
        }
        sa_tile_row(tile, r, c * 32, o, inv);
      }
      sa_tile_out<C::PANELS>(tile, &tmO, q0, h, b, 1, 128, threadIdx.x == 128);
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)C::TM_COLS) : "memory");
  }
}

__device__ int g_span_attn_err = 0;

template <int DT, bool CAP, bool BIAS>
int launch_fwd(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const CUtensorMap &to, const SpanArgs &a, long long grid, cudaStream_t st) {
  static unsigned long long done = 0;
  const cudaError_t e = ffk_allow_smem(span_attn_fwd_kernel<DT, CAP, BIAS>, SafCfg<DT>::SMEM, done);
  if (e != cudaSuccess) return (int)e;
  return ffk_launch(span_attn_fwd_kernel<DT, CAP, BIAS>, (unsigned)grid, SAF_THREADS, SafCfg<DT>::SMEM, st, tq, tk, tv, to, a);
}

}  // namespace

int *ffk_span_attention_err() {
  void *p = nullptr;
  return cudaGetSymbolAddress(&p, g_span_attn_err) == cudaSuccess ? (int *)p : nullptr;
}

FFK_API int ffk_span_attention_fwd(const FfkSpanAttnDesc *d, cudaStream_t st) {
  if (d->B <= 0 || d->H <= 0 || d->S <= 0) return 0;
  if (!sa_shape_ok(d)) return -2;
  if (!sa_aligned(d->Q, d->ldq) || !sa_aligned(d->K, d->ldk) || !sa_aligned(d->V, d->ldv) || !sa_aligned(d->O, d->ldo)) return -2;
  CUtensorMap tq, tk, tv, to;
  int r;
  if ((r = sa_head_map(&tq, d->Q, d->D, d->S, d->ldq, d->H, d->B))) return r;
  if ((r = sa_head_map(&tk, d->K, d->D, d->S, d->ldk, d->KH, d->B))) return r;
  if ((r = sa_head_map(&tv, d->V, d->D, d->S, d->ldv, d->KH, d->B))) return r;
  if ((r = sa_head_map(&to, d->O, d->D, d->S, d->ldo, d->H, d->B))) return r;
  SpanArgs a = {};
  sa_args(d, a, ffk_span_attention_err());
  const long long heads = (long long)d->B * d->H;
  const long long grid = heads * ((d->S + SA_T - 1) / SA_T);
  if (heads > 0x7fffffffll || grid > 0x7fffffffll) return -2;
  FfkTraffic traffic((long long)d->B * d->S * d->D * 2 * (2 * d->H + 2 * d->KH));
  const bool cap = d->cap > 0.f, bias = d->slopes != nullptr;
  if (d->D <= 64) {
    if (cap) return bias ? launch_fwd<64, true, true>(tq, tk, tv, to, a, grid, st) : launch_fwd<64, true, false>(tq, tk, tv, to, a, grid, st);
    return bias ? launch_fwd<64, false, true>(tq, tk, tv, to, a, grid, st) : launch_fwd<64, false, false>(tq, tk, tv, to, a, grid, st);
  }
  if (cap) return bias ? launch_fwd<128, true, true>(tq, tk, tv, to, a, grid, st) : launch_fwd<128, true, false>(tq, tk, tv, to, a, grid, st);
  return bias ? launch_fwd<128, false, true>(tq, tk, tv, to, a, grid, st) : launch_fwd<128, false, false>(tq, tk, tv, to, a, grid, st);
}

// Reads (and clears) the error word of the bounded waits of both directions.  Synchronises the device.
FFK_API int ffk_span_attention_last_error() {
  int v = 0, z = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  cudaMemcpyFromSymbol(&v, g_span_attn_err, sizeof(int));
  cudaMemcpyToSymbol(g_span_attn_err, &z, sizeof(int));
  return v;
}
