// rmsnorm.cu -- root-mean-square norm with the residual's addition, forward and backward.
//
//   h = a + r  (rounded to the type it is stored in: the residual stream),   y = h * rstd * gamma,   rstd = (mean(h^2) + eps)^(-1/2)
//   g = dy * gamma,   dh = rstd * (g - h * rstd^2 * mean(g h)) + dsum,   dgamma = sum over rows of dy * h * rstd
//
// dsum is the gradient that reaches h past the norm; dh is the gradient of a and of r.  Statistics, products and sums are held in 32 bits;
// y, dh and dgamma are rounded once, when they are stored.
//
// What bounds it: HBM.  A row is read once into registers and written once: forward 4, backward 4 row's worth of bytes.  A row belongs to
// WARPS warps (one exchange through shared memory among them; none for one warp), as many as give a thread one piece of V elements (16
// bytes, or one element where the width or an address does not allow that), up to 16 warps (8 of single elements); wider rows give N pieces.  More pieces and fewer
// warps cost registers and with them the loads under way: 32768 x 1024 backward 60 us with one warp and four pieces.  Backward's blocks stay
// for many rows: a thread keeps the columns it owns of dgamma in registers and the block leaves one partial row, which the fold adds in a
// fixed order.  Rows too wide for registers take the kernels at the end, which read a row twice.  32768 x 2048 bf16 with residual: forward 80
// us (6.7 TB/s), backward 92 with the fold (5.8 TB/s); 4004 x 1001 fp32, single elements: 29 both ways; 128 x 512 bf16 forward: 2.1.
#include "common.cuh"

namespace {

template <typename T> __device__ __forceinline__ float rms_ld(const T *p);
template <> __device__ __forceinline__ float rms_ld<float>(const float *p) { return *p; }
template <> __device__ __forceinline__ float rms_ld<bf16>(const bf16 *p) { return bf2f(*p); }
__device__ __forceinline__ void rms_st(float *p, float v) { *p = v; }
__device__ __forceinline__ void rms_st(bf16 *p, float v) { *p = f2bf(v); }
__device__ __forceinline__ float rms_round(float v, const float *) { return v; }
__device__ __forceinline__ float rms_round(float v, const bf16 *) { return bf2f(f2bf(v)); }

// V elements as they lie in memory
template <typename T, int V> struct Piece;
template <> struct Piece<float, 1> {
  float u;
  __device__ __forceinline__ void load(const float *p) { u = *p; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = u; }
  __device__ __forceinline__ void set(const float (&v)[1]) { u = v[0]; }
  __device__ __forceinline__ void store(float *p) const { *p = u; }
  __device__ __forceinline__ void zero() { u = 0.f; }
};
template <> struct Piece<bf16, 1> {
  bf16 u;
  __device__ __forceinline__ void load(const bf16 *p) { u = *p; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = bf2f(u); }
  __device__ __forceinline__ void set(const float (&v)[1]) { u = f2bf(v[0]); }
  __device__ __forceinline__ void store(bf16 *p) const { *p = u; }
  __device__ __forceinline__ void zero() { u = f2bf(0.f); }
};
template <> struct Piece<float, 4> {
  float4 u;
  __device__ __forceinline__ void load(const float *p) { u = *reinterpret_cast<const float4 *>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w; }
  __device__ __forceinline__ void set(const float (&v)[4]) { u = make_float4(v[0], v[1], v[2], v[3]); }
  __device__ __forceinline__ void store(float *p) const { *reinterpret_cast<float4 *>(p) = u; }
  __device__ __forceinline__ void zero() { u = make_float4(0.f, 0.f, 0.f, 0.f); }
};
template <> struct Piece<bf16, 8> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16 *p) { u = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const float2 a = unpack_bf162(u.x), b = unpack_bf162(u.y), c = unpack_bf162(u.z), d = unpack_bf162(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    u = make_uint4(pack_bf162(v[0], v[1]), pack_bf162(v[2], v[3]), pack_bf162(v[4], v[5]), pack_bf162(v[6], v[7]));
  }
  __device__ __forceinline__ void store(bf16 *p) const { *reinterpret_cast<uint4 *>(p) = u; }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
};

// Sum over the WARPS warps that share a row (group `group` of the block).  `red`: two sets of WARPS floats per group, which successive rows use
// in turn, so that one barrier a row is enough.
template <int WARPS>
__device__ __forceinline__ float row_sum(float v, float *red, int group, int parity) {
  v = warp_sum(v);
  if constexpr (WARPS > 1) {
    float *r = red + (group * 2 + parity) * WARPS;
    if ((threadIdx.x & 31) == 0) r[(threadIdx.x >> 5) % WARPS] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(WARPS * 32) : "memory");
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += r[w];
  }
  return v;
}
__host__ __device__ constexpr int rms_threads(int warps) { return warps > 8 ? warps * 32 : 256; }      // of a block at most: several rows where they are narrow

// a, r, xsum and y are read and written element by element by the same thread: y or xsum may be a or r
template <typename T, int V, int N, int WARPS>
__global__ void __launch_bounds__(rms_threads(WARPS)) rms_fwd_kernel(const T *a, const T *b, const T *gamma, T *xsum, T *y, float *__restrict__ rstd, int rows,
                                                      int cols, float eps) {
  pdl_entry(xsum, y);
  __shared__ float red[2 * rms_threads(WARPS) / 32];
  const int slot = threadIdx.x % (WARPS * 32), group = threadIdx.x / (WARPS * 32);
  const int per_block = blockDim.x / (WARPS * 32);
  const float inv = 1.f / (float)cols;
  int parity = 0;
  for (long long row = (long long)blockIdx.x * per_block + group; row < rows; row += (long long)gridDim.x * per_block) {
    const long long base = row * cols;
    Piece<T, V> pa[N], pb[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * WARPS * 32 + slot) * V;
      pa[i].zero();
      pb[i].zero();
      if (c < cols) {
        pa[i].load(a + base + c);
        if (b) pb[i].load(b + base + c);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float u[V], w[V];
      pa[i].get(u);
      if (b) {
        pb[i].get(w);
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] += w[j];
        pa[i].set(u);
        pa[i].get(u);                        // the sum as it is stored
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ss = fmaf(u[j], u[j], ss);
    }
    ss = row_sum<WARPS>(ss, red, group, parity);
    parity ^= 1;
    const float rs = rsqrtf(ss * inv + eps);
    if (slot == 0 && rstd) rstd[row] = rs;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * WARPS * 32 + slot) * V;
      if (c < cols) {
        if (b && xsum) pa[i].store(xsum + base + c);
        float u[V], g[V];
        Piece<T, V> pg;
        pg.load(gamma + c);
        pg.get(g);
        pa[i].get(u);
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = u[j] * rs * g[j];
        pa[i].set(u);
        pa[i].store(y + base + c);
      }
    }
  }
}

__device__ __forceinline__ uint32_t smem_place(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes from global to shared memory while the thread goes on; the end of a group of them; the wait for all but the latest LEFT groups
__device__ __forceinline__ void rms_fetch(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void rms_fetch_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void rms_fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Pieces of 16 bytes come through shared memory, each thread's own: the next row is under way while this one is reduced and written, without a
// barrier among threads or registers for it.  32768 x 2048 bf16: 92 us with the fold, 102 with loads into registers; 8192 x 4096: 51
// and 62; 2048 x 8192: 34 and 41; two rows ahead: the same within 2 %.
template <int V, int N, int WARPS>
constexpr size_t rms_bwd_smem() { return V == 1 ? 0 : (size_t)2 * N * 3 * 16 * rms_threads(WARPS); }

// dh may be dy or dsum.  `partial`: [gridDim.x][cols]
template <typename T, int V, int N, int WARPS>
__global__ void __launch_bounds__(rms_threads(WARPS)) rms_bwd_kernel(const T *dy, const T *h, const T *gamma, const float *rstd, const T *dsum, T *dh,
                                                      float *__restrict__ partial, int rows, int cols) {
  pdl_entry(dh);
  __shared__ float red[2 * rms_threads(WARPS) / 32];
  extern __shared__ float4 rms_smem[];       // pieces on their way; then (several rows a block) its sum of dgamma, [cols]
  float *part = reinterpret_cast<float *>(rms_smem);
  constexpr int GROUPS = rms_threads(WARPS) / (WARPS * 32);
  const int slot = threadIdx.x % (WARPS * 32), group = threadIdx.x / (WARPS * 32);
  const float inv = 1.f / (float)cols;
  float acc[N][V];
  Piece<T, V> pg[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * WARPS * 32 + slot) * V;
    pg[i].zero();
    if (c < cols) pg[i].load(gamma + c);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[i][j] = 0.f;
  }
  int parity = 0;
  const long long step = (long long)gridDim.x * GROUPS;
  long long row = (long long)blockIdx.x * GROUPS + group;
  constexpr int THREADS = rms_threads(WARPS);
  int stage = 0;
  float rs_next = 0.f;
  // place of piece i of dy (0), h (1), dsum (2)
  auto place = [&](int at, int i, int what) { return ((at * N + i) * 3 + what) * THREADS + (int)threadIdx.x; };
  auto fetch = [&](long long r, int at) {
    if (r < rows) {
      const long long base = r * cols;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * WARPS * 32 + slot) * V;
        if (c < cols) {
          rms_fetch(smem_place(&rms_smem[place(at, i, 0)]), dy + base + c);
          rms_fetch(smem_place(&rms_smem[place(at, i, 1)]), h + base + c);
          if (dsum) rms_fetch(smem_place(&rms_smem[place(at, i, 2)]), dsum + base + c);
        }
      }
    }
    rms_fetch_end();
  };
  auto take = [&](Piece<T, V> &to, int i, int what) { to.load(reinterpret_cast<const T *>(&rms_smem[place(stage, i, what)])); };
  if constexpr (V > 1) {
    fetch(row, 0);
    if (row < rows) rs_next = rstd[row];
  }
  for (; row < rows; row += step) {
    const long long base = row * cols;
    Piece<T, V> py[N], ph[N], ps[N];
    float rs = rs_next;
    if constexpr (V > 1) {
      if (row + step < rows) rs_next = rstd[row + step];
      fetch(row + step, stage ^ 1);
      rms_fetch_wait<1>();
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * WARPS * 32 + slot) * V;
      py[i].zero();
      ph[i].zero();
      ps[i].zero();
      if (c < cols) {
        if constexpr (V > 1) {
          take(py[i], i, 0);
          take(ph[i], i, 1);
        } else {
          py[i].load(dy + base + c);
          ph[i].load(h + base + c);
          if (dsum) ps[i].load(dsum + base + c);
        }
      }
    }
    if constexpr (V == 1) rs = rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float y[V], x[V], g[V];
      py[i].get(y);
      ph[i].get(x);
      pg[i].get(g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float yx = y[j] * x[j];
        dot = fmaf(yx, g[j], dot);
        acc[i][j] = fmaf(yx, rs, acc[i][j]);
      }
    }
    dot = row_sum<WARPS>(dot, red, group, parity);
    parity ^= 1;
    const float k = dot * inv * rs * rs;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * WARPS * 32 + slot) * V;
      if (c < cols) {
        float y[V], x[V], g[V], s[V];
        if constexpr (V > 1) {            // again: registers for them would cost resident blocks
          take(py[i], i, 0);
          take(ph[i], i, 1);
          if (dsum) take(ps[i], i, 2);
        }
        py[i].get(y);
        ph[i].get(x);
        pg[i].get(g);
        ps[i].get(s);
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = fmaf(rs, fmaf(y[j], g[j], -x[j] * k), s[j]);
        py[i].set(y);
        py[i].store(dh + base + c);
      }
    }
    stage ^= 1;
  }
  if constexpr (V > 1) rms_fetch_wait<0>();
  if (!partial) return;
  float *out = partial + (long long)blockIdx.x * cols;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * WARPS * 32 + slot) * V;
      if (c < cols) {
#pragma unroll
        for (int j = 0; j < V; ++j) out[c + j] = acc[i][j];
      }
    }
  } else {
    // the groups add up their columns one after the other, where their pieces were
    __syncthreads();
    for (int w = 0; w < GROUPS; ++w) {
      if (group == w) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = (i * WARPS * 32 + slot) * V;
          if (c < cols) {
#pragma unroll
            for (int j = 0; j < V; ++j) part[c + j] = w == 0 ? acc[i][j] : part[c + j] + acc[i][j];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += blockDim.x) out[c] = part[c];
  }
}

// dgamma (+)= column sums of the `parts` partial rows, in their order: 32 columns a block, 128 threads of four columns (or one, STEP 1) down the
// rows, so that the loads of a thousand partial rows are under way at once (a thread per column: 12 us for 888 x 2048)
template <typename T, int STEP>
__global__ void __launch_bounds__(1024) rms_fold_kernel(const float *partial, int parts, int cols, T *dgamma, int accumulate) {
  pdl_entry(dgamma);
  constexpr int LANES = 32 / STEP, DOWN = 1024 / LANES;
  __shared__ float sum[DOWN][33];
  const int x = threadIdx.x % LANES, y = threadIdx.x / LANES;
  const int c = blockIdx.x * 32 + x * STEP;
  float s[STEP];
#pragma unroll
  for (int j = 0; j < STEP; ++j) s[j] = 0.f;
  if (c < cols) {
    const float *from = partial + c;
    int p = y;
    for (; p + 7 * DOWN < parts; p += 8 * DOWN) {
      float v[8][STEP];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float *q = from + (long long)(p + k * DOWN) * cols;
        if constexpr (STEP == 4) {
          const float4 u = *reinterpret_cast<const float4 *>(q);
          v[k][0] = u.x; v[k][1] = u.y; v[k][2] = u.z; v[k][3] = u.w;
        } else {
          v[k][0] = *q;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < STEP; ++j) s[j] += v[k][j];
    }
#pragma unroll 4
    for (; p < parts; p += DOWN)
#pragma unroll
      for (int j = 0; j < STEP; ++j) s[j] += from[(long long)p * cols + j];
  }
#pragma unroll
  for (int j = 0; j < STEP; ++j) sum[y][x * STEP + j] = s[j];
  __syncthreads();
  // a warp per column, its lanes down the rows
  const int col = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < DOWN / 32; ++k) t += sum[k * 32 + lane][col];
  t = warp_sum(t);
  const int out = blockIdx.x * 32 + col;
  if (lane == 0 && out < cols) {
    if (accumulate) t += rms_ld(dgamma + out);
    rms_st(dgamma + out, t);
  }
}

// ---- rows too wide for registers: a block per row, two passes
template <typename T>
__global__ void __launch_bounds__(512) rms_fwd_wide_kernel(const T *a, const T *b, const T *gamma, T *xsum, T *y, float *__restrict__ rstd, int rows,
                                                           int cols, float eps) {
  pdl_entry(xsum, y);
  __shared__ float red[32];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long long base = row * cols;
    float ss = 0.f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float v = b ? rms_round(rms_ld(a + base + c) + rms_ld(b + base + c), a) : rms_ld(a + base + c);
      ss = fmaf(v, v, ss);
    }
    ss = block_sum(ss, red);
    const float rs = rsqrtf(ss / (float)cols + eps);
    if (threadIdx.x == 0 && rstd) rstd[row] = rs;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float v = b ? rms_round(rms_ld(a + base + c) + rms_ld(b + base + c), a) : rms_ld(a + base + c);
      if (b && xsum) rms_st(xsum + base + c, v);
      rms_st(y + base + c, v * rs * rms_ld(gamma + c));
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(512) rms_bwd_wide_kernel(const T *dy, const T *h, const T *gamma, const float *rstd, const T *dsum, T *dh,
                                                           float *partial, int rows, int cols) {
  pdl_entry(dh, partial);
  __shared__ float red[32];
  float *out = partial ? partial + (long long)blockIdx.x * cols : nullptr;
  bool first = true;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, first = false) {
    const long long base = row * cols;
    float dot = 0.f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) dot = fmaf(rms_ld(dy + base + c) * rms_ld(h + base + c), rms_ld(gamma + c), dot);
    dot = block_sum(dot, red);
    const float rs = rstd[row], k = dot / (float)cols * rs * rs;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float y = rms_ld(dy + base + c), x = rms_ld(h + base + c);
      const float s = dsum ? rms_ld(dsum + base + c) : 0.f;
      if (out) out[c] = (first ? 0.f : out[c]) + y * x * rs;      // a column belongs to one thread of the block
      rms_st(dh + base + c, fmaf(rs, fmaf(y, rms_ld(gamma + c), -x * k), s));
    }
    __syncthreads();
  }
}

// How a row is spread: elements of a piece, warps, pieces of a thread (0: too wide for registers)
struct RmsForm { int v, warps, n; };
RmsForm rms_form(int cols, int es, bool whole) {
  const int v = whole && cols % (16 / es) == 0 ? 16 / es : 1;
  const int pieces = (cols + v * 32 - 1) / (v * 32);       // of a warp
  const int most_warps = v == 1 ? 8 : 16, most = v == 1 ? 8 : 4;       // single elements: fewer threads with more of them
  RmsForm f = {v, 1, 1};
  while (f.warps < most_warps && f.warps < pieces) f.warps *= 2;
  while (f.n < most && f.warps * f.n < pieces) f.n *= 2;
  if (f.warps * f.n < pieces) f.n = 0;
  return f;
}
int rms_fwd_grid(const RmsForm &f, int rows, int &threads) {
  if (f.n == 0) { threads = 512; return rows < 148 * 4 ? rows : 148 * 4; }
  // few rows: one a block, so that they spread over the SMs
  threads = rows >= 148 * 8 ? rms_threads(f.warps) : f.warps * 32;
  const int per = threads / (f.warps * 32), want = (rows + per - 1) / per;
  return want < 148 * 8 ? want : 148 * 8;
}
// backward's blocks stay for their rows: as many as are resident at once, at most RMS_BWD_PER_SM per SM of single elements; of whole pieces half
// of that, which the row ahead keeps busy (32768 x 2048 bf16: 92 us with 4, 97 with 6, 114 with 2; 4004 x 1001 fp32: 18.5 with 8, 20 with 4)
constexpr int RMS_BWD_PER_SM = 8;
int rms_bwd_grid(const RmsForm &f, int rows, int per_sm) {
  const int at_most = f.v > 1 ? RMS_BWD_PER_SM / 2 : RMS_BWD_PER_SM;
  if (per_sm > at_most) per_sm = at_most;
  const int groups = f.n == 0 ? 1 : rms_threads(f.warps) / (f.warps * 32);
  const int want = (rows + groups - 1) / groups, most = 148 * (per_sm < 1 ? 1 : per_sm);
  return want < most ? want : most;
}
template <typename K>
int rms_resident(K kernel, int threads, size_t smem) {
  int n = 0;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) == cudaSuccess ? n : 1;
}
// steps of a loop past the end of rows or columns stay within 32 bits
bool rms_sizes_ok(int rows, int cols) { return rows <= 0x7fffffff - 4096 && cols <= (1 << 30); }
bool rms_aligned(const void *p) { return (((uintptr_t)p) & 15) == 0; }

template <typename T, int V, int N, int WARPS>
int rms_fwd_run(const void *a, const void *b, const void *gamma, void *xsum, void *y, float *rstd, int rows, int cols, float eps, int grid, int threads,
                cudaStream_t st) {
  return ffk_launch(rms_fwd_kernel<T, V, N, WARPS>, grid, threads, 0, st, (const T *)a, (const T *)b, (const T *)gamma, (T *)xsum, (T *)y, rstd, rows,
                    cols, eps);
}
template <typename T, int V, int N, int WARPS>
int rms_bwd_run(const void *dy, const void *h, const void *gamma, const float *rstd, const void *dsum, void *dh, float *partial, int rows, int cols,
                int &grid, cudaStream_t st) {
  constexpr int threads = rms_threads(WARPS);
  constexpr bool several = threads > WARPS * 32;
  constexpr size_t sums = several ? (size_t)V * N * WARPS * 128 : 0, smem = sums > rms_bwd_smem<V, N, WARPS>() ? sums : rms_bwd_smem<V, N, WARPS>();
  static unsigned long long done = 0;
  const cudaError_t e = ffk_allow_smem(rms_bwd_kernel<T, V, N, WARPS>, (int)smem, done);
  if (e != cudaSuccess) return (int)e;
  static const int per_sm = rms_resident(rms_bwd_kernel<T, V, N, WARPS>, threads, smem);
  grid = rms_bwd_grid({V, WARPS, N}, rows, per_sm);
  return ffk_launch(rms_bwd_kernel<T, V, N, WARPS>, grid, threads, smem, st, (const T *)dy, (const T *)h, (const T *)gamma,
                    rstd, (const T *)dsum, (T *)dh, partial, rows, cols);
}
#define RMS_FORMS(RUN, T, V, ...)                            \
  switch (f.warps * f.n) {                                  \
    case 1: return RUN<T, V, 1, 1>(__VA_ARGS__);            \
    case 2: return RUN<T, V, 1, 2>(__VA_ARGS__);            \
    case 4: return RUN<T, V, 1, 4>(__VA_ARGS__);            \
    case 8: return RUN<T, V, 1, 8>(__VA_ARGS__);            \
    case 16: return RUN<T, V, V == 1 ? 2 : 1, V == 1 ? 8 : 16>(__VA_ARGS__); \
    case 32: return RUN<T, V, V == 1 ? 4 : 2, V == 1 ? 8 : 16>(__VA_ARGS__); \
    default: return RUN<T, V, V == 1 ? 8 : 4, V == 1 ? 8 : 16>(__VA_ARGS__); \
  }

template <typename T, int WHOLE>
int rms_fwd_typed(const RmsForm &f, const void *a, const void *b, const void *gamma, void *xsum, void *y, float *rstd, int rows, int cols, float eps,
                  int grid, int threads, cudaStream_t st) {
  if (f.n == 0)
    return ffk_launch(rms_fwd_wide_kernel<T>, grid, threads, 0, st, (const T *)a, (const T *)b, (const T *)gamma, (T *)xsum, (T *)y, rstd, rows, cols, eps);
  if (f.v == 1) { RMS_FORMS(rms_fwd_run, T, 1, a, b, gamma, xsum, y, rstd, rows, cols, eps, grid, threads, st) }
  RMS_FORMS(rms_fwd_run, T, WHOLE, a, b, gamma, xsum, y, rstd, rows, cols, eps, grid, threads, st)
}
template <typename T, int WHOLE>
int rms_bwd_typed(const RmsForm &f, const void *dy, const void *h, const void *gamma, const float *rstd, const void *dsum, void *dh, float *partial,
                  int rows, int cols, int &grid, cudaStream_t st) {
  if (f.n == 0) grid = rms_bwd_grid(f, rows, 2);
  if (f.n == 0)
    return ffk_launch(rms_bwd_wide_kernel<T>, grid, 512, 0, st, (const T *)dy, (const T *)h, (const T *)gamma, rstd, (const T *)dsum, (T *)dh, partial,
                      rows, cols);
  if (f.v == 1) { RMS_FORMS(rms_bwd_run, T, 1, dy, h, gamma, rstd, dsum, dh, partial, rows, cols, grid, st) }
  RMS_FORMS(rms_bwd_run, T, WHOLE, dy, h, gamma, rstd, dsum, dh, partial, rows, cols, grid, st)
}

}  // namespace

// dt: 0 fp32, 1 bf16 (gamma too).  b, xsum, rstd may be null; b is the residual, xsum receives a + b.
FFK_API int ffk_rmsnorm_fwd(const void *a, const void *b, const void *gamma, void *xsum, void *y, float *rstd, int rows, int cols, float eps, int dt,
                            cudaStream_t st) {
  if (dt != 0 && dt != 1) return -2;
  if (rows <= 0) return 0;
  if (cols <= 0 || !rms_sizes_ok(rows, cols)) return -2;
  const int es = dt == 1 ? 2 : 4;
  FfkTraffic traffic((long long)rows * cols * es * (b ? xsum ? 4 : 3 : 2));
  const RmsForm f = rms_form(cols, es, rms_aligned(a) && rms_aligned(b) && rms_aligned(gamma) && rms_aligned(xsum) && rms_aligned(y));
  int threads = 0;
  const int grid = rms_fwd_grid(f, rows, threads);
  return dt == 1 ? rms_fwd_typed<bf16, 8>(f, a, b, gamma, xsum, y, rstd, rows, cols, eps, grid, threads, st)
                 : rms_fwd_typed<float, 4>(f, a, b, gamma, xsum, y, rstd, rows, cols, eps, grid, threads, st);
}

// floats of scratch: the partial rows of dgamma, for either form of the addresses
FFK_API long long ffk_rmsnorm_bwd_scratch(int rows, int cols) {
  if (rows <= 0 || cols <= 0 || !rms_sizes_ok(rows, cols)) return 0;
  long long most = 0;
  for (int es = 2; es <= 4; es += 2)
    for (int whole = 0; whole < 2; ++whole) {
      const long long g = rms_bwd_grid(rms_form(cols, es, whole), rows, RMS_BWD_PER_SM);
      most = g > most ? g : most;
    }
  return most * cols;
}

// dsum, dgamma and (without dgamma) partial may be null
FFK_API int ffk_rmsnorm_bwd(const void *dy, const void *h, const void *gamma, const float *rstd, const void *dsum, void *dh, void *dgamma, float *partial,
                            int rows, int cols, int dt, int accumulate_params, cudaStream_t st) {
  if (dt != 0 && dt != 1) return -2;
  if (cols <= 0) return rows <= 0 ? 0 : -2;
  if (!rms_sizes_ok(rows, cols)) return -2;
  const int es = dt == 1 ? 2 : 4;
  int grid = 0;
  if (dgamma && rows > 0 && !partial) return -2;
  if (rows > 0) {
    FfkTraffic traffic((long long)rows * cols * es * (dsum ? 4 : 3));
    const RmsForm f = rms_form(cols, es, rms_aligned(dy) && rms_aligned(h) && rms_aligned(gamma) && rms_aligned(dsum) && rms_aligned(dh));
    float *part = dgamma ? partial : nullptr;
    const int e = dt == 1 ? rms_bwd_typed<bf16, 8>(f, dy, h, gamma, rstd, dsum, dh, part, rows, cols, grid, st)
                          : rms_bwd_typed<float, 4>(f, dy, h, gamma, rstd, dsum, dh, part, rows, cols, grid, st);
    if (e) return e;
  }
  if (!dgamma) return 0;
  const bool four = cols % 4 == 0 && rms_aligned(partial);
  const unsigned blocks = (unsigned)(cols + 31) / 32;
  if (dt == 1)
    return four ? ffk_launch(rms_fold_kernel<bf16, 4>, blocks, 1024, 0, st, partial, grid, cols, (bf16 *)dgamma, accumulate_params)
                : ffk_launch(rms_fold_kernel<bf16, 1>, blocks, 1024, 0, st, partial, grid, cols, (bf16 *)dgamma, accumulate_params);
  return four ? ffk_launch(rms_fold_kernel<float, 4>, blocks, 1024, 0, st, partial, grid, cols, (float *)dgamma, accumulate_params)
              : ffk_launch(rms_fold_kernel<float, 1>, blocks, 1024, 0, st, partial, grid, cols, (float *)dgamma, accumulate_params);
}
