// grad_norm.cu -- the norm of many gradient tensors taken as one vector, and clipping by it.
//
//   n = sqrt(sum over all tensors and elements of g^2),   g <- g * min(1, max_norm / n)
//
// The tensors are cut into pieces of PIECE elements, listed in device memory once when the list is made (address, destination, length,
// type); a block takes pieces in steps of the grid.  Squares of one 16-byte vector are added in 32 bits, vectors in 64: that costs one
// conversion and one 64-bit addition per vector and keeps the sum of 1e9 elements exact to a few 1e-8.  A vector whose squares leave the
// range of 32 bits (elements beyond 1e18, or below 1e-16 and not zero, infinities, NaN) is squared in 64 bits.  Each block leaves one partial
// sum; whoever needs the norm adds the partial sums in their fixed order, so the result does not depend on which block came first, and there
// is no counter to reset.  The clipping kernel's blocks each add them up (at most 1184 numbers from L2), which saves a launch between the
// passes.  A clipped element is rounded once, when it is stored.
//
// What bounds it: HBM, read once for the norm and read again and written for the clipping.  The second pass goes over the pieces in the
// opposite order: it begins with what the first left in L2.  403 million bf16 elements (805 MB) in the tensors of eight layers of width 2048:
// norm 114 us (7.1 TB/s, reads only), with the clipping 385 us (three passes over the gradients at the copy rate: 370); 6.3 million fp32
// elements: 20 us.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int PIECE = 16384;            // elements of a piece at most
constexpr int PIECE_LEAST = 1024;
constexpr int NORM_BLOCKS = 148 * 8;    // partial sums at most
constexpr int NORM_THREADS = 256;
constexpr int NORM_UNROLL = 8;          // 16-byte loads of a thread under way
constexpr long long NORM_KEEP = 80ll << 20;   // bytes of the gradients that stay in L2 (126 MB) between the passes

struct GradPiece {
  const void *src;
  void *dst;
  int n;
  int dt;                               // 0 fp32, 1 bf16, 4 fp16
};

template <typename T> struct GradVec;
template <> struct GradVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ float one(const float *p) { return *p; }
  static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
};
template <> struct GradVec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
    const float2 a = unpack_bf162(u.x), b = unpack_bf162(u.y), c = unpack_bf162(u.z), d = unpack_bf162(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf162(v[0], v[1]), pack_bf162(v[2], v[3]), pack_bf162(v[4], v[5]), pack_bf162(v[6], v[7]));
  }
  static __device__ __forceinline__ float one(const bf16 *p) { return bf2f(*p); }
  static __device__ __forceinline__ void put(bf16 *p, float v) { *p = f2bf(v); }
};
template <> struct GradVec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float2 two(uint32_t u) { return __half22float2(*reinterpret_cast<__half2 *>(&u)); }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
    const float2 a = two(u.x), b = two(u.y), c = two(u.z), d = two(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(two(v[0], v[1]), two(v[2], v[3]), two(v[4], v[5]), two(v[6], v[7]));
  }
  static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
  static __device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
};

// the sum of squares of one vector, in 64 bits where 32 do not hold it
template <int N>
__device__ __forceinline__ double squares(const float (&v)[N]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(v[i], v[i], s);
  if (s <= 1e36f && s >= 1e-32f) return (double)s;
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) bits |= __float_as_uint(v[i]) << 1;
  if (bits == 0) return 0.0;
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) t = fma((double)v[i], (double)v[i], t);
  return t;
}

template <typename T>
__device__ __forceinline__ double piece_squares(const T *p, int n, bool stream) {
  constexpr int N = GradVec<T>::N;
  double sum = 0.0;
  if ((((uintptr_t)p) & 15) == 0) {
    const int whole = n / N;
    const uint4 *q = reinterpret_cast<const uint4 *>(p);
    int i = threadIdx.x;
    for (; i + (NORM_UNROLL - 1) * NORM_THREADS < whole; i += NORM_UNROLL * NORM_THREADS) {
      uint4 u[NORM_UNROLL];
#pragma unroll
      for (int k = 0; k < NORM_UNROLL; ++k) u[k] = stream ? __ldcs(q + i + k * NORM_THREADS) : q[i + k * NORM_THREADS];
#pragma unroll
      for (int k = 0; k < NORM_UNROLL; ++k) {
        float v[N];
        GradVec<T>::unpack(u[k], v);
        sum += squares(v);
      }
    }
    for (; i < whole; i += NORM_THREADS) {
      float v[N];
      GradVec<T>::unpack(q[i], v);
      sum += squares(v);
    }
    const int rest = whole * N + (int)threadIdx.x;
    if (rest < n) {
      const double x = GradVec<T>::one(p + rest);
      sum = fma(x, x, sum);
    }
  } else {
    for (int i = threadIdx.x; i < n; i += NORM_THREADS) {
      const float v[1] = {GradVec<T>::one(p + i)};
      sum += squares(v);
    }
  }
  return sum;
}

// block-wide sum in a fixed order; every thread gets it
__device__ __forceinline__ double block_sum_wide(double v, double *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < NORM_THREADS / 32; ++w) t += red[w];
  return t;
}

__global__ void __launch_bounds__(NORM_THREADS) grad_squares_kernel(const GradPiece *pieces, int count, int keep, double *__restrict__ partial) {
  pdl_entry();
  __shared__ double red[NORM_THREADS / 32];
  double sum = 0.0;
  // the last `keep` pieces are left in L2 for the clipping, which begins with them; the others stream past it
  GradPiece next = {};
  if ((int)blockIdx.x < count) next = pieces[blockIdx.x];
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const GradPiece g = next;
    if (c + (int)gridDim.x < count) next = pieces[c + gridDim.x];      // the next entry comes in under this piece's loads
    if (g.dt == 1) sum += piece_squares((const bf16 *)g.src, g.n, c < count - keep);
    else if (g.dt == 0) sum += piece_squares((const float *)g.src, g.n, c < count - keep);
    else sum += piece_squares((const __half *)g.src, g.n, c < count - keep);
  }
  sum = block_sum_wide(sum, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ double folded_norm(const double *partial, int blocks, double *red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < blocks; i += NORM_THREADS) v += partial[i];
  return sqrt(block_sum_wide(v, red));
}

__global__ void __launch_bounds__(NORM_THREADS) grad_norm_kernel(const double *partial, int blocks, float *__restrict__ norm) {
  pdl_entry();
  __shared__ double red[NORM_THREADS / 32];
  const double n = folded_norm(partial, blocks, red);
  if (threadIdx.x == 0) *norm = (float)n;
}

// `over`: multiplied by f; otherwise a copy, bit by bit
template <typename T>
__device__ __forceinline__ uint4 scaled(uint4 u, bool over, float f) {
  if (!over) return u;
  float v[GradVec<T>::N];
  GradVec<T>::unpack(u, v);
#pragma unroll
  for (int j = 0; j < GradVec<T>::N; ++j) v[j] *= f;
  return GradVec<T>::pack(v);
}
template <typename T>
__device__ __forceinline__ void piece_scale(const T *src, T *dst, int n, bool over, float f) {
  constexpr int N = GradVec<T>::N;
  if (((((uintptr_t)src) | ((uintptr_t)dst)) & 15) == 0) {
    const int whole = n / N;
    const uint4 *q = reinterpret_cast<const uint4 *>(src);
    uint4 *o = reinterpret_cast<uint4 *>(dst);
    int i = threadIdx.x;
    for (; i + (NORM_UNROLL - 1) * NORM_THREADS < whole; i += NORM_UNROLL * NORM_THREADS) {
      uint4 u[NORM_UNROLL];
#pragma unroll
      for (int k = 0; k < NORM_UNROLL; ++k) u[k] = q[i + k * NORM_THREADS];
#pragma unroll
      for (int k = 0; k < NORM_UNROLL; ++k) o[i + k * NORM_THREADS] = scaled<T>(u[k], over, f);
    }
    for (; i < whole; i += NORM_THREADS) o[i] = scaled<T>(q[i], over, f);
    const int rest = whole * N + (int)threadIdx.x;
    if (rest < n) {
      if (over) GradVec<T>::put(dst + rest, GradVec<T>::one(src + rest) * f);
      else dst[rest] = src[rest];
    }
  } else {
    for (int i = threadIdx.x; i < n; i += NORM_THREADS) {
      if (over) GradVec<T>::put(dst + i, GradVec<T>::one(src + i) * f);
      else dst[i] = src[i];
    }
  }
}

// A norm that is not above max_norm, or not finite, leaves the gradients as they are (in place: nothing is read).
__global__ void __launch_bounds__(NORM_THREADS) grad_clip_kernel(const GradPiece *pieces, int count, const double *partial, int blocks, float max_norm,
                                                                 float *__restrict__ norm) {
  pdl_entry();
  __shared__ double red[NORM_THREADS / 32];
  GradPiece next = {};
  if (count - 1 - (int)blockIdx.x >= 0) next = pieces[count - 1 - (int)blockIdx.x];
  const double n = folded_norm(partial, blocks, red);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const bool over = n > (double)max_norm && n <= 1.7e308;
  const float f = over ? (float)((double)max_norm / n) : 1.f;
  for (int c = count - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const GradPiece g = next;
    if (c - (int)gridDim.x >= 0) next = pieces[c - gridDim.x];
    if (!over && g.src == g.dst) continue;
    if (g.dt == 1) piece_scale((const bf16 *)g.src, (bf16 *)g.dst, g.n, over, f);
    else if (g.dt == 0) piece_scale((const float *)g.src, (float *)g.dst, g.n, over, f);
    else piece_scale((const __half *)g.src, (__half *)g.dst, g.n, over, f);
  }
}

int norm_blocks(int count) { return count < 1 ? 1 : count < NORM_BLOCKS ? count : NORM_BLOCKS; }

}  // namespace

// elements of a piece of a list of `total`: two pieces a block, where that leaves them long enough to be worth their table entry
FFK_API int ffk_grad_piece_elements(long long total) {
  const long long n = (total / (2 * NORM_BLOCKS) + PIECE_LEAST - 1) / PIECE_LEAST * PIECE_LEAST;
  return (int)(n < PIECE_LEAST ? PIECE_LEAST : n > PIECE ? PIECE : n);
}
FFK_API int ffk_grad_partials() { return NORM_BLOCKS; }

// pieces: `count` GradPiece in device memory; partial: ffk_grad_partials() doubles of scratch; norm: one float
FFK_API int ffk_grad_norm(const void *pieces, int count, double *partial, float *norm, long long bytes, cudaStream_t st) {
  const int blocks = norm_blocks(count);
  FfkTraffic traffic(bytes);
  int e = ffk_launch(grad_squares_kernel, blocks, NORM_THREADS, 0, st, (const GradPiece *)pieces, count, 0, partial);
  traffic.done();
  if (e) return e;
  return ffk_launch(grad_norm_kernel, 1, NORM_THREADS, 0, st, partial, blocks, norm);
}

FFK_API int ffk_grad_clip(const void *pieces, int count, double *partial, float max_norm, float *norm, long long bytes, cudaStream_t st) {
  const int blocks = norm_blocks(count);
  FfkTraffic traffic(2 * bytes);
  const int keep = bytes <= NORM_KEEP ? count : (int)((double)NORM_KEEP / (double)bytes * count);
  int e = ffk_launch(grad_squares_kernel, blocks, NORM_THREADS, 0, st, (const GradPiece *)pieces, count, keep, partial);
  if (e) return e;
  return ffk_launch(grad_clip_kernel, blocks, NORM_THREADS, 0, st, (const GradPiece *)pieces, count, partial, blocks, max_norm, norm);
}
