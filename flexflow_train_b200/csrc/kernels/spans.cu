// spans.cu -- first and last visible key of every token of a batch of packed documents.
//
// A document is a run of equal numbers in a row of `documents`; tokens with a negative number are padding.  For token t of the run
// [a, e] (a, e its first and last token) and f = number of flagged tokens that the run begins with:
//   low = a,   high = causal ? max(t, a + f - 1) : e;     padding: low = 0, high = -1 (an empty span).
// So every mask of attention over packed sequences (causal, document, prefix, padding, and any product of them) is one interval per
// query, 8 bytes a token instead of a row of flags.
//
// What bounds it: launch and load latency (12 bytes a token).  A block takes SEG tokens of one row; what it needs of the rest of the row
// is one number each -- where the run at its first token began, where the run at its last token ends, where that run's flags end -- and
// the block looks for those by itself, in steps of its width, so blocks share nothing and there is one launch and no scratch.
// 8 x 256: 1.7 us; 16 x 16384 in documents of about 1500 with prompts: 8.7 us, of which two searches of up to 2048 places each way.
#include "common.cuh"

namespace {

constexpr int SPAN_THREADS = 256;
constexpr int SPAN_PER = 4;
constexpr int SEG = SPAN_THREADS * SPAN_PER;

// The largest i < `from` with test(i), or `none`: the block looks at LOOK places at a time, going down; all threads get it.  Its loads do not
// depend on one another, so a run of thousands of tokens costs a few latencies.
constexpr int LOOK_PER = 8;
constexpr int LOOK = SPAN_THREADS * LOOK_PER;
template <typename F>
__device__ __forceinline__ int block_find_down(int from, int none, int *slots, F test) {
  for (int hi = from; hi > 0; hi -= LOOK) {
    int best = -1;
#pragma unroll
    for (int k = 0; k < LOOK_PER; ++k) {
      const int i = hi - 1 - k * SPAN_THREADS - (int)threadIdx.x;
      best = max(best, test(max(i, 0)) ? i : -1);                  // no branch around the loads: they all start at once
    }
    best = __reduce_max_sync(0xffffffffu, best);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SPAN_THREADS / 32; ++w) best = max(best, slots[w]);
    if (best >= 0) return best;
  }
  return none;
}
// The smallest i >= `from` (and < n) with test(i), or n.
template <typename F>
__device__ __forceinline__ int block_find_up(int from, int n, int *slots, F test) {
  for (int lo = from; lo < n; lo += LOOK) {
    int best = n;
#pragma unroll
    for (int k = 0; k < LOOK_PER; ++k) {
      const int i = lo + k * SPAN_THREADS + (int)threadIdx.x;
      const bool hit = test(min(i, n - 1));
      if (hit & (i < n)) best = min(best, i);
    }
    best = __reduce_min_sync(0xffffffffu, best);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SPAN_THREADS / 32; ++w) best = min(best, slots[w]);
    if (best < n) return best;
  }
  return n;
}

__global__ void __launch_bounds__(SPAN_THREADS) attention_spans_kernel(const int *documents, const unsigned char *prompt, int2 *__restrict__ spans, int S,
                                                                       int segments, int causal) {
  pdl_entry();
  __shared__ int scan[SPAN_THREADS / 32];
  __shared__ int stops[SEG];
  __shared__ int slot[SPAN_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / segments;
  const int s0 = (int)(blockIdx.x % segments) * SEG;
  const int s1 = min(s0 + SEG, S);
  const int *doc = documents + row * S;
  const unsigned char *flag = prompt ? prompt + row * S : nullptr;
  const bool flags = causal && flag;
  auto opens = [&](int i) { return (doc[i] != doc[max(i - 1, 0)]) | (i == 0); };   // i begins a run
  auto ends_prompt = [&](int i) { return flag[i] == 0; };

  // four consecutive tokens a thread
  const int t0 = s0 + tid * SPAN_PER;
  int d[SPAN_PER + 2];                       // with the neighbours on either side
#pragma unroll
  for (int j = 0; j < SPAN_PER + 2; ++j) {
    const int t = t0 - 1 + j;
    d[j] = t >= 0 && t < S ? doc[t] : 0;
  }
  int start[SPAN_PER];
  bool last[SPAN_PER];
#pragma unroll
  for (int j = 0; j < SPAN_PER; ++j) {
    const int t = t0 + j;
    start[j] = t < s1 && (t == 0 || d[j + 1] != d[j]) ? t : -1;
    last[j] = t >= S - 1 || d[j + 2] != d[j + 1];
  }
  // low: running maximum of the run starts, over the thread, the warp, the block; what lies before the segment where none is in it
  int mine = max(max(start[0], start[1]), max(start[2], start[3]));
  int up = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up = max(up, v);
  }
  if (lane == 31) scan[warp] = up;
  int before = __shfl_up_sync(0xffffffffu, up, 1);
  if (lane == 0) before = -1;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before = max(before, scan[w]);
  const int first = opens(s0) ? s0 : block_find_down(s0, 0, slot, opens);      // start of the run that s0 belongs to
  int low[SPAN_PER];
  int run = max(before, first);
#pragma unroll
  for (int j = 0; j < SPAN_PER; ++j) {
    run = max(run, start[j]);
    low[j] = run;
  }
  int high[SPAN_PER];
  if (causal && !flags) {
#pragma unroll
    for (int j = 0; j < SPAN_PER; ++j) high[j] = t0 + j;
  } else {
    // running minimum from the right: of the runs' last tokens, or (causal with prompts) of the places where the flags of a run that is
    // flagged up to there end: the first token that is not flagged, or the one behind the run
    int stop[SPAN_PER];
#pragma unroll
    for (int j = 0; j < SPAN_PER; ++j) {
      const int t = t0 + j;
      if (t >= s1) stop[j] = 0x7fffffff;
      else if (flags) stop[j] = flag[t] == 0 ? t : last[j] ? t + 1 : 0x7fffffff;
      else stop[j] = last[j] ? t : 0x7fffffff;
    }
    int down = min(min(stop[0], stop[1]), min(stop[2], stop[3]));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_down_sync(0xffffffffu, down, o);
      if (lane + o < 32) down = min(down, v);
    }
    __syncthreads();
    if (lane == 0) scan[warp] = down;
    int after = __shfl_down_sync(0xffffffffu, down, 1);
    if (lane == 31) after = 0x7fffffff;
    __syncthreads();
    for (int w = warp + 1; w < SPAN_THREADS / 32; ++w) after = min(after, scan[w]);
    // the first such place behind the segment: the run of its last token may go on there
    int beyond;
    if (s1 >= S || opens(s1)) beyond = flags ? s1 : s1 - 1;
    else if (flags) beyond = block_find_up(s1, S, slot, [&](int i) { return opens(i) | ends_prompt(i); });
    else beyond = block_find_up(s1, S, slot, opens) - 1;
    run = min(after, beyond);
    int back[SPAN_PER];
#pragma unroll
    for (int j = SPAN_PER - 1; j >= 0; --j) {
      run = min(run, stop[j]);
      back[j] = run;
    }
    if (flags) {
      // the flags' end of each run, read where the run begins; for the run that came into the segment, looked for from its own start
#pragma unroll
      for (int j = 0; j < SPAN_PER; ++j) stops[tid * SPAN_PER + j] = back[j];
      int came = first;
      if (first < s0) came = block_find_up(first, s1, slot, [&](int i) { return (opens(i) & (i > first)) | ends_prompt(i); });
      if (first < s0 && came == s1) came = beyond;       // flagged throughout: as far as it goes behind the segment
      __syncthreads();
#pragma unroll
      for (int j = 0; j < SPAN_PER; ++j) {
        const int f = low[j] >= s0 ? stops[low[j] - s0] : came;
        high[j] = max(t0 + j, f - 1);
      }
    } else {
#pragma unroll
      for (int j = 0; j < SPAN_PER; ++j) high[j] = back[j];
    }
  }
  int2 *out = spans + row * S;
#pragma unroll
  for (int j = 0; j < SPAN_PER; ++j)
    if (t0 + j < s1) out[t0 + j] = d[j + 1] < 0 ? make_int2(0, -1) : make_int2(low[j], high[j]);
}

}  // namespace

// documents: [B, S] int32; prompt: [B, S] bytes or null; spans: [B, S] pairs of int32
FFK_API int ffk_attention_spans(const int *documents, const unsigned char *prompt, int *spans, int B, int S, int causal, cudaStream_t st) {
  if (B <= 0 || S <= 0) return 0;
  if (((uintptr_t)spans) & 7) return -2;
  const long long segments = ((long long)S + SEG - 1) / SEG, grid = segments * B;
  if (grid > 0x7fffffffll || (long long)S > 0x7fffffffll - LOOK - SEG) return -2;
  FfkTraffic traffic((long long)B * S * 12);
  return ffk_launch(attention_spans_kernel, (unsigned)grid, SPAN_THREADS, 0, st, documents, prompt, (int2 *)spans, S, (int)segments, causal);
}
