// spans.cu -- first and last visible key of every token of a batch of packed documents.
//
// A document is a run of equal numbers in a row of `documents`; tokens with a negative number are padding.  For token t of the run
// [a, e] (a, e its first and last token) and f = number of flagged tokens that the run begins with:
//   low = a,   high = causal ? max(t, a + f - 1) : e;     padding: low = 0, high = -1 (an empty span).
// So every mask of attention over packed sequences (causal, document, prefix, padding, and any product of them) is one interval per
// query, 8 bytes a token instead of a row of flags.
//
// What bounds it: launch and load latency (12 bytes a token).  A block takes SEG tokens of one row; what it needs of the rest of the row
// is one number each -- where the run at its first token began, where the run at its last token ends, where that run's flags end.  In short
// rows the block looks for those by itself, so blocks share nothing and there is one launch and no scratch; in long ones it looks through
// what a launch before has written down of each segment.  8 x 256: 1.7 us; 16 x 16384 in documents of about 1500 with prompts: 8.7 us in
// a step, most of it two searches of up to 2048 places each way; 4194304 as one document: 31.
#include "common.cuh"

namespace {

constexpr int SPAN_THREADS = 256;
constexpr int SPAN_PER = 4;
// Rows of up to so many segments look for themselves.  That costs a latency per 2048 tokens of a document, the summaries a launch: 16 x 16384 in
// documents of 1500, prompts: 12.6 us against 13.8 with summaries, as one document 17.3 against 13.8; 32768 as one document, prompts: 26.5 against
// 7.2; 1048576: 2360 against 19.
constexpr int SPAN_ALONE = 16;
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

constexpr int SPAN_NONE = 0x7fffffff;

// What a segment says to the others: the last place that begins a run (-1: none), the first one, and the first that begins a run or is not
// flagged (SPAN_NONE: none).
__global__ void __launch_bounds__(SPAN_THREADS) span_segments_kernel(const int *documents, const unsigned char *prompt, int4 *summary, int S, int segments) {
  pdl_entry();
  __shared__ int4 part[SPAN_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / segments;
  const int s0 = (int)(blockIdx.x % segments) * SEG;
  const int *doc = documents + row * S;
  const unsigned char *flag = prompt ? prompt + row * S : nullptr;
  int last = -1, first = SPAN_NONE, stop = SPAN_NONE;
#pragma unroll
  for (int j = 0; j < SPAN_PER; ++j) {
    const int t = s0 + j * SPAN_THREADS + tid;
    if (t >= S) break;
    const bool opens = t == 0 || doc[t] != doc[t - 1];
    if (opens) { last = t; first = min(first, t); }
    if (opens || (flag && flag[t] == 0)) stop = min(stop, t);
  }
  last = __reduce_max_sync(0xffffffffu, last);
  first = __reduce_min_sync(0xffffffffu, first);
  stop = __reduce_min_sync(0xffffffffu, stop);
  if (lane == 0) part[warp] = make_int4(last, first, stop, 0);
  __syncthreads();
  if (tid == 0) {
    for (int w = 0; w < SPAN_THREADS / 32; ++w) { last = max(last, part[w].x); first = min(first, part[w].y); stop = min(stop, part[w].z); }
    summary[blockIdx.x] = make_int4(last, first, stop, 0);
  }
}

// SUMMED: what lies outside the segment is looked up in the segments' summaries instead of the tokens
template <bool SUMMED>
__global__ void __launch_bounds__(SPAN_THREADS) attention_spans_kernel(const int *documents, const unsigned char *prompt, const int4 *summary,
                                                                       int2 *__restrict__ spans, int S, int segments, int causal) {
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
  const int seg = s0 / SEG;
  const int4 *sum = SUMMED ? summary + row * segments : nullptr;
  int first = s0;                            // start of the run that s0 belongs to
  if (!opens(s0)) {
    if constexpr (SUMMED) first = sum[block_find_down(seg, 0, slot, [&](int i) { return sum[i].x >= 0; })].x;
    else first = block_find_down(s0, 0, slot, opens);
  }
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
    else if constexpr (SUMMED) {
      const int at = block_find_up(seg + 1, segments, slot, [&](int i) { return (flags ? sum[i].z : sum[i].y) != SPAN_NONE; });
      beyond = at == segments ? S : flags ? sum[at].z : sum[at].y;
      if (!flags) --beyond;
    } else if (flags) beyond = block_find_up(s1, S, slot, [&](int i) { return opens(i) | ends_prompt(i); });
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
      if (first < s0) {
        const int upto = SUMMED ? (first / SEG + 1) * SEG : s1;              // its own segment, then the others' summaries
        came = block_find_up(first, upto, slot, [&](int i) { return (opens(i) & (i > first)) | ends_prompt(i); });
        if (SUMMED && came == upto) {
          const int at = block_find_up(first / SEG + 1, seg + 1, slot, [&](int i) { return sum[i].z != SPAN_NONE; });
          came = at > seg ? s1 : sum[at].z;
        }
      }
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

// ints of scratch for [B, S]: none where a block looks for itself
FFK_API long long ffk_attention_spans_scratch(int B, int S) {
  const long long segments = ((long long)S + SEG - 1) / SEG;
  return B <= 0 || segments <= SPAN_ALONE ? 0 : 4 * segments * B;
}

// documents: [B, S] int32; prompt: [B, S] bytes or null; spans: [B, S] pairs of int32; scratch: on a 16-byte boundary, or null where none is needed
FFK_API int ffk_attention_spans(const int *documents, const unsigned char *prompt, int *spans, int *scratch, int B, int S, int causal, cudaStream_t st) {
  if (B <= 0 || S <= 0) return 0;
  const bool summed = ffk_attention_spans_scratch(B, S) > 0;
  if (((uintptr_t)spans) & 7 || ((uintptr_t)scratch) & 15 || (summed && !scratch)) return -2;
  const long long segments = ((long long)S + SEG - 1) / SEG, grid = segments * B;
  if (grid > 0x7fffffffll || (long long)S > 0x7fffffffll - LOOK - SEG) return -2;
  FfkTraffic traffic((long long)B * S * 12);
  if (!summed)
    return ffk_launch(attention_spans_kernel<false>, (unsigned)grid, SPAN_THREADS, 0, st, documents, prompt, (const int4 *)nullptr, (int2 *)spans, S,
                      (int)segments, causal);
  if (!causal) prompt = nullptr;
  const int r = ffk_launch(span_segments_kernel, (unsigned)grid, SPAN_THREADS, 0, st, documents, prompt, (int4 *)scratch, S, (int)segments);
  if (r) return r;
  return ffk_launch(attention_spans_kernel<true>, (unsigned)grid, SPAN_THREADS, 0, st, documents, prompt, (const int4 *)scratch, (int2 *)spans, S,
                    (int)segments, causal);
}
