// Sampling with temperature, top-k, top-p and min-p from one given uniform number per row (mllm_sample).
//
// With x the row (NaN as -inf), m its maximum and r = 1 / T, token i weighs w_i = floor(2^40 exp((x_i - m) r)).
// Tokens are ordered by falling x, ties by rising index: by the 64-bit number (key of x, ~index).  The
// tokens that top-k or top-p keep are those at or above an edge in that order, the lowest number before
// which few enough tokens (top-k) or little enough weight (top-p) lies.  The id is found in index order, at
// the place where the running kept weight passes floor(u Z).  Weights are integers of at most 2^40 (a sum
// of 2^19 of them fits 64 bits), so every sum is exact and no result depends on the order in which threads
// add.  What the whole part cuts off a weight is below 2^-40 of the top token's: over the 2^19 tokens that a row may
// have less than 2^-21 of its weight, a few f32 roundings.
//
// A row is read once, into the shared memory of one CTA, or of a cluster's CTAs, each of which has a
// contiguous part, where rows are fewer than SMs or do not fit.  The edge is found without sorting the row:
//   - top_k up to 512: the step of 1/16 of a unit of (x - m) r in which the k-th largest of the threads' own
//     maxima lies bounds the k-th token from below, so the few tokens down to that step are gathered, and
//     everything else happens in that list;
//   - otherwise by a histogram of tokens or weight over 512 such steps, then among the tokens of one step,
//     or of a 512th of it where they are too many for a list;
//   - and by halving, one pass per bit, where those are too many as well (thousands of tokens of one value).
// A short list is not sorted either: several threads per token count, and weigh, what precedes it.  One of up to
// 512 tokens is sorted in registers, for the id a second time by index (33 rows with top_p, medians of five: 37.2 us,
// by steps 38.9, with runs of either up to 2.4 apart; 256 rows 58.7 and 58.6).  A longer one goes through the same
// two levels of steps until few enough are left, for the id by steps of the index; it is sorted where one step
// holds too many.
// The CTAs of a cluster meet at a barrier only to exchange a maximum, a histogram, a list (the first one's) or
// a sum.
//
// Of a few microseconds per row much goes into fetching instructions, so the code is kept small: what runs
// once is called, not inlined, and the passes over the row either test 16 bytes at a time and do the rest
// for the few that pass, or take a token at a time.
//
// B200: 256 rows of 49,152 f32 with mixed settings 59 us, one row 14 us, 33 rows of 50,257 bf16 with top_p and
// probabilities 37 us (36 to 39).  Bound by latency where rows are few (a chain of some 20 barriers), by instruction
// issue and colliding shared-memory atomics where every token's weight goes into a histogram (about 24,000
// cycles of one SM for 49,152 tokens).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <climits>

#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleList = 2048;   // tokens of a list
constexpr int kShortList = 192;     // tokens of a list that is counted at once (the square of them)
constexpr int kSortList = 512;     // tokens of a list that is sorted in registers, one per thread
constexpr int kMiniList = 64;       // tokens of a step of a longer list
constexpr int kSampleMaxK = 512;    // top_k that starts from the threads' maxima
constexpr int kFewTokens = 4 * kSampleThreads;  // of a CTA: all are counted for top_k
constexpr int kSteps = 512;         // steps of a histogram level
constexpr int kMaxCluster = 16;
constexpr float kOne = 1099511627776.f;  // 2^40
constexpr float kFar = -31.9998779296875f;  // 1/8192 short of -32: nothing at or below weighs anything (2^-40 is 27.7 down)

// Order-preserving key: a < b as floats iff key(a) < key(b); -0 counts as +0.  Not for NaN.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint64_t order_of(float x, int i) { return (uint64_t)key_of(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float value_of(uint64_t o) { return of_key((uint32_t)(o >> 32)); }
__device__ __forceinline__ int index_of(uint64_t o) { return (int)~(uint32_t)o; }

struct SampleArgs {
  const void* x;
  int64_t row_stride;
  int vocab, part;  // part: tokens per CTA of a cluster
  int rows;
  bool long_first;  // more rows than run at once: those without a small top_k, which take longest, begin first
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *u;
  int32_t* id;
  float* logprob;
  int32_t* kept;
  float* probs;
};

// What a CTA's threads share, beside their part of the row.  What other CTAs write or read is there twice, used
// in turn: a CTA cannot be two exchanges ahead of another.
struct alignas(16) SampleShared {
  uint64_t list[kSampleList];
  uint32_t lo[2][kSteps], hi[2][kSteps];  // a histogram of 64-bit sums
  uint64_t slot[2][kMaxCluster][2];       // two words from every CTA of the cluster
  uint64_t weights[kShortList], mini[kMiniList];
  uint64_t wsum[kSampleWarps];
  uint64_t word, word2;
  uint32_t pick, count[2], minis;
};

// ---- over a CTA's threads
// Sum over a warp, in three parts whose sums 32 bits hold.
__device__ __forceinline__ uint64_t warp_add(uint64_t v) {
  const uint32_t a = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x7FFFFFFu);
  const uint32_t b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 27) & 0x7FFFFFFu);
  const uint32_t c = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 54));
  return ((uint64_t)c << 54) + ((uint64_t)b << 27) + a;
}
__device__ __forceinline__ uint64_t warp_most(uint64_t v) {
  const uint32_t h = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t l = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == h ? (uint32_t)v : 0u);
  return (uint64_t)h << 32 | l;
}
template <bool MAX>
__device__ __noinline__ uint64_t cta_reduce(uint64_t* wsum, uint64_t v) {
  v = MAX ? warp_most(v) : warp_add(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = wsum[threadIdx.x & 31];
  return MAX ? warp_most(v) : warp_add(v);
}
// Sum of what lies before this thread in its warp, and of the whole warp.
struct Scan {
  uint64_t before, all;
};
__device__ __forceinline__ Scan warp_scan(uint64_t v) {
  uint64_t run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
    if ((threadIdx.x & 31) >= o) run += up;
  }
  return {run - v, __shfl_sync(0xffffffffu, run, 31)};
}
__device__ __noinline__ Scan cta_scan(uint64_t* wsum, uint64_t v) {
  const Scan in = warp_scan(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = in.all;
  __syncthreads();
  const Scan of = warp_scan(wsum[threadIdx.x & 31]);
  return {__shfl_sync(0xffffffffu, of.before, threadIdx.x >> 5) + in.before, of.all};
}
// Sorts list[0 .. n) to falling order.
__device__ __noinline__ void cta_sort(uint64_t* list, int n) {
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kSampleThreads) list[i] = 0;
  __syncthreads();
  for (int h = 2; h <= size; h <<= 1) {
    for (int j = h >> 1; j >= 32; j >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += kSampleThreads) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const uint64_t u = list[a], v = list[b];
        if ((u < v) == ((a & h) == 0)) {
          list[a] = v;
          list[b] = u;
        }
      }
      __syncthreads();
    }
    for (int t = threadIdx.x; t < size; t += kSampleThreads) {  // strides within a warp
      uint64_t v = list[t];
      for (int j = min(h >> 1, 16); j > 0; j >>= 1) {
        const uint64_t u = __shfl_xor_sync(0xffffffffu, v, j);
        const bool big = ((t & j) == 0) == ((t & h) == 0);  // this place takes the larger
        v = (u > v) == big ? u : v;
      }
      list[t] = v;
    }
    if (h >= 32) __syncthreads();  // smaller ones stay within a warp's 32 places
  }
  __syncthreads();
}

// Sorts one number per thread to falling order (bitonic), the first n of them; the others are 0 and come last.
// Returns the thread's.  Exchanges between warps go through list, of 2 kSortList places, its halves in turn, so
// that one barrier each is enough; only the warps that n reaches do more than meet them.
__device__ __noinline__ uint64_t sort_one(uint64_t* list, uint64_t v, int n) {
  const int t = threadIdx.x;
  int size = 32, half = 0;
  while (size < n) size <<= 1;
#pragma unroll 1
  for (int h = 2; h <= size; h <<= 1) {
    const bool falls = (t & h) == 0;
    auto keep = [&](uint64_t u, int j) { v = (u > v) == (((t & j) == 0) == falls) ? u : v; };
#pragma unroll 1
    for (int j = h >> 1; j >= 32; j >>= 1) {
      if (t < size) list[half + t] = v;
      __syncthreads();
      if (t < size) keep(list[half + (t ^ j)], j);
      half ^= kSortList;
    }
    if (t < size) {
#pragma unroll 1
      for (int j = min(h >> 1, 16); j > 0; j >>= 1) keep(__shfl_xor_sync(0xffffffffu, v, j), j);
    }
  }
  __syncthreads();  // list may be written again
  return v;
}

// (x - m) / T; m is finite here, and 1 / T above 0.
__device__ __forceinline__ float gap_of(float v, float m, float r) { return __fmul_rn(__fsub_rn(v, m), r); }
// floor(2^40 e^g), with shifts of the mantissa: conversions share a slow unit with the exponential's.
__device__ __forceinline__ uint64_t weigh(float g) {
  const float e = expf(g);
  const uint32_t b = __float_as_uint(e), m24 = (b & 0x7FFFFFu) | 0x800000u;
  const int up = (int)(b >> 23) - 110;  // e = m24 2^(up - 40); a subnormal e, or 0, weighs nothing by the shift
  const uint32_t lo = __funnelshift_lc(0u, m24, (uint32_t)up) | __funnelshift_rc(m24, 0u, (uint32_t)-up);
  return (uint64_t)__funnelshift_rc(m24, 0u, (uint32_t)(32 - up)) << 32 | lo;
}
__device__ __noinline__ uint64_t weight_of(float v, float m, float r) { return weigh(gap_of(v, m, r)); }
// Whole part of 0 <= v < 2^23, without a conversion.
__device__ __forceinline__ uint32_t whole(float v) { return __float_as_uint(__fadd_rz(v, 8388608.f)) & 0x7FFFFFu; }

// A short list: this thread's token (-1: none), which `team` neighbouring threads share, its order and, on the
// first of them, its weight; the number and weight of the tokens before it in the list.
struct Place {
  int t, team;
  uint64_t order, w, weight_before;
  uint32_t count_before;
};
__device__ __noinline__ Place place_of(SampleShared& sh, int n, float m, float r) {
  Place q;
  q.team = n <= 32 ? 32 : n <= 64 ? 16 : n <= 128 ? 8 : 4;
  if (threadIdx.x < n) sh.weights[threadIdx.x] = weight_of(value_of(sh.list[threadIdx.x]), m, r);
  __syncthreads();
  q.t = threadIdx.x / q.team;
  if (q.t >= n) q.t = -1;
  q.order = q.t < 0 ? ~0ull : sh.list[q.t];
  q.w = q.t < 0 || (threadIdx.x & (q.team - 1)) ? 0 : sh.weights[q.t];
  q.weight_before = 0;
  q.count_before = 0;
#pragma unroll 4
  for (int j = threadIdx.x & (q.team - 1); j < n; j += q.team) {
    const uint64_t w = sh.weights[j];
    const bool higher = sh.list[j] > q.order;
    q.count_before += higher;
    q.weight_before += higher ? w : 0;
  }
  for (int o = q.team >> 1; o > 0; o >>= 1) {
    q.count_before += __shfl_xor_sync(0xffffffffu, q.count_before, o);
    q.weight_before += __shfl_xor_sync(0xffffffffu, q.weight_before, o);
  }
  return q;
}

template <class T>
struct Sampler {
  static constexpr int E = 16 / sizeof(T);  // tokens of a 16-byte piece
  SampleShared& sh;
  T* x;              // this CTA's part of the row, at the row's own alignment within 16 bytes; -inf around it
  int pieces;        // 16-byte pieces of it
  int base;          // index of x[0]; below the part's first token when that is not at a 16-byte boundary
  int ranks, rank;
  int flip, hist, listed;  // which of the two slots, histograms and counts is in use
  float m, r;        // the row's maximum, 1 / T
  uint64_t k;        // top_k
  float p;           // top_p
  uint64_t total;    // of the last histogram
  double want;       // weight before which a token is still taken by top_p
  uint64_t least;    // weight that min_p asks for
  float xe;          // the edge: tokens above xe, and those equal to it up to index ie
  int ie;

  __device__ __forceinline__ float gap(float v) const { return gap_of(v, m, r); }
  __device__ __forceinline__ uint64_t weight(float v) const { return weight_of(v, m, r); }
  __device__ __forceinline__ bool above_edge(float v, int i) const { return v > xe || (v == xe && i <= ie); }
  __device__ __forceinline__ void set_edge(uint64_t o) {
    xe = value_of(o);
    ie = index_of(o);
  }
  // Whether a token before which b lies (weight, or tokens) is taken.
  __device__ __forceinline__ bool taken(bool mass, uint64_t b) const { return mass ? b == 0 || (double)b < want : b < k; }

  __device__ __forceinline__ void sync() const {
    if (ranks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  __device__ __forceinline__ uint64_t sum(uint64_t v) const { return cta_reduce<false>(sh.wsum, v); }
  __device__ __forceinline__ uint64_t most(uint64_t v) const { return cta_reduce<true>(sh.wsum, v); }
  // Each warp has a contiguous run of pieces, its lanes interleaved.
  __device__ __forceinline__ void share(int& b, int& e) const {
    const int each = (pieces + kSampleWarps - 1) / kSampleWarps;
    b = min((int)(threadIdx.x >> 5) * each, pieces);
    e = min(b + each, pieces);
  }
  // Bit j: f(value, index) of token j of piece c.
  template <class F>
  __device__ __forceinline__ uint32_t test(int c, F f) const {
    const uint4 u = reinterpret_cast<const uint4*>(x)[c];
    const T* t = reinterpret_cast<const T*>(&u);
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (f(to_f32(t[j]), base + c * E + j)) mask |= 1u << j;
    return mask;
  }

  // f(value, index, weight) of the kept tokens of this warp's share.  Few are kept as a rule: a thread marks its
  // own first, then weighs those.
  template <class F>
  __device__ __forceinline__ void each_kept(F f) const {
    constexpr int kMark = 32 / E;  // pieces of a mask
    int b, e;
    share(b, e);
#pragma unroll 1
    for (int c0 = b + (threadIdx.x & 31); c0 < e; c0 += 32 * kMark) {
      uint32_t mask = 0;
#pragma unroll
      for (int q = 0; q < kMark; ++q)
        if (c0 + 32 * q < e) mask |= test(c0 + 32 * q, [&](float v, int i) { return above_edge(v, i); }) << (q * E);
      while (mask) {
        const int bit = __ffs((int)mask) - 1, i = (c0 + 32 * (bit / E)) * E + bit % E;
        mask &= mask - 1;
        const float v = to_f32(x[i]);
        const uint64_t w = weigh(gap(v));
        if (w >= least) f(v, base + i, w);
      }
    }
  }

  // Two words of every CTA of the cluster (thread 0's), left in slot[flip].
  __device__ __forceinline__ void exchange(uint64_t v, uint64_t w) {
    flip ^= 1;
    if (threadIdx.x < 32) {
      v = __shfl_sync(0xffffffffu, v, 0);
      w = __shfl_sync(0xffffffffu, w, 0);
      if (threadIdx.x < ranks) {
        uint64_t* to = sh.slot[flip][rank];
        if (ranks > 1) to = cg::this_cluster().map_shared_rank(to, threadIdx.x);
        to[0] = v;
        to[1] = w;
      }
    }
    sync();
  }
  // Gathers the tokens with f(value, index) into the first CTA's list, in no order.  Returns their number; the
  // list is cut off at its length.
  template <class F>
  __device__ __forceinline__ int gather(F f) {
    listed ^= 1;
    uint32_t* count = &sh.count[listed];
    uint64_t* list = sh.list;
    if (ranks > 1) {
      count = cg::this_cluster().map_shared_rank(count, 0);
      list = cg::this_cluster().map_shared_rank(list, 0);
    }
    int b, e;
    share(b, e);
#pragma unroll 1
    for (int c = b + (threadIdx.x & 31); c < e; c += 32) {
      uint32_t mask = test(c, f);
      while (mask) {
        const int i = c * E + __ffs((int)mask) - 1;
        mask &= mask - 1;
        const uint32_t at = atomicAdd(count, 1u);
        if (at < kSampleList) list[at] = order_of(to_f32(x[i]), base + i);
      }
    }
    sync();
    const int n = (int)*(volatile uint32_t*)count;
    // The other count was read by all before the barrier above, and is used again only after another one: there is
    // an exchange between any two gathers.  (This one may still be read by other CTAs.)
    if (rank == 0 && threadIdx.x == 0) sh.count[listed ^ 1] = 0;
    return n;
  }

  // Adds to a 64-bit sum.  The carry out of the low word is seen by the one thread that caused it: exact.
  __device__ __forceinline__ static void add(uint32_t* lo, uint32_t* hi, uint64_t w) {
    const uint32_t l = (uint32_t)w, was = atomicAdd(lo, l), h = (uint32_t)(w >> 32) + (was + l < l);
    if (h) atomicAdd(hi, h);
  }
  // Thread s has the sum v of step s (0 past the last): the last step that holds something and before which
  // b with taken(b) lies.  `above`: what lies before step 0, then before that step; total: the sum of all.
  template <class F>
  __device__ __forceinline__ uint32_t choose(uint64_t v, bool limit, uint64_t& above, F taken) {
    const Scan q = cta_scan(sh.wsum, v);
    const uint64_t b = above + q.before;
    total = q.all;
    if (limit) want = (double)p * (double)total;  // top_p's limit is of this histogram's sum
    if (v && taken(b)) atomicMax(&sh.pick, threadIdx.x);
    __syncthreads();
    const uint32_t s = sh.pick;
    if (threadIdx.x == s) sh.word = b;
    __syncthreads();
    above = sh.word;
    return s;
  }
  // A cleared histogram of f's tokens: f gives a token's step, or none (>= kSteps).
  template <class F>
  __device__ __forceinline__ void fill(bool mass, F f) {
    hist ^= 1;
    for (int i = threadIdx.x; i < kSteps; i += kSampleThreads) sh.lo[hist][i] = sh.hi[hist][i] = 0;
    __syncthreads();
    uint32_t* const lo = sh.lo[hist];
    uint32_t* const hi = sh.hi[hist];
#pragma unroll 4
    for (int i = threadIdx.x; i < pieces * E; i += kSampleThreads) {
      const float v = to_f32(x[i]), g = gap(v);
      const uint32_t s = f(v, g, base + i);
      if (s >= kSteps) continue;
      uint64_t w = 1;
      if (mass) w = weigh(g);
      add(lo + s, hi + s, w);
    }
  }
  // Of the cluster's histogram: the last step, counted from the top, whose first token is taken.  `above`:
  // what lies before it, at first what lies before step 0.  limit: top_p's is of this histogram's sum.
  __device__ __forceinline__ uint32_t pick(bool mass, bool limit, uint64_t& above) {
    if (threadIdx.x == 0) sh.pick = 0;
    sync();
    uint64_t v = 0;
    if (threadIdx.x < kSteps) {
#pragma unroll 4
      for (int c = 0; c < ranks; ++c) {  // every CTA sums all: none has to tell the others
        const SampleShared* o = ranks == 1 ? &sh : cg::this_cluster().map_shared_rank(&sh, c);
        v += (uint64_t)o->hi[hist][threadIdx.x] << 32 | o->lo[hist][threadIdx.x];
      }
    }
    return choose(v, limit, above, [&](uint64_t b) { return taken(mass, b); });
  }
  // How many of a sorted list's n tokens are taken, `above` before them.
  __device__ __forceinline__ int taken_of_sorted(bool mass, int n, uint64_t above) {
    const int per = (n + kSampleThreads - 1) / kSampleThreads, i0 = threadIdx.x * per, i1 = min(i0 + per, n);
    uint64_t mine = 0;
    for (int i = i0; i < i1; ++i) mine += mass ? weight(value_of(sh.list[i])) : 1;
    uint64_t b = above + cta_scan(sh.wsum, mine).before;
    uint32_t yes = 0;
    for (int i = i0; i < i1; ++i) {
      yes += taken(mass, b);
      b += mass ? weight(value_of(sh.list[i])) : 1;
    }
    return (int)sum(yes);
  }
  // The same over this CTA's list: step(o) of its tokens, or none (>= kSteps), each with weight(o).
  template <class S, class W, class F>
  __device__ __forceinline__ uint32_t list_level(int n, uint64_t& above, S step, W weight, F taken) {
    uint32_t* const lo = sh.lo[hist];  // nobody else reads it any more
    uint32_t* const hi = sh.hi[hist];
    __syncthreads();
    if (threadIdx.x < kSteps) lo[threadIdx.x] = hi[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.pick = sh.minis = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      const uint64_t o = sh.list[i];
      const uint32_t s = step(o);
      if (s < kSteps) add(lo + s, hi + s, weight(o));
    }
    __syncthreads();
    const int s = threadIdx.x;
    return choose(s < kSteps ? (uint64_t)hi[s] << 32 | lo[s] : 0, false, above, taken);
  }
  // The list's tokens with f(o), in no order; false when they are too many.
  template <class F>
  __device__ __forceinline__ bool mini_list(int n, F f) {
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      const uint64_t o = sh.list[i];
      if (!f(o)) continue;
      const uint32_t at = atomicAdd(&sh.minis, 1u);
      if (at < kMiniList) sh.mini[at] = o;
    }
    __syncthreads();
    return sh.minis <= kMiniList;
  }
  // The edge among the list's tokens above the present one, `above` before them; false: undecided, by a step
  // with too many tokens.
  __device__ __forceinline__ bool edge_in_list(bool mass, int n, uint64_t above) {
    auto weigh_one = [&](uint64_t o) { return mass ? weight(value_of(o)) : (uint64_t)1; };
    auto is_taken = [&](uint64_t b) { return taken(mass, b); };
    auto in = [&](uint64_t o) { return above_edge(value_of(o), index_of(o)) && gap(value_of(o)) > kFar; };
    const uint32_t s1 = list_level(n, above, [&](uint64_t o) { return in(o) ? whole(gap(value_of(o)) * -16.f) : kSteps; }, weigh_one, is_taken);
    auto fine = [&](uint64_t o) { return whole(gap(value_of(o)) * -8192.f); };
    const uint32_t s2 = list_level(n, above, [&](uint64_t o) { return in(o) && fine(o) / kSteps == s1 ? fine(o) % kSteps : kSteps; },
                                   weigh_one, is_taken);
    if (!mini_list(n, [&](uint64_t o) { return in(o) && fine(o) == s1 * kSteps + s2; })) return false;
    const int c = sh.minis;
    if (threadIdx.x < c) sh.weights[threadIdx.x] = weigh_one(sh.mini[threadIdx.x]);
    __syncthreads();
    uint64_t low = 0;
    if (threadIdx.x < c) {
      const uint64_t o = sh.mini[threadIdx.x];
      uint64_t b = above;
      for (int j = 0; j < c; ++j) b += sh.mini[j] > o ? sh.weights[j] : 0;
      if (taken(mass, b)) low = ~o;
    }
    set_edge(~most(low));
    return true;
  }
  // The edge within a list of n tokens with `above` before them: the first CTA finds it and tells the others.
  __device__ __forceinline__ void edge_of_list(bool mass, int n, uint64_t above) {
    uint64_t o = 0;
    if (rank == 0) {
      if (n <= kShortList) {
        const Place q = place_of(sh, n, m, r);
        const bool keep = q.t >= 0 && taken(mass, above + (mass ? q.weight_before : q.count_before));
        o = ~most(keep ? ~q.order : 0);
      } else if (n <= kSortList) {
        o = sort_one(sh.list, threadIdx.x < n ? sh.list[threadIdx.x] : 0, n);
        uint64_t b = threadIdx.x;
        if (mass) b = cta_scan(sh.wsum, threadIdx.x < n ? weight(value_of(o)) : 0).before;
        const int c = max(__syncthreads_count(threadIdx.x < n && taken(mass, above + b)), 1);
        if (threadIdx.x == c - 1) sh.word = o;
        __syncthreads();
        o = sh.word;
      } else if (edge_in_list(mass, n, above)) {
        o = order_of(xe, ie);
      } else {
        cta_sort(sh.list, n);
        o = sh.list[max(taken_of_sorted(mass, n, above), 1) - 1];
      }
      __syncthreads();  // the list may be written again
    }
    if (ranks > 1) {
      exchange(o, 0);
      o = sh.slot[flip][0][0];
    }
    set_edge(o);
  }
  // The edge among the tokens of step s1 where they are too many for a list: by 512ths of the step, and where
  // those of one are too many as well, by halving: the lowest number above which little enough lies.
  __device__ __noinline__ void refine(bool mass, uint32_t s1, uint64_t above) {
    const float from = -0.0625f * (float)s1, to = fmaxf(from - 0.0625f, kFar);
    fill(mass, [&](float v, float g, int i) { return g <= from && g > to && above_edge(v, i) ? whole(g * -8192.f) % kSteps : kSteps; });
    const uint32_t s2 = s1 * kSteps + pick(mass, false, above);
    auto in = [&](float v, int i) {
      const float g = gap(v);
      return g <= from && g > to && above_edge(v, i) && whole(g * -8192.f) == s2;
    };
    const int n = gather(in);
    if (n <= kSampleList) return edge_of_list(mass, n, above);
    uint64_t low = ~0ull, high = 0;
    for (int i = threadIdx.x; i < pieces * E; i += kSampleThreads) {
      const float v = to_f32(x[i]);
      if (!in(v, base + i)) continue;
      low = min(low, order_of(v, base + i));
      high = max(high, order_of(v, base + i));
    }
    low = most(~low);
    high = most(high);
    exchange(low, high);
    for (int c = 0; c < ranks; ++c) {
      low = max(low, sh.slot[flip][c][0]);
      high = max(high, sh.slot[flip][c][1]);
    }
    low = ~low;
    while (low < high) {
      const uint64_t mid = low + (high - low) / 2;
      uint64_t b = 0;
      for (int i = threadIdx.x; i < pieces * E; i += kSampleThreads) {
        const float v = to_f32(x[i]);
        if (in(v, base + i) && order_of(v, base + i) > mid) b += mass ? weight(v) : 1;
      }
      exchange(sum(b), 0);
      b = above;
      for (int c = 0; c < ranks; ++c) b += sh.slot[flip][c][0];
      if (taken(mass, b))
        high = mid;
      else
        low = mid + 1;
    }
    set_edge(low);
  }
  // The edge of top_k (by tokens) or top_p (by weight) among the tokens above the present one.
  __device__ __forceinline__ void find_edge(bool mass) {
    uint64_t above = 0;
    fill(mass, [&](float v, float g, int i) { return g > kFar && above_edge(v, i) ? whole(g * -16.f) : kSteps; });
    const uint32_t s1 = pick(mass, mass, above);
    const float from = -0.0625f * (float)s1, to = fmaxf(from - 0.0625f, kFar);
    const int n = gather([&](float v, int i) {
      const float g = gap(v);
      return g <= from && g > to && above_edge(v, i);
    });
    if (n <= kSampleList) return edge_of_list(mass, n, above);
    Sampler rare = *this;  // a copy, so that this one can stay in registers
    rare.refine(mass, s1, above);
    flip = rare.flip;
    hist = rare.hist;
    listed = rare.listed;
    xe = rare.xe;
    ie = rare.ie;
  }

  __device__ __forceinline__ uint64_t aim(float u, uint64_t z) const {
    return u > 0.f ? min((uint64_t)((double)u * (double)z), z - 1) : 0;
  }
  __device__ __forceinline__ void answer(const SampleArgs& a, int rw, int id, float v, uint64_t z, uint64_t kept) const {
    a.id[rw] = id;
    if (a.kept) a.kept[rw] = (int32_t)kept;
    if (a.logprob) a.logprob[rw] = gap(v) - logf(__fdiv_rn((float)(double)z, kOne));
  }
  // Everything from the first CTA's list, which holds the top k tokens: the edge of top_p, the kept weight and
  // the id.  Leaves the edge and Z for the others in sh.word and sh.word2.
  __device__ __forceinline__ void finish_list(const SampleArgs& a, int rw, float u, int n) {
    int t = -1, team = 1;  // this thread's kept token, and how many neighbours share it
    uint64_t order = 0, w = 0;
    if (n <= kShortList) {
      const Place q = place_of(sh, n, m, r);
      t = q.t;
      team = q.team;
      order = q.order;
      bool keep = t >= 0 && q.count_before < k;
      if (!(p >= 1.f)) {
        want = (double)p * (double)sum(keep ? q.w : 0);
        keep = keep && taken(true, q.weight_before);
      }
      if (a.probs) {
        const uint64_t o = ~most(keep ? ~order : 0);
        if (threadIdx.x == 0) sh.word = o;
      }
      w = keep && q.w >= least ? q.w : 0;
    } else if (n <= kSortList) {
      return finish_sort(a, rw, u, n);
    } else {
      return finish_long(a, rw, u, n);
    }
    const uint64_t z = sum(w), at = aim(u, z);
    const int kept = __syncthreads_count(w > 0);
    if (t >= 0 && (threadIdx.x & (team - 1)) == 0) sh.weights[t] = w;
    __syncthreads();
    uint64_t b = 0;  // kept weight at lower indexes
#pragma unroll 4
    for (int j = threadIdx.x & (team - 1); j < n; j += team) {
      const uint64_t v = sh.weights[j];
      b += (uint32_t)sh.list[j] > (uint32_t)order ? v : 0;
    }
    for (int o = team >> 1; o > 0; o >>= 1) b += __shfl_xor_sync(0xffffffffu, b, o);
    if (b <= at && at < b + w) answer(a, rw, index_of(order), value_of(order), z, kept);
    if (threadIdx.x == 0) sh.word2 = z;
  }
  // The same for a list that is sorted: what is kept are its first tokens, which are sorted again by index.
  __device__ __forceinline__ void finish_sort(const SampleArgs& a, int rw, float u, int n) {
    uint64_t o = sort_one(sh.list, threadIdx.x < n ? sh.list[threadIdx.x] : 0, n);
    bool keep = threadIdx.x < n && threadIdx.x < k;
    uint64_t w = keep ? weight(value_of(o)) : 0;
    if (!(p >= 1.f)) {
      const Scan q = cta_scan(sh.wsum, w);
      want = (double)p * (double)q.all;
      keep = keep && taken(true, q.before);
    }
    const int last = __syncthreads_count(keep) - 1;
    if (threadIdx.x == last) sh.word = o;
    keep = keep && w >= least && w > 0;
    const int kept = __syncthreads_count(keep);
    o = sort_one(sh.list, keep ? o << 32 | o >> 32 : 0, last + 1);
    w = threadIdx.x < kept ? weight(of_key((uint32_t)o)) : 0;
    const Scan q = cta_scan(sh.wsum, w);
    const uint64_t z = q.all, at = aim(u, z);
    if (q.before <= at && at < q.before + w) answer(a, rw, index_of(o >> 32), of_key((uint32_t)o), z, kept);
    if (threadIdx.x == 0) sh.word2 = z;
  }
  // The same for a longer list.
  __device__ __forceinline__ void finish_long(const SampleArgs& a, int rw, float u, int n) {
    bool sure = (uint64_t)n <= k || edge_in_list(false, n, 0);
    auto kept_weight = [&](uint64_t o) -> uint64_t {
      if (!above_edge(value_of(o), index_of(o))) return 0;
      const uint64_t w = weight(value_of(o));
      return w < least ? 0 : w;
    };
    if (sure && !(p >= 1.f)) {
      uint64_t all = 0;
      for (int i = threadIdx.x; i < n; i += kSampleThreads) {
        const uint64_t o = sh.list[i];
        if (above_edge(value_of(o), index_of(o))) all += weight(value_of(o));
      }
      want = (double)p * (double)sum(all);
      sure = edge_in_list(true, n, 0);
    }
    if (sure) {
      uint64_t mine = 0, some = 0;
      for (int i = threadIdx.x; i < n; i += kSampleThreads) {
        const uint64_t w = kept_weight(sh.list[i]);
        mine += w;
        some += w > 0;
      }
      const uint64_t z = sum(mine), at = aim(u, z);
      const uint64_t kept = sum(some);
      // the step of the index in which the running weight passes `at`, then the place in it
      const int width = (a.vocab + kSteps - 1) / kSteps;
      uint64_t before = 0;
      const int s = list_level(n, before, [&](uint64_t o) { return kept_weight(o) ? (uint32_t)(index_of(o) / width) : kSteps; },
                               kept_weight, [&](uint64_t b) { return b <= at; });
      if (mini_list(n, [&](uint64_t o) { return index_of(o) / width == s && kept_weight(o) > 0; })) {
        const int c = sh.minis;
        if (threadIdx.x < c) sh.weights[threadIdx.x] = kept_weight(sh.mini[threadIdx.x]);
        __syncthreads();
        if (threadIdx.x < c) {
          const uint64_t o = sh.mini[threadIdx.x];
          for (int j = 0; j < c; ++j) before += index_of(sh.mini[j]) < index_of(o) ? sh.weights[j] : 0;
          if (before <= at && at < before + sh.weights[threadIdx.x]) answer(a, rw, index_of(o), value_of(o), z, kept);
        }
        if (threadIdx.x == 0) {
          sh.word = order_of(xe, ie);
          sh.word2 = z;
        }
        return;
      }
    }
    cta_sort(sh.list, n);
    n = (int)min((uint64_t)n, k);
    if (!(p >= 1.f)) {
      uint64_t all = 0;
      for (int i = threadIdx.x; i < n; i += kSampleThreads) all += weight(value_of(sh.list[i]));
      want = (double)p * (double)sum(all);
      n = taken_of_sorted(true, n, 0);
    }
    if (threadIdx.x == 0) sh.word = sh.list[n - 1];
    finish_sorted(a, rw, u, n);
  }
  // The same for a sorted list of n kept tokens: sorted again, by rising index.
  __device__ __forceinline__ void finish_sorted(const SampleArgs& a, int rw, float u, int n) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      const uint64_t v = sh.list[i];
      sh.list[i] = v << 32 | v >> 32;
    }
    __syncthreads();
    cta_sort(sh.list, n);
    const int per = (n + kSampleThreads - 1) / kSampleThreads, i0 = threadIdx.x * per, i1 = min(i0 + per, n);
    uint64_t mass = 0, some = 0;
    for (int i = i0; i < i1; ++i) {
      const uint64_t w = weight(of_key((uint32_t)sh.list[i]));
      if (w < least) continue;
      mass += w;
      some += w > 0;
    }
    const uint64_t kept = sum(some);
    const Scan q = cta_scan(sh.wsum, mass);
    const uint64_t z = q.all, at = aim(u, z);
    uint64_t b = q.before;
    if (b <= at && at < b + mass) {
      for (int i = i0; i < i1; ++i) {
        const uint64_t v = sh.list[i];
        uint64_t w = weight(of_key((uint32_t)v));
        if (w < least) w = 0;
        if (at < b + w) {
          answer(a, rw, index_of(v >> 32), of_key((uint32_t)v), z, kept);
          break;
        }
        b += w;
      }
    }
    if (threadIdx.x == 0) sh.word2 = z;
  }
};

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  using S = Sampler<T>;
  constexpr int E = S::E;
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  const int tid = threadIdx.x, lane = tid & 31;
  int rw = blockIdx.y;
  S s{sh, reinterpret_cast<T*>(smem + sizeof(SampleShared))};
  s.ranks = gridDim.x;
  s.rank = blockIdx.x;
  s.flip = s.hist = s.listed = 0;
  // no CTA's memory is written before it runs: the wait comes with the first exchange
  if (s.ranks > 1) cg::this_cluster().barrier_arrive();
  if (a.long_first) {  // CTA c takes the c-th of the long rows, then of the others
    const float t = tid < a.rows && a.temperature ? a.temperature[tid] : 1.f;
    const int k = tid < a.rows && a.top_k ? a.top_k[tid] : 0;
    const bool is_long = tid < a.rows && t > 0.f && (k <= 0 || k > kSampleMaxK);
    const Scan q = cta_scan(sh.wsum, is_long);
    if (tid < a.rows && (int)(is_long ? q.before : q.all + tid - q.before) == rw) sh.pick = tid;
    __syncthreads();
    rw = sh.pick;
  }
  const int first = min(s.rank * a.part, a.vocab), n = min(a.part, a.vocab - first);  // this CTA's tokens
  const T* const row = static_cast<const T*>(a.x) + (int64_t)rw * a.row_stride + first;
  const int lead = (int)((uintptr_t)row & 15) / (int)sizeof(T);
  s.base = first - lead;
  s.pieces = (lead + n + E - 1) / E;
  float* const probs = a.probs ? a.probs + (int64_t)rw * a.vocab : nullptr;
  const float min_p = a.min_p ? a.min_p[rw] : 0.f, t = a.temperature ? a.temperature[rw] : 1.f, u = a.u[rw];
  const int top_k = a.top_k ? a.top_k[rw] : 0;
  s.p = a.top_p ? a.top_p[rw] : 1.f;
  if (tid < 2) sh.count[tid] = 0;
  for (int i = tid; i < kSteps; i += kSampleThreads) sh.lo[0][i] = sh.hi[0][i] = 0;
  // ---- the row, and every thread's maximum; the first and last piece, which may hold less, by token
  float mine = -INFINITY;
  {
    const uint4* const from = reinterpret_cast<const uint4*>(row - lead);
    const bool begins = lead > 0 || n < E, cut[2] = {begins, (lead + n) % E != 0 && !(begins && s.pieces == 1)};
    int b, e;
    s.share(b, e);
#pragma unroll 4
    for (int c = b + lane; c < e; c += 32) {
      if ((c == 0 && cut[0]) || (c == s.pieces - 1 && cut[1])) continue;
      const uint4 u = __ldcs(from + c);
      reinterpret_cast<uint4*>(s.x)[c] = u;
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < E; ++j) mine = fmaxf(mine, to_f32(t[j]));  // not NaN's
    }
    if (tid < 2 * E && cut[tid / E]) {
      const int at = (tid < E ? 0 : s.pieces - 1) * E + tid % E, i = at - lead;
      const T v = i >= 0 && i < n ? row[i] : from_f32<T>(-INFINITY);
      s.x[at] = v;
      mine = fmaxf(mine, to_f32(v));
    }
  }
  if (s.ranks > 1) cg::this_cluster().barrier_wait();
  uint64_t top = s.most(key_of(mine));
  if (s.ranks > 1) {
    s.exchange(top, 0);
    for (int c = 0; c < s.ranks; ++c) top = max(top, sh.slot[s.flip][c][0]);
  }
  s.m = of_key((uint32_t)top);
  if (s.m == -INFINITY || min_p > 1.f) {  // no token to draw
    if (s.rank == 0 && tid == 0) {
      a.id[rw] = -1;
      if (a.logprob) a.logprob[rw] = -INFINITY;
      if (a.kept) a.kept[rw] = 0;
    }
    if (probs)
      for (int i = tid; i < n; i += kSampleThreads) probs[first + i] = 0.f;
    return;
  }
  s.least = min_p > 0.f ? (uint64_t)ceil((double)min_p * (double)kOne) : 0;  // weights are whole numbers
  const bool greedy = !(t > 0.f);
  s.r = greedy ? 1.f : fminf(fmaxf(__fdiv_rn(1.f, t), 1e-37f), 1e38f);  // not 0 for an infinite T, nor infinite for a tiny one
  if (s.m == INFINITY) {  // infinite logits are all the row has: 0 among -inf
    for (int i = tid; i < s.pieces * E; i += kSampleThreads) s.x[i] = from_f32<T>(to_f32(s.x[i]) == INFINITY ? 0.f : -INFINITY);
    s.m = 0.f;
    mine = mine == INFINITY ? 0.f : -INFINITY;
    __syncthreads();
  }
  int k = greedy ? 1 : top_k;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  s.k = k;
  s.xe = -INFINITY;  // every token above -inf, and none of what surrounds the part (its indexes may be below 0)
  s.ie = INT_MIN;

  // ---- the edge: tokens at or above it are kept
  bool done = false;
  uint64_t z = 0;
  if (k == 1) {  // the first of the tokens that are equal to the maximum
    int b, e;
    s.share(b, e);
    uint32_t at = ~0u;
    for (int c = b + lane; c < e; c += 32) {
      const uint32_t mask = s.test(c, [&](float v, int) { return v == s.m; });
      if (mask) {
        at = (uint32_t)(s.base + c * E + __ffs((int)mask) - 1);
        break;
      }
    }
    uint64_t id = s.most(~at);
    if (s.ranks > 1) {
      s.exchange(id, 0);
      for (int c = 0; c < s.ranks; ++c) id = max(id, sh.slot[s.flip][c][0]);
    }
    s.xe = s.m;
    s.ie = (int)~(uint32_t)id;
    z = (uint64_t)1 << 40;
    if (s.rank == 0 && tid == 0) s.answer(a, rw, s.ie, s.m, z, 1);
    done = true;
  } else if (k < a.vocab && k <= kSampleMaxK) {
    // the step in which the k-th largest of the threads' maxima lies, and all that is above it; where a thread has
    // few tokens these count themselves, as few threads have a maximum there (730 tokens, k 109: 19,600 cycles
    // instead of 37,200)
    const bool few = s.pieces * E <= kFewTokens;
    for (int i = tid; i < (few ? s.pieces * E : kSampleThreads); i += kSampleThreads) {
      const float g = s.gap(few ? to_f32(s.x[i]) : mine);
      if (g > kFar) atomicAdd(&sh.lo[0][whole(g * -16.f)], 1u);
    }
    uint64_t above = 0;
    float to = fmaxf(-0.0625f * (float)(s.pick(false, false, above) + 1), kFar);
    if (s.total < s.k) to = kFar;  // fewer than k of them have any weight
    const int c = s.gather([&](float v, int) { return s.gap(v) > to; });
    done = c <= kSampleList;
    if (done) {
      if (s.rank == 0) s.finish_list(a, rw, u, c);
      if (probs) {
        s.sync();
        const SampleShared* o = s.ranks > 1 ? cg::this_cluster().map_shared_rank(&sh, 0) : &sh;
        s.set_edge(o->word);
        z = o->word2;
      }
    }
  }
  if (!done) {
#pragma unroll 1
    for (int by = 0; by < 2; ++by)
      if (by ? !(s.p >= 1.f) : k < a.vocab) s.find_edge(by);
    // ---- the kept weight Z, and the token in index order where the running weight passes floor(u Z)
    int b, e;
    s.share(b, e);
    uint64_t v = 0, some = 0;
    s.each_kept([&](float, int, uint64_t w) {
      v += w;
      some += w > 0;
    });
    const Scan q = cta_scan(sh.wsum, v);
    uint64_t kept = s.sum(some), ahead = q.before;
    s.exchange(q.all, kept);
    kept = 0;
    for (int c = 0; c < s.ranks; ++c) {
      if (c < s.rank) ahead += sh.slot[s.flip][c][0];
      z += sh.slot[s.flip][c][0];
      kept += sh.slot[s.flip][c][1];
    }
    ahead = __shfl_sync(0xffffffffu, ahead, 0);  // before this warp's share
    uint64_t aim = s.aim(u, z);
    if (ahead <= aim && aim < ahead + warp_add(v)) {  // one warp of one CTA: the place in its share
      aim -= ahead;
#pragma unroll 1
      for (int c = b; c < e; c += 32) {
        auto kept_weight = [&](int j) -> uint64_t {
          const int i = (c + lane) * E + j;
          const float f = to_f32(s.x[i]);
          const uint64_t w = s.above_edge(f, s.base + i) ? s.weight(f) : 0;
          return w < s.least ? 0 : w;
        };
        uint64_t own = 0;
        if (c + lane < e) {
#pragma unroll 1
          for (int j = 0; j < E; ++j) own += kept_weight(j);
        }
        const Scan in = warp_scan(own);
        if (aim >= in.all) {
          aim -= in.all;
          continue;
        }
        if (in.before <= aim && aim < in.before + own) {
          aim -= in.before;
          int j = 0;
          for (uint64_t w; aim >= (w = kept_weight(j)); ++j) aim -= w;
          const int i = (c + lane) * E + j;
          s.answer(a, rw, s.base + i, to_f32(s.x[i]), z, kept);
        }
        break;
      }
    }
  }
  if (probs) {  // nothing for all, then their shares for the few that are kept
#pragma unroll 4
    for (int i = tid; i < n; i += kSampleThreads) probs[first + i] = 0.f;
    __syncthreads();
    const float share = __fdiv_rn(1.f, (float)z);
    s.each_kept([&](float, int i, uint64_t w) { probs[i] = (float)w * share; });
  }
  if (s.ranks > 1) s.sync();  // no CTA leaves while another may still read its histogram
}

// Opt in to the shared memory, and to clusters of 16, once per kernel and device.
template <class T>
bool allow_sample(int dev) {
  static std::atomic<uint64_t> done{0};
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return true;
  if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess ||
      cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return false;
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

template <class T>
int launch_sample(SampleArgs a, int rows, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      !allow_sample<T>(dev))
    return refuse(MLLM_ERR_CUDA, "mllm_sample: no current CUDA device, or too little shared memory");
  // CTAs per row: as many as its tokens need room for, and more while SMs are left and each keeps 4,096 tokens
  const int64_t room = (227 * 1024 - 32 - (int64_t)sizeof(SampleShared)) / sizeof(T) / 32 * 32;
  int ranks = 1;
  while (ranks < kMaxCluster && ((int64_t)ranks * room < a.vocab || ((int64_t)rows * ranks * 2 <= sms && a.vocab / (2 * ranks) >= 4096)))
    ranks *= 2;
  a.part = ((a.vocab + ranks - 1) / ranks + 31) / 32 * 32;
  a.rows = rows;
  a.long_first = (int64_t)rows * ranks > sms && rows <= kSampleThreads && a.top_k;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, rows);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared) + (size_t)a.part * sizeof(T) + 32;  // a piece at either end
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)ranks, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = ranks > 1;
  if (cudaLaunchKernelEx(&cfg, sample_kernel<T>, a) != cudaSuccess) {
    (void)cudaGetLastError();
    return refuse(MLLM_ERR_CUDA, "mllm_sample: launch failed");
  }
  return MLLM_OK;
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_sample(int dtype, const void* d_logits, int64_t row_stride, int rows, int vocab,
                           const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                           const float* d_min_p, const float* d_u, int32_t* d_id, float* d_logprob, int32_t* d_kept,
                           float* d_probs, void* stream) {
  using namespace mllm;
  using namespace mllm::paged;
  if (!is_float_kind(dtype)) return refuse(MLLM_ERR_UNSUPPORTED, "mllm_sample: logits must be f32, f16 or bf16");
  if (rows < 0 || rows > 65535 || vocab < 1 || row_stride < vocab)
    return refuse(MLLM_ERR_ARG, "mllm_sample: rows outside 0 to 65,535, an empty vocabulary, or a row stride below it");
  if (vocab > 524288) return refuse(MLLM_ERR_UNSUPPORTED, "mllm_sample: vocab above 524,288");
  if (rows == 0) return MLLM_OK;
  if (!d_logits || !d_u || !d_id) return refuse(MLLM_ERR_ARG, "mllm_sample: null pointer");
  if ((uintptr_t)d_logits % esize(dtype)) return refuse(MLLM_ERR_ARG, "mllm_sample: misaligned logits");
  const SampleArgs a = {d_logits, row_stride, vocab, 0, rows, false, d_temperature, d_top_k, d_top_p, d_min_p, d_u, d_id, d_logprob,
                        d_kept, d_probs};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16) return launch_sample<__half>(a, rows, st);
  if (dtype == MLLM_DTYPE_BF16) return launch_sample<__nv_bfloat16>(a, rows, st);
  return launch_sample<float>(a, rows, st);
}
