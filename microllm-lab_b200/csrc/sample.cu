// Sampling with temperature, top-k, top-p and min-p from one given uniform number per row (mllm_sample).
//
// With x the row (NaN as -inf), m its maximum and r = 1 / T, token i weighs w_i = floor(2^40 exp((x_i - m) r)).
// Tokens are ordered by falling x, ties by rising index: by the 64-bit number (key of x, ~index).  The
// tokens that top-k or top-p keep are those at or above an edge in that order, the lowest number before
// which few enough tokens (top-k) or little enough weight (top-p) lies.  The id is found in index order, at
// the place where the running kept weight passes floor(u Z).  Weights are integers of at most 2^40 (a sum
// of 2^19 of them fits 64 bits), so every sum is exact and no result depends on the order in which threads
// add.  The 2^-40 that a weight loses is 2^-40 of the top token's: over 2^18 tokens at most 2^-22 of the
// row, the size of an f32 rounding.
//
// A row is read once, into the shared memory of one CTA, or of a cluster's CTAs, each of which has a
// contiguous part, where rows are fewer than SMs or do not fit.  The edge is found without sorting the row:
//   - top_k up to 512: the step of 1/16 of a unit of (x - m) r in which the k-th largest of the threads' own
//     maxima lies bounds the k-th token from below, so the few tokens down to that step are gathered, and
//     everything else happens in that list;
//   - otherwise by a histogram of tokens or weight over 512 such steps, then among the tokens of one step,
//     or of a 512th of it where they are too many for a list;
//   - and by halving, one pass per bit, where those are too many as well (thousands of tokens of one value).
// A list is sorted and summed by one warp when it is short, by the CTA otherwise.
#include <cooperative_groups.h>

#include <atomic>

#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleList = 2048;   // tokens of a list
constexpr int kWarpList = 128;      // tokens of a list that one warp handles
constexpr int kSampleMaxK = 512;    // top_k that starts from the threads' maxima
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
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *u;
  int32_t* id;
  float* logprob;
  int32_t* kept;
  float* probs;
};

// What a CTA's threads share, beside their part of the row.
struct SampleShared {
  uint64_t list[kSampleList];
  uint32_t lo[kSteps], hi[kSteps];  // a histogram of 64-bit sums
  uint64_t slot[2][kMaxCluster];    // one word from every CTA of the cluster
  uint64_t wsum[kSampleWarps], wbase[kSampleWarps], all;
  uint64_t word[2];  // what the first CTA has decided
  uint32_t pick, count;
};

static_assert(sizeof(SampleShared) % 16 == 0, "the row follows it");

template <class T>
struct Sampler {
  static constexpr int E = 16 / sizeof(T);  // tokens of a 16-byte piece
  SampleShared& sh;
  T* x;              // this CTA's part of the row, at the row's own alignment within 16 bytes; -inf around it
  int pieces;        // 16-byte pieces of it
  int base;          // index of x[0]; below the part's first token when that is not at a 16-byte boundary
  int ranks, rank;
  int flip;          // slot in use
  float m, r;        // the row's maximum, 1 / T
  uint64_t k;        // top_k
  float p;           // top_p
  uint64_t total;    // of the last histogram
  double want, least;  // weight before which a token is still taken by top_p; weight that min_p asks for
  float xe;          // the edge: tokens above xe, and those equal to it up to index ie
  int ie;

  // (x - m) / T; the maximum itself may be infinite.
  __device__ __forceinline__ float gap(float v) const { return v == m ? 0.f : __fmul_rn(__fsub_rn(v, m), r); }
  __device__ __forceinline__ uint64_t weigh(float g) const {  // g = NaN (an infinite gap times 1 / T = 0): nothing
    const float e = expf(g);
    return e > 0.f ? (uint64_t)__fmul_rn(e, kOne) : 0;
  }
  __device__ __forceinline__ uint64_t weight(float v) const { return weigh(gap(v)); }
  __device__ __forceinline__ bool above_edge(float v, int i) const { return v > xe || (v == xe && i <= ie); }
  __device__ __forceinline__ void set_edge(uint64_t o) {
    xe = value_of(o);
    ie = index_of(o);
  }
  template <bool MASS>
  __device__ __forceinline__ bool taken(uint64_t b) const {  // whether a token before which b lies is taken
    return MASS ? b == 0 || (double)b < want : b < k;
  }

  __device__ __forceinline__ void sync() const {
    if (ranks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  // f(value, index) of this thread's tokens: each warp has a contiguous run of pieces, lanes interleaved.
  __device__ __forceinline__ void share(int& b, int& e) const {
    const int each = (pieces + kSampleWarps - 1) / kSampleWarps;
    b = min((int)(threadIdx.x >> 5) * each, pieces);
    e = min(b + each, pieces);
  }
  __device__ __forceinline__ void piece(int c, float (&v)[E]) const {
    const uint4 u = reinterpret_cast<const uint4*>(x)[c];
    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = to_f32(t[e]);
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    int b, e;
    share(b, e);
#pragma unroll 2
    for (int c = b + (threadIdx.x & 31); c < e; c += 32) {
      float v[E];
      piece(c, v);
#pragma unroll
      for (int j = 0; j < E; ++j) f(v[j], base + c * E + j);
    }
  }

  // One word of every CTA (its thread 0's), on every thread, combined in the order of the CTAs.
  template <class F>
  __device__ __forceinline__ uint64_t combine(uint64_t v, F f) {
    flip ^= 1;
    if (ranks == 1) {
      if (threadIdx.x == 0) sh.slot[flip][0] = v;
    } else if (threadIdx.x < 32) {
      v = __shfl_sync(0xffffffffu, v, 0);
      if (threadIdx.x < ranks) *cg::this_cluster().map_shared_rank(&sh.slot[flip][rank], threadIdx.x) = v;
    }
    sync();
    v = sh.slot[flip][0];
    for (int c = 1; c < ranks; ++c) v = f(v, sh.slot[flip][c]);
    return v;
  }
  template <class F>
  __device__ __forceinline__ uint64_t reduce(uint64_t v, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
      v = sh.wsum[threadIdx.x];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return combine(v, f);
  }
  __device__ __forceinline__ uint64_t sum(uint64_t v) {
    return reduce(v, [](uint64_t a, uint64_t b) { return a + b; });
  }
  __device__ __forceinline__ uint64_t largest(uint64_t v) {
    return reduce(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
  }

  // ---- teams: the first warp, or the CTA
  template <bool WARP>
  __device__ __forceinline__ static void team_sync() {
    if (WARP)
      __syncwarp();
    else
      __syncthreads();
  }
  // Sum of what lies before this thread in the team; `all`: of the whole team.
  template <bool WARP>
  __device__ __forceinline__ uint64_t before(uint64_t v, uint64_t& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (WARP) {
      all = __shfl_sync(0xffffffffu, run, 31);
      return run - v;
    }
    __syncthreads();
    if (lane == 31) sh.wsum[warp] = run;
    __syncthreads();
    if (warp == 0) {
      uint64_t w = sh.wsum[lane], t = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += up;
      }
      sh.wbase[lane] = t - w;
      if (lane == 31) sh.all = t;
    }
    __syncthreads();
    all = sh.all;
    return sh.wbase[warp] + run - v;
  }
  // Sorts list[0 .. n) to falling order.
  template <bool WARP>
  __device__ __noinline__ static void sort(uint64_t* list, int n) {
    const int me = threadIdx.x;
    constexpr int team = WARP ? 32 : kSampleThreads;
    int size = 32;
    while (size < n) size <<= 1;
    for (int i = n + me; i < size; i += team) list[i] = 0;
    team_sync<WARP>();
    for (int h = 2; h <= size; h <<= 1) {
      for (int j = h >> 1; j >= 32; j >>= 1) {
        for (int t = me; t < size / 2; t += team) {
          const int a = 2 * t - (t & (j - 1)), b = a + j;
          const uint64_t u = list[a], v = list[b];
          if ((u < v) == ((a & h) == 0)) {
            list[a] = v;
            list[b] = u;
          }
        }
        team_sync<WARP>();
      }
      for (int t = me; t < size; t += team) {  // strides within a warp
        uint64_t v = list[t];
        for (int j = min(h >> 1, 16); j > 0; j >>= 1) {
          const uint64_t u = __shfl_xor_sync(0xffffffffu, v, j);
          const bool big = ((t & j) == 0) == ((t & h) == 0);  // this place takes the larger
          v = (u > v) == big ? u : v;
        }
        list[t] = v;
      }
      if (h >= 32) team_sync<WARP>();  // smaller ones stay within a warp's 32 places
    }
    team_sync<WARP>();
  }
  // For a falling list of n tokens, `above` before them: how many are taken.
  template <bool WARP, bool MASS>
  __device__ __forceinline__ int taken_of_list(int n, uint64_t above) {
    const int per = (n + (WARP ? 32 : kSampleThreads) - 1) / (WARP ? 32 : kSampleThreads), i0 = threadIdx.x * per;
    uint64_t mine = 0, all;
    for (int i = i0; i < min(i0 + per, n); ++i) mine += MASS ? weight(value_of(sh.list[i])) : 1;
    uint64_t b = above + before<WARP>(mine, all);
    uint32_t yes = 0;
    for (int i = i0; i < min(i0 + per, n); ++i) {
      yes += taken<MASS>(b);
      b += MASS ? weight(value_of(sh.list[i])) : 1;
    }
    (void)before<WARP>(yes, all);
    return (int)all;
  }
  __device__ __forceinline__ uint64_t aim(float u, uint64_t z) const {
    return u > 0.f ? min((uint64_t)((double)u * (double)z), z - 1) : 0;
  }
  __device__ __forceinline__ void answer(const SampleArgs& a, int rw, int id, float v, uint64_t z, uint64_t kept) const {
    a.id[rw] = id;
    if (a.kept) a.kept[rw] = (int32_t)kept;
    if (a.logprob) a.logprob[rw] = gap(v) - logf(__fdiv_rn((float)(double)z, kOne));
  }
  // Everything from a list that holds the top k tokens: the edge of top_p, the kept weight and the id.
  template <bool WARP>
  __device__ __forceinline__ void finish_list(const SampleArgs& a, int rw, int n) {
    constexpr int team = WARP ? 32 : kSampleThreads;
    const int me = threadIdx.x;
    sort<WARP>(sh.list, n);
    int c = (int)min((uint64_t)n, k);
    if (!(p >= 1.f)) {
      uint64_t total = 0, all;
      for (int i = me; i < c; i += team) total += weight(value_of(sh.list[i]));
      (void)before<WARP>(total, all);
      want = (double)p * (double)all;
      c = taken_of_list<WARP, true>(c, 0);
    }
    if (me == 0) sh.word[0] = sh.list[c - 1];
    // the kept ones by rising index: sorted by (~index, key)
    team_sync<WARP>();
    for (int i = me; i < c; i += team) {
      const uint64_t v = sh.list[i];
      sh.list[i] = v << 32 | v >> 32;
    }
    team_sync<WARP>();
    sort<WARP>(sh.list, c);
    const int per = (c + team - 1) / team, i0 = me * per, i1 = min(i0 + per, c);
    uint64_t mass = 0, some = 0, z, kept;
    for (int i = i0; i < i1; ++i) {
      const uint64_t w = weight(of_key((uint32_t)sh.list[i]));
      if (w == 0 || (double)w < least) continue;
      mass += w;
      ++some;
    }
    (void)before<WARP>(some, kept);
    uint64_t b = before<WARP>(mass, z);
    const uint64_t at = aim(a.u[rw], z);
    if (b <= at && at < b + mass) {
      for (int i = i0; i < i1; ++i) {
        const uint64_t v = sh.list[i], w = weight(of_key((uint32_t)v));
        if (w == 0 || (double)w < least) continue;
        if (at < b + w) {
          answer(a, rw, index_of(v >> 32), of_key((uint32_t)v), z, kept);
          break;
        }
        b += w;
      }
    }
    if (me == 0) sh.word[1] = z;
  }

  // Gathers the tokens with f(value, index) into the first CTA's list, in no order.  Returns their number;
  // the list is cut off at its length.  sh.count of the first CTA is 0 before.
  template <class F>
  __device__ __forceinline__ int gather(F f) {
    uint64_t* list = sh.list;
    uint32_t* count = &sh.count;
    if (ranks > 1) {
      list = cg::this_cluster().map_shared_rank(list, 0);
      count = cg::this_cluster().map_shared_rank(count, 0);
    }
    each([&](float v, int i) {
      if (!f(v, i)) return;
      const uint32_t at = atomicAdd(count, 1u);
      if (at < kSampleList) list[at] = order_of(v, i);
    });
    sync();
    const int n = (int)*(volatile uint32_t*)count;
    sync();
    if (rank == 0 && threadIdx.x == 0) sh.count = 0;
    return n;
  }

  // Histogram step: adds v to the 64-bit sum of step s.  The carry out of the low word is seen by the one
  // thread that caused it, so the sum is exact.
  __device__ __forceinline__ void add(uint32_t s, uint64_t v) {
    const uint32_t l = (uint32_t)v;
    const uint32_t was = atomicAdd(&sh.lo[s], l);
    const uint32_t h = (uint32_t)(v >> 32) + (was + l < l);
    if (h) atomicAdd(&sh.hi[s], h);
  }
  __device__ __forceinline__ void clear() {
    __syncthreads();
    for (int i = threadIdx.x; i < kSteps; i += kSampleThreads) sh.lo[i] = sh.hi[i] = 0;
    __syncthreads();
  }
  // Of the cluster's histogram: the last step, counted from the top, whose first token is taken.  `above`:
  // what lies before it, at first what lies before step 0.  TOTAL: top_p's limit is of this histogram's sum.
  template <bool MASS, bool TOTAL>
  __device__ __forceinline__ uint32_t pick(uint64_t& above) {
    sync();
    uint64_t v = 0, all;
    if (threadIdx.x < kSteps) {
      for (int c = 0; c < ranks; ++c) {  // every CTA sums all: none has to tell the others
        const SampleShared* o = ranks == 1 ? &sh : cg::this_cluster().map_shared_rank(&sh, c);
        v += (uint64_t)o->hi[threadIdx.x] << 32 | o->lo[threadIdx.x];
      }
    }
    if (threadIdx.x == 0) sh.pick = 0;
    const uint64_t b = above + before<false>(v, all);
    total = all;
    if (TOTAL) want = (double)p * (double)all;
    if (v && taken<MASS>(b)) atomicMax(&sh.pick, threadIdx.x);
    __syncthreads();
    const uint32_t s = sh.pick;
    if (threadIdx.x == s) sh.word[1] = b;
    sync();  // also: the other CTAs have read this one's sums
    above = sh.word[1];
    return s;
  }
  // The edge of top_k (by tokens) or top_p (by weight) among the tokens above the present one.
  template <bool MASS>
  __device__ __forceinline__ void find_edge() {
    uint64_t above = 0;
    clear();
    each([&](float v, int i) {
      const float g = gap(v);
      if (!(g > kFar) || !above_edge(v, i)) return;
      const uint32_t s = (uint32_t)(g * -16.f);
      if (MASS) {
        const uint64_t w = weigh(g);
        if (w) add(s, w);
      } else {
        atomicAdd(&sh.lo[s], 1u);
      }
    });
    const uint32_t s1 = pick<MASS, MASS>(above);
    const float from = -0.0625f * (float)s1, to = from - 0.0625f;
    auto in1 = [&](float v, int i) {
      const float g = gap(v);
      return g <= from && g > to && g > kFar && above_edge(v, i);
    };
    int n = gather(in1);
    if (n > kSampleList) {
      clear();
      each([&](float v, int i) {
        if (!in1(v, i)) return;
        const float g = gap(v);
        const uint32_t s = (uint32_t)(g * -8192.f) % kSteps;
        if (MASS) {
          const uint64_t w = weigh(g);
          if (w) add(s, w);
        } else {
          atomicAdd(&sh.lo[s], 1u);
        }
      });
      const uint32_t s2 = s1 * kSteps + pick<MASS, false>(above);
      auto in2 = [&](float v, int i) { return in1(v, i) && (uint32_t)(gap(v) * -8192.f) == s2; };
      n = gather(in2);
      if (n > kSampleList) return halve<MASS>(above, in2);
    }
    if (rank == 0) {
      if (n <= kWarpList) {
        if (threadIdx.x < 32) {
          sort<true>(sh.list, n);
          const int c = taken_of_list<true, MASS>(n, above);
          if (threadIdx.x == 0) sh.word[0] = sh.list[max(c, 1) - 1];
        }
      } else {
        sort<false>(sh.list, n);
        const int c = taken_of_list<false, MASS>(n, above);
        if (threadIdx.x == 0) sh.word[0] = sh.list[max(c, 1) - 1];
      }
    }
    sync();
    set_edge(ranks == 1 ? sh.word[0] : *cg::this_cluster().map_shared_rank(&sh.word[0], 0));
    sync();
  }
  // The lowest number above which little enough lies, among the tokens of `in`.
  template <bool MASS, class F>
  __device__ __forceinline__ void halve(uint64_t above, F in) {
    uint64_t low = ~0ull, high = 0;
    each([&](float v, int i) {
      if (!in(v, i)) return;
      low = min(low, order_of(v, i));
      high = max(high, order_of(v, i));
    });
    low = ~largest(~low);
    high = largest(high);
    while (low < high) {
      const uint64_t mid = low + (high - low) / 2;
      uint64_t b = 0;
      each([&](float v, int i) {
        if (in(v, i) && order_of(v, i) > mid) b += MASS ? weight(v) : 1;
      });
      if (taken<MASS>(above + sum(b)))
        high = mid;
      else
        low = mid + 1;
    }
    set_edge(low);
  }
};

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  using S = Sampler<T>;
  constexpr int E = S::E;
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  const int rw = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  S s{sh, reinterpret_cast<T*>(smem + sizeof(SampleShared))};
  s.ranks = gridDim.x;
  s.rank = blockIdx.x;
  s.flip = 0;
  const int first = min(s.rank * a.part, a.vocab), n = min(a.part, a.vocab - first);  // this CTA's tokens
  const T* const row = static_cast<const T*>(a.x) + (int64_t)rw * a.row_stride + first;
  const int lead = (int)((uintptr_t)row & 15) / (int)sizeof(T);
  s.base = first - lead;
  s.pieces = (lead + n + E - 1) / E;
  float* const probs = a.probs ? a.probs + (int64_t)rw * a.vocab : nullptr;
  if (tid == 0) sh.count = 0;
  for (int i = tid; i < kSteps; i += kSampleThreads) sh.lo[i] = sh.hi[i] = 0;
  // ---- the row, and every thread's maximum
  float mine = -INFINITY;
  {
    const uint4* const from = reinterpret_cast<const uint4*>(row - lead);
    int b, e;
    s.share(b, e);
#pragma unroll 4
    for (int c = b + lane; c < e; c += 32) {
      uint4 u;
      if (c * E >= lead && (c + 1) * E <= lead + n) {
        u = __ldcs(from + c);
      } else {  // the row ends within this piece: token by token
        T v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int i = c * E + j - lead;
          v[j] = i >= 0 && i < n ? row[i] : from_f32<T>(-INFINITY);
        }
        u = *reinterpret_cast<const uint4*>(v);
      }
      reinterpret_cast<uint4*>(s.x)[c] = u;
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < E; ++j) mine = fmaxf(mine, to_f32(t[j]));  // not NaN's
    }
  }
  if (s.ranks > 1) s.sync();  // every CTA of the cluster runs before its memory is written
  s.m = of_key((uint32_t)s.largest(key_of(mine)));
  const float min_p = a.min_p ? a.min_p[rw] : 0.f, t = a.temperature ? a.temperature[rw] : 1.f;
  s.least = (double)min_p * (double)kOne;
  if (s.m == -INFINITY || min_p > 1.f) {  // no token to draw
    if (s.rank == 0 && tid == 0) {
      a.id[rw] = -1;
      if (a.logprob) a.logprob[rw] = -INFINITY;
      if (a.kept) a.kept[rw] = 0;
    }
    if (probs)
      for (int i = tid; i < n; i += kSampleThreads) probs[first + i] = 0.f;
    if (s.ranks > 1) s.sync();  // no CTA leaves while another may still write its words
    return;
  }
  const bool greedy = !(t > 0.f);
  s.r = greedy ? 1.f : __fdiv_rn(1.f, t);
  int k = greedy ? 1 : (a.top_k ? a.top_k[rw] : 0);
  if (k <= 0 || k > a.vocab) k = a.vocab;
  s.k = k;
  s.p = a.top_p ? a.top_p[rw] : 1.f;
  s.xe = -INFINITY;  // every token that weighs anything
  s.ie = -1;

  // ---- the edge: tokens at or above it are kept
  bool listed = false;  // the first CTA's list holds the top k
  if (k < a.vocab && k <= kSampleMaxK) {
    // the step in which the k-th largest of the threads' maxima lies, and all that is above it
    float to = 0.f;
    if (k == 1) {
      to = -1e-30f;
    } else {
      const float g = s.gap(mine);
      if (g > kFar) atomicAdd(&sh.lo[(uint32_t)(g * -16.f)], 1u);
      uint64_t above = 0;
      to = -0.0625f * (float)(s.template pick<false, false>(above) + 1);
      if (s.total < s.k) to = kFar;  // fewer threads than k hold a token of weight
    }
    const int c = s.gather([&](float v, int) {
      const float g = s.gap(v);
      return g > to && g > kFar;
    });
    if (c <= kSampleList) {
      listed = true;
      if (s.rank == 0) {
        if (c > kWarpList)
          s.template finish_list<false>(a, rw, c);
        else if (tid < 32)
          s.template finish_list<true>(a, rw, c);
      }
    }
  }
  uint64_t z = 0;
  if (listed) {
    if (probs) {
      s.sync();
      const uint64_t* word = s.ranks == 1 ? sh.word : cg::this_cluster().map_shared_rank(sh.word, 0);
      s.set_edge(word[0]);
      z = word[1];
    }
  } else {
    if (k < a.vocab) s.template find_edge<false>();
    if (!(s.p >= 1.f)) s.template find_edge<true>();
    // ---- the kept weight Z, and the token in index order where the running weight passes floor(u Z).  Few
    // tokens are kept as a rule: a thread marks its own first, then weighs those.
    auto kept_weight = [&](float v, int i) -> uint64_t {
      if (!s.above_edge(v, i)) return 0;
      const uint64_t w = s.weight(v);
      return (double)w >= s.least ? w : 0;
    };
    int b, e;
    s.share(b, e);
    uint64_t v = 0, some = 0;
    constexpr int kMark = 32 / E;  // pieces of a mask
    for (int c0 = b + lane; c0 < e; c0 += 32 * kMark) {
      uint32_t mask = 0;
#pragma unroll
      for (int q = 0; q < kMark; ++q) {
        const int c = c0 + 32 * q;
        if (c >= e) break;
        float f[E];
        s.piece(c, f);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (s.above_edge(f[j], s.base + c * E + j)) mask |= 1u << (q * E + j);
      }
      while (mask) {
        const int bit = __ffs((int)mask) - 1;
        mask &= mask - 1;
        const uint64_t w = s.weight(to_f32(s.x[(c0 + 32 * (bit / E)) * E + bit % E]));
        if ((double)w < s.least) continue;
        v += w;
        some += w > 0;
      }
    }
    const uint64_t kept = s.sum(some);
    uint64_t all;
    uint64_t ahead = s.template before<false>(v, all);
    z = s.combine(all, [](uint64_t x, uint64_t y) { return x + y; });
    for (int c = 0; c < s.rank; ++c) ahead += sh.slot[s.flip][c];
    ahead = __shfl_sync(0xffffffffu, ahead, 0);  // before this warp's share
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    uint64_t aim = s.aim(a.u[rw], z);
    if (ahead <= aim && aim < ahead + v) {  // one warp of one CTA: the place in its share
      aim -= ahead;
      for (int c = b; c < e; c += 32) {
        float f[E];
        uint64_t w[E], own = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) w[j] = 0;
        if (c + lane < e) {
          s.piece(c + lane, f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            w[j] = kept_weight(f[j], s.base + (c + lane) * E + j);
            own += w[j];
          }
        }
        uint64_t sum;
        uint64_t before = s.template before<true>(own, sum);
        if (aim < sum) {
          if (before <= aim && aim < before + own) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
              if (before <= aim && aim < before + w[j]) s.answer(a, rw, s.base + (c + lane) * E + j, f[j], z, kept);
              before += w[j];
            }
          }
          break;
        }
        aim -= sum;
      }
    }
  }
  if (probs) {
    const float zf = (float)z;
    for (int i = tid; i < n; i += kSampleThreads) {
      const float v = to_f32(s.x[lead + i]);
      float q = 0.f;
      if (s.above_edge(v, first + i)) {
        const uint64_t w = s.weight(v);
        if ((double)w >= s.least) q = __fdiv_rn((float)w, zf);
      }
      probs[first + i] = q;
    }
  }
  if (s.ranks > 1) s.sync();  // no CTA leaves while another may still read or write its words
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
  const SampleArgs a = {d_logits, row_stride, vocab, 0, d_temperature, d_top_k, d_top_p, d_min_p, d_u, d_id, d_logprob,
                        d_kept, d_probs};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16) return launch_sample<__half>(a, rows, st);
  if (dtype == MLLM_DTYPE_BF16) return launch_sample<__nv_bfloat16>(a, rows, st);
  return launch_sample<float>(a, rows, st);
}
