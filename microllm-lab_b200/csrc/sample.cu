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
//   - top_k up to 512: the k-th largest of the threads' own maxima bounds the k-th token from below, so the
//     few tokens at or above it are gathered, and everything else happens in that list;
//   - otherwise by a histogram of tokens or weight over x in two levels of 512 steps (of 1/16, then 1/8192
//     of a unit of (x - m) r), then among the tokens of one step;
//   - and by halving, one pass per bit, where a list would not fit (thousands of tokens of one value).
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
constexpr int kSampleMaxK = 512;    // top_k that starts from the threads' maxima
constexpr int kSampleSteps = 512;   // steps of a histogram level
constexpr int kMaxCluster = 16;
constexpr float kOne = 1099511627776.f;  // 2^40
constexpr uint32_t kKeyNone = 0x007FFFFFu;  // key of -inf

// Order-preserving key: a < b as floats iff key(a) < key(b); -0 counts as +0, NaN as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint64_t order_of(uint32_t key, uint32_t i) { return (uint64_t)key << 32 | (uint32_t)~i; }

// Scale of a row: its maximum and 1 / T.
struct Scale {
  uint32_t top;
  float m, r;
  // (x - m) / T; the top itself may be infinite
  __device__ __forceinline__ float gap(uint32_t k) const { return k == top ? 0.f : __fmul_rn(__fsub_rn(of_key(k), m), r); }
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    const float e = expf(gap(k));
    return k != kKeyNone && e > 0.f ? (uint64_t)__fmul_rn(e, kOne) : 0;  // not for NaN: an infinite gap times 1 / T = 0
  }
  // Step of 1/8192 below the maximum; the last one holds all that weighs nothing (beyond 40 ln 2 = 27.7).
  __device__ __forceinline__ uint32_t step(uint32_t k) const {
    const float d = gap(k) * -8192.f;
    return d < (float)(kSampleSteps * kSampleSteps - 1) ? (uint32_t)d : kSampleSteps * kSampleSteps - 1;
  }
};
constexpr uint32_t kLastStep = kSampleSteps * kSampleSteps - 1;

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
  uint32_t lo[kSampleSteps], hi[kSampleSteps];  // a histogram of 64-bit sums
  uint64_t slot[2][kMaxCluster];                // one word from every CTA of the cluster
  uint64_t wsum[kSampleWarps], wbase[kSampleWarps];
  uint64_t word[2];  // what the first CTA has decided
  uint32_t pick;
};

template <class T>
struct Sampler {
  SampleShared& sh;
  const T* x;        // this CTA's part of the row
  int n, base, ranks, rank;
  int flip = 0;      // slot in use
  Scale sc;

  __device__ __forceinline__ uint32_t key(int i) const { return key_of(to_f32(x[i])); }
  __device__ __forceinline__ void sync() const {
    if (ranks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  // One word of every CTA, on every thread, combined in the order of the CTAs.
  template <class F>
  __device__ __forceinline__ uint64_t combine(uint64_t v, F f) {  // v: of thread 0
    flip ^= 1;
    if (threadIdx.x == 0) {
      if (ranks == 1) {
        sh.slot[flip][0] = v;
      } else {
        for (int k = 0; k < ranks; ++k) *cg::this_cluster().map_shared_rank(&sh.slot[flip][rank], k) = v;
      }
    }
    sync();
    v = sh.slot[flip][0];
    for (int k = 1; k < ranks; ++k) v = f(v, sh.slot[flip][k]);
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
  // Sum of what lies before this thread in the CTA (threads in order); `all`: of the whole CTA.
  __device__ __forceinline__ uint64_t before(uint64_t v, uint64_t& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
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
      if (lane == 31) sh.word[1] = t;
    }
    __syncthreads();
    all = sh.word[1];
    return sh.wbase[warp] + run - v;
  }
  // The words that the first CTA wrote into sh.word, on every CTA.
  __device__ __forceinline__ uint64_t decided() {
    sync();
    const uint64_t w = ranks == 1 ? sh.word[0] : *cg::this_cluster().map_shared_rank(&sh.word[0], 0);
    sync();
    return w;
  }

  // Warp w's contiguous share of the part.
  __device__ __forceinline__ void share(int& b, int& e) const {
    const int len = ((n + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32;
    b = min((int)(threadIdx.x >> 5) * len, n);
    e = min(b + len, n);
  }
  // Gathers (key, ~index) of the tokens with f(key, index) into the first CTA's list, in index order.
  // Returns their number; nothing is written when the list cannot hold them.
  template <class F>
  __device__ __forceinline__ int gather(F f) {
    const int lane = threadIdx.x & 31;
    int b, e, count = 0;
    share(b, e);
    for (int i = b; i < e; i += 32) {
      const int at = i + lane;
      bool in = false;
      if (at < e) in = f(key(at), base + at);
      count += __popc(__ballot_sync(0xffffffffu, in));
    }
    uint64_t mine;
    int place = (int)before(lane == 0 ? count : 0, mine);
    place = __shfl_sync(0xffffffffu, place, 0);
    const uint64_t all = combine(mine, [](uint64_t a, uint64_t c) { return a + c; });
    for (int k = 0; k < rank; ++k) place += (int)sh.slot[flip][k];
    if (all <= kSampleList) {
      uint64_t* list = ranks == 1 ? sh.list : cg::this_cluster().map_shared_rank(sh.list, 0);
      for (int i = b; i < e; i += 32) {
        const int at = i + lane;
        uint32_t k = 0;
        bool in = false;
        if (at < e) {
          k = key(at);
          in = f(k, base + at);
        }
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (in) list[place + __popc(who & ((1u << lane) - 1))] = order_of(k, base + at);
        place += __popc(who);
      }
    }
    sync();
    return (int)min(all, (uint64_t)0x7FFFFFFF);
  }
  // Sorts list[0 .. m) of this CTA to falling order.
  __device__ void sort_list(int m) {
    int size = 32;
    while (size < m) size <<= 1;
    for (int i = m + threadIdx.x; i < size; i += kSampleThreads) sh.list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1) {
      for (int j = k >> 1; j >= 32; j >>= 1) {
        for (int t = threadIdx.x; t < size / 2; t += kSampleThreads) {
          const int a = 2 * t - (t & (j - 1)), b = a + j;
          const uint64_t u = sh.list[a], v = sh.list[b];
          if ((u < v) == ((a & k) == 0)) {
            sh.list[a] = v;
            sh.list[b] = u;
          }
        }
        __syncthreads();
      }
      for (int t = threadIdx.x; t < size; t += kSampleThreads) {  // strides within a warp
        uint64_t v = sh.list[t];
        for (int j = min(k >> 1, 16); j > 0; j >>= 1) {
          const uint64_t u = __shfl_xor_sync(0xffffffffu, v, j);
          const bool big = ((t & j) == 0) == ((t & k) == 0);  // this place takes the larger
          v = (u > v) == big ? u : v;
        }
        sh.list[t] = v;
      }
      __syncthreads();
    }
  }
  // For a falling list of m tokens: how many are taken, where taken(b) says whether one with measure b
  // before it is (it holds for none before, and never again once it does not).
  template <bool MASS, class Taken>
  __device__ int taken_of_list(int m, uint64_t above, Taken taken) {
    constexpr int kEach = kSampleList / kSampleThreads;
    const int i0 = threadIdx.x * kEach;
    uint64_t w[kEach], mine = 0, all;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      w[e] = i0 + e < m ? (MASS ? sc.weight((uint32_t)(sh.list[i0 + e] >> 32)) : 1) : 0;
      mine += w[e];
    }
    uint64_t b = above + before(mine, all);
    int yes = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      yes += i0 + e < m && taken(b);
      b += w[e];
    }
    return count_of(yes);
  }
  __device__ __forceinline__ int count_of(int v) {
    uint64_t all;
    (void)before((uint64_t)v, all);
    return (int)all;
  }

  // Histogram step: adds v to the 64-bit sum of step s.  The carry out of the low word is seen by the one
  // thread that caused it, so the sum is exact.
  __device__ __forceinline__ void add(uint32_t s, uint64_t v) {
    const uint32_t l = (uint32_t)v;
    const uint32_t was = atomicAdd(&sh.lo[s], l);
    const uint32_t h = (uint32_t)(v >> 32) + (was + l < l);
    if (h) atomicAdd(&sh.hi[s], h);
  }
  // One level: the last step, counted from the top, before which little enough lies, of the tokens with
  // f(key, index, step) (which also gives the token's step of this level).  `above`: what lies before it.
  template <bool MASS, class F, class Taken>
  __device__ uint32_t level(uint64_t& above, F f, Taken taken) {
    __syncthreads();
    for (int i = threadIdx.x; i < kSampleSteps; i += kSampleThreads) sh.lo[i] = sh.hi[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      const uint32_t k = key(i);
      uint32_t s;
      if (!f(k, base + i, s)) continue;
      if (MASS) {
        const uint64_t w = sc.weight(k);
        if (w) add(s, w);
      } else {
        atomicAdd(&sh.lo[s], 1u);
      }
    }
    sync();
    uint64_t v = 0, all;
    if (threadIdx.x < kSampleSteps) {
      for (int c = 0; c < ranks; ++c) {  // every CTA sums all: none has to tell the others
        const SampleShared* o = ranks == 1 ? &sh : cg::this_cluster().map_shared_rank(&sh, c);
        v += (uint64_t)o->hi[threadIdx.x] << 32 | o->lo[threadIdx.x];
      }
    }
    if (threadIdx.x == 0) sh.pick = 0;
    const uint64_t b = above + before(v, all);
    if (v && taken(b)) atomicMax(&sh.pick, threadIdx.x);
    __syncthreads();
    const uint32_t s = sh.pick;
    if (threadIdx.x == s) sh.word[0] = b;
    sync();  // also: the other CTAs have read this one's sums
    above = sh.word[0];
    return s;
  }
  // The edge among the tokens at or above `edge`: see taken_of_list.
  template <bool MASS, class Taken>
  __device__ uint64_t find_edge(uint64_t edge, Taken taken) {
    uint64_t above = 0;
    const uint32_t s1 = level<MASS>(above, [&](uint32_t k, int i, uint32_t& s) {
      const uint32_t t = sc.step(k);
      s = t / kSampleSteps;
      return t != kLastStep && order_of(k, i) >= edge;
    }, taken);
    const uint32_t s2 = level<MASS>(above, [&](uint32_t k, int i, uint32_t& s) {
      const uint32_t t = sc.step(k);
      s = t % kSampleSteps;
      return t / kSampleSteps == s1 && t != kLastStep && order_of(k, i) >= edge;
    }, taken);
    const uint32_t want = s1 * kSampleSteps + s2;
    auto in = [&](uint32_t k, int i) { return sc.step(k) == want && order_of(k, i) >= edge; };
    const int m = gather(in);
    if (m <= kSampleList) {
      if (rank == 0) {
        sort_list(m);
        const int c = taken_of_list<MASS>(m, above, taken);
        if (threadIdx.x == 0) sh.word[0] = sh.list[max(c, 1) - 1];
      }
      return decided();
    }
    // halving: the lowest number above which little enough lies
    uint64_t low = ~0ull, high = 0;  // of the tokens of this step
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      const uint32_t k = key(i);
      if (!in(k, base + i)) continue;
      low = min(low, order_of(k, base + i));
      high = max(high, order_of(k, base + i));
    }
    low = ~largest(~low);
    high = largest(high);
    while (low < high) {
      const uint64_t mid = low + (high - low) / 2;
      uint64_t v = 0;
      for (int i = threadIdx.x; i < n; i += kSampleThreads) {
        const uint32_t k = key(i);
        if (order_of(k, base + i) > mid && in(k, base + i)) v += MASS ? sc.weight(k) : 1;
      }
      if (taken(above + sum(v)))
        high = mid;
      else
        low = mid + 1;
    }
    return low;
  }
};

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  T* const x = reinterpret_cast<T*>(smem + sizeof(SampleShared));
  const int ranks = gridDim.x, rank = blockIdx.x, rw = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31;
  Sampler<T> s{sh, x, 0, 0, ranks, rank};
  s.base = min(rank * a.part, a.vocab);
  s.n = min(a.part, a.vocab - s.base);
  const int n = s.n;
  float* const probs = a.probs ? a.probs + (int64_t)rw * a.vocab + s.base : nullptr;
  // ---- the row, and every thread's maximum
  const T* const row = static_cast<const T*>(a.x) + (int64_t)rw * a.row_stride + s.base;
  uint32_t mine = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += kSampleThreads) {
    const T v = row[i];
    x[i] = v;
    mine = max(mine, key_of(to_f32(v)));
  }
  if (ranks > 1) s.sync();  // every CTA of the cluster runs before its memory is written
  s.sc.top = (uint32_t)s.largest(mine);
  s.sc.m = of_key(s.sc.top);
  s.sc.r = 1.f;
  auto none = [&] {  // no token to draw
    if (rank == 0 && tid == 0) {
      a.id[rw] = -1;
      if (a.logprob) a.logprob[rw] = -INFINITY;
      if (a.kept) a.kept[rw] = 0;
    }
    if (probs)
      for (int i = tid; i < n; i += kSampleThreads) probs[i] = 0.f;
  };
  const double least = (double)(a.min_p ? a.min_p[rw] : 0.f) * (double)kOne;
  if (s.sc.top <= kKeyNone || least > (double)kOne) {
    none();
    if (ranks > 1) s.sync();  // no CTA leaves while another may still write its words
    return;
  }
  const float t = a.temperature ? a.temperature[rw] : 1.f;
  const bool greedy = !(t > 0.f);
  if (!greedy) s.sc.r = __fdiv_rn(1.f, t);
  int k = greedy ? 1 : (a.top_k ? a.top_k[rw] : 0);
  if (k <= 0 || k > a.vocab) k = a.vocab;
  const float p = a.top_p ? a.top_p[rw] : 1.f;
  const float u = a.u[rw];

  // ---- the edge: tokens at or above it are kept
  uint64_t edge = 0;
  bool listed = false;  // the first CTA's list holds all kept tokens
  int kept_list = 0;
  if (k < a.vocab && k <= kSampleMaxK) {
    // the k-th largest of this CTA's thread maxima, to 16 bits: at least k tokens are as large
    uint32_t low = 0;
    if (k == 1) {
      low = s.sc.top;
    } else {
      for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
        if (__syncthreads_count(mine >= (low | bit)) >= k) low |= bit;
      if (ranks > 1) low = (uint32_t)s.combine(low, [](uint64_t b, uint64_t c) { return b > c ? b : c; });
    }
    low = max(low, kKeyNone + 1);
    const int m = s.gather([&](uint32_t key, int) { return key >= low; });
    if (m <= kSampleList) {
      listed = true;
      if (rank == 0) {
        s.sort_list(m);
        int c = min(m, k);
        if (!(p >= 1.f)) {
          uint64_t total = 0, all;
          for (int i = tid; i < c; i += kSampleThreads) total += s.sc.weight((uint32_t)(sh.list[i] >> 32));
          (void)s.before(total, all);
          const double want = (double)p * (double)all;
          c = max(1, s.template taken_of_list<true>(c, 0, [&](uint64_t b) { return b == 0 || (double)b < want; }));
        }
        kept_list = c;
      }
    }
  }
  if (!listed) {
    if (k < a.vocab) edge = s.template find_edge<false>(0, [&](uint64_t b) { return b < (uint64_t)k; });
    if (!(p >= 1.f)) {
      uint64_t v = 0;
      for (int i = tid; i < n; i += kSampleThreads) {
        const uint32_t key = s.key(i);
        if (order_of(key, s.base + i) >= edge) v += s.sc.weight(key);
      }
      const double want = (double)p * (double)s.sum(v);
      edge = s.template find_edge<true>(edge, [&](uint64_t b) { return b == 0 || (double)b < want; });
    }
  }
  auto kept_weight = [&](uint32_t key, int i) -> uint64_t {
    if (order_of(key, i) < edge) return 0;
    const uint64_t w = s.sc.weight(key);
    return (double)w >= least ? w : 0;
  };
  auto aim_of = [&](uint64_t z) { return u > 0.f ? min((uint64_t)((double)u * (double)z), z - 1) : 0; };
  auto answer = [&](int id, uint32_t key, uint64_t z, uint64_t kept) {
    a.id[rw] = id;
    if (a.kept) a.kept[rw] = (int32_t)kept;
    if (a.logprob) a.logprob[rw] = s.sc.gap(key) - logf(__fdiv_rn((float)(double)z, kOne));
  };
  // ---- the kept weight Z, and the token in index order where the running weight passes floor(u Z)
  uint64_t z = 0;
  if (listed) {
    if (rank == 0) {
      edge = sh.list[kept_list - 1];
      __syncthreads();
      for (int i = tid; i < kept_list; i += kSampleThreads) {  // to rising index: sorted by (~index, key)
        const uint64_t v = sh.list[i];
        sh.list[i] = v << 32 | v >> 32;
      }
      __syncthreads();
      s.sort_list(kept_list);
      constexpr int kEach = kSampleList / kSampleThreads;
      uint64_t w[kEach], mass = 0;
      int some = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = tid * kEach + e;
        w[e] = i < kept_list ? s.sc.weight((uint32_t)sh.list[i]) : 0;
        if ((double)w[e] < least) w[e] = 0;
        mass += w[e];
        some += w[e] > 0;
      }
      const uint64_t kept = s.count_of(some);
      uint64_t b = s.before(mass, z);
      const uint64_t aim = aim_of(z);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (w[e] && b <= aim && aim < b + w[e]) {
          const uint64_t v = sh.list[tid * kEach + e];
          answer((int)~(uint32_t)(v >> 32), (uint32_t)v, z, kept);
        }
        b += w[e];
      }
      if (tid == 0) {
        sh.word[0] = edge;
        sh.word[1] = z;
      }
    }
    if (probs) {
      s.sync();
      const uint64_t* word = ranks == 1 ? sh.word : cg::this_cluster().map_shared_rank(sh.word, 0);
      edge = word[0];
      z = word[1];
    }
  } else {
    int b, e;
    s.share(b, e);
    uint64_t v = 0;
    int some = 0;
    for (int i = b + lane; i < e; i += 32) {
      const uint64_t w = kept_weight(s.key(i), s.base + i);
      v += w;
      some += w > 0;
    }
    const uint64_t kept = s.sum(some);
    uint64_t all;
    uint64_t lead = s.before(v, all);  // this warp's, then the CTA's
    z = s.combine(all, [](uint64_t c, uint64_t d) { return c + d; });
    uint64_t aim = aim_of(z);
    for (int c = 0; c < rank; ++c) lead += sh.slot[s.flip][c];
    const uint64_t first = __shfl_sync(0xffffffffu, lead, 0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (first <= aim && aim < first + v) {  // one warp of one CTA: the place in its share
      aim -= first;
      for (int i = b; i < e; i += 32) {
        const uint32_t key = i + lane < e ? s.key(i + lane) : kKeyNone;
        const uint64_t w = i + lane < e ? kept_weight(key, s.base + i + lane) : 0;
        uint64_t run = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += up;
        }
        const uint64_t past = __ballot_sync(0xffffffffu, run > aim);
        if (past) {
          if (lane == __ffs((int)past) - 1) answer(s.base + i + lane, key, z, kept);
          break;
        }
        aim -= __shfl_sync(0xffffffffu, run, 31);
      }
    }
  }
  if (probs) {
    const float zf = (float)z;
    for (int i = tid; i < n; i += kSampleThreads) probs[i] = __fdiv_rn((float)kept_weight(s.key(i), s.base + i), zf);
  }
  if (ranks > 1) s.sync();  // no CTA leaves while another may still read or write its words
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
  const int64_t room = (227 * 1024 - (int64_t)sizeof(SampleShared)) / sizeof(T) / 32 * 32;
  int ranks = 1;
  while (ranks < kMaxCluster && ((int64_t)ranks * room < a.vocab || ((int64_t)rows * ranks * 2 <= sms && a.vocab / (2 * ranks) >= 4096)))
    ranks *= 2;
  a.part = ((a.vocab + ranks - 1) / ranks + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, rows);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared) + (size_t)a.part * sizeof(T);
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
