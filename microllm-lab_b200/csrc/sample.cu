// Sampling with temperature, top-k, top-p and min-p from one given uniform number per row (mllm_sample).
//
// With x the row (NaN as -inf), m its maximum and r = 1 / T, token i weighs w_i = floor(2^40 exp((x_i - m) r)).
// Sorting is not needed: the tokens that top-k and top-p keep are those above a boundary value and, of
// those equal to it, the first few by index.  The boundary is found digit by digit on order-preserving
// integer keys of x, counting tokens (top-k) or adding their weights (top-p).  The id is then found in
// index order: the part of the row where the running weight passes floor(u Z), then the place in it.
// Weights are integers of at most 2^40 (a sum of 2^19 of them fits 64 bits), so every sum is exact and no
// result depends on the order in which threads add.  The 2^-40 that a weight loses is 2^-40 of the top
// token's: over 2^18 tokens at most 2^-22 of the row, the size of an f32 rounding.
//
// One CTA per row; each warp owns a contiguous part of the row, lanes take neighbouring elements.
#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr float kOne = 1099511627776.f;  // 2^40

// Order-preserving key: a < b as floats iff key(a) < key(b); -0 counts as +0, NaN as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kKeyNone = 0x007FFFFFu;  // key of -inf
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ float gap(uint32_t k, uint32_t top, float r) {
  return k == top ? 0.f : __fmul_rn(__fsub_rn(of_key(k), of_key(top)), r);
}
__device__ __forceinline__ uint64_t weight(uint32_t k, uint32_t top, float r) {
  if (k == kKeyNone) return 0;
  return (uint64_t)__fmul_rn(expf(gap(k, top, r)), kOne);
}

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct SampleArgs {
  const void* x;
  int64_t row_stride;
  int vocab;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *u;
  int32_t* id;
  float* logprob;
  int32_t* kept;
  float* probs;
};

// What a row's CTA shares.
struct SampleShared {
  uint64_t mass[256];
  uint32_t count[256];
  uint64_t part[kSampleWarps];
  uint64_t sum;
  int at;
  uint32_t digit;
};

template <class T>
struct Row {
  const T* x;
  int n;
  __device__ __forceinline__ uint32_t key(int i) const { return key_of(to_f32(x[i])); }
};

// Sum of f(i) over the row, on every thread.
template <class F>
__device__ uint64_t row_sum(SampleShared& sh, int n, F f) {
  uint64_t s = 0;
  for (int i = threadIdx.x; i < n; i += kSampleThreads) s += f(i);
  s = warp_sum_u64(s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
  for (int w = 0; w < kSampleWarps; ++w) s += sh.part[w];
  return s;
}

// First index at which the running sum of f over the row exceeds `aim` (the whole sum does).  Two rounds:
// the sums of the warps' parts of the row, then of the parts of that part; one warp walks the last.
template <class F>
__device__ int row_find(SampleShared& sh, int n, uint64_t aim, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  for (int round = 0; round < 2; ++round) {
    const int len = (hi - lo + kSampleWarps - 1) / kSampleWarps;
    const int b = min(lo + warp * len, hi), e = min(b + len, hi);
    uint64_t s = 0;
    for (int i = b + lane; i < e; i += 32) s += f(i);
    s = warp_sum_u64(s);
    __syncthreads();
    if (lane == 0) sh.part[warp] = s;
    __syncthreads();
    int w = 0;
    for (; w < kSampleWarps - 1; ++w) {
      if (sh.part[w] > aim) break;
      aim -= sh.part[w];
    }
    const int l0 = lo;
    lo = min(l0 + w * len, hi);
    hi = min(lo + len, hi);
  }
  __syncthreads();
  if (warp == 0) {
    int found = hi - 1;
    for (int b = lo; b < hi; b += 32) {
      const uint64_t v = b + lane < hi ? f(b + lane) : 0;
      uint64_t run = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, run > aim);
      if (past) {
        found = b + __ffs(past) - 1;
        break;
      }
      aim -= __shfl_sync(0xffffffffu, run, 31);
    }
    if (lane == 0) sh.at = found;
  }
  __syncthreads();
  return sh.at;
}

// The last key, counted from the top, whose first token is still taken: taken(b) says whether a token with
// b (tokens, or weight) before it is, and holds for b = 0.  Only tokens with in(i, key) count.  `above` is
// what lies above the returned key, `equal` the number of tokens at it.
template <bool MASS, class R, class In, class Taken>
__device__ uint32_t boundary(SampleShared& sh, const R& row, uint32_t top, float r, In in, Taken taken, uint64_t& above,
                             uint32_t& equal) {
  uint32_t prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kSampleThreads) {
      sh.mass[i] = 0;
      sh.count[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < row.n; i += kSampleThreads) {
      const uint32_t k = row.key(i);
      if (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8))) continue;
      if (!in(i, k)) continue;
      const uint32_t d = (k >> shift) & 255u;
      atomicAdd(&sh.count[d], 1u);
      if (MASS) atomicAdd((unsigned long long*)&sh.mass[d], (unsigned long long)weight(k, top, r));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t before = above;
      for (int d = 255; d >= 0; --d) {
        if (!sh.count[d]) continue;
        if (!taken(before)) break;
        sh.digit = d;
        sh.sum = before;
        before += MASS ? sh.mass[d] : sh.count[d];
      }
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    above = sh.sum;
    equal = sh.count[sh.digit];
  }
  return prefix;
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  __shared__ SampleShared sh;
  const int rw = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> row{static_cast<const T*>(a.x) + (int64_t)rw * a.row_stride, a.vocab};
  const int n = row.n;
  float* probs = a.probs ? a.probs + (int64_t)rw * n : nullptr;
  // ---- the maximum
  uint32_t top = 0;
  for (int i = tid; i < n; i += kSampleThreads) top = max(top, row.key(i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sh.count[warp] = top;
  __syncthreads();
  for (int w = 0; w < kSampleWarps; ++w) top = max(top, sh.count[w]);
  auto none = [&] {  // no token to draw
    if (tid == 0) {
      a.id[rw] = -1;
      if (a.logprob) a.logprob[rw] = -INFINITY;
      if (a.kept) a.kept[rw] = 0;
    }
    if (probs)
      for (int i = tid; i < n; i += kSampleThreads) probs[i] = 0.f;
  };
  if (top == kKeyNone) return none();
  const float t = a.temperature ? a.temperature[rw] : 1.f;
  const bool greedy = !(t > 0.f);
  const float r = greedy ? 1.f : __fdiv_rn(1.f, t);
  int k = greedy ? 1 : (a.top_k ? a.top_k[rw] : 0);
  if (k <= 0 || k > n) k = n;
  const float p = a.top_p ? a.top_p[rw] : 1.f;
  const double least = (double)(a.min_p ? a.min_p[rw] : 0.f) * (double)kOne;
  // ---- the boundary: tokens above `edge` are kept, of those equal to it the ones up to index `last`
  uint32_t edge = 0;
  int last = n;
  auto in = [&](int i, uint32_t key) { return key > edge || (key == edge && i <= last); };
  auto cut = [&](uint32_t key, uint64_t ties) {  // the first `ties` of the kept tokens equal to `key` stay
    const int at = row_find(sh, n, ties - 1, [&](int i) { return (uint64_t)(row.key(i) == key); });
    last = key == edge ? min(last, at) : at;
    edge = key;
  };
  if (k < n) {
    uint64_t above;
    uint32_t equal;
    const uint32_t key = boundary<false>(sh, row, top, r, in, [&](uint64_t b) { return b < (uint64_t)k; }, above, equal);
    cut(key, min((uint64_t)equal, (uint64_t)k - above));
  }
  if (!(p >= 1.f)) {
    const uint64_t total = row_sum(sh, n, [&](int i) {
      const uint32_t key = row.key(i);
      return in(i, key) ? weight(key, top, r) : 0;
    });
    const double want = (double)p * (double)total;
    auto taken = [&](uint64_t b) { return b == 0 || (double)b < want; };
    uint64_t above;
    uint32_t equal;
    const uint32_t key = boundary<true>(sh, row, top, r, in, taken, above, equal);
    const uint64_t w = weight(key, top, r);
    uint32_t lo = 1, hi = equal;  // how many of the equal ones are taken: at least one
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1) / 2;
      if (taken(above + (mid - 1) * w))
        lo = mid;
      else
        hi = mid - 1;
    }
    cut(key, lo);
  }
  auto kept_weight = [&](int i) -> uint64_t {
    const uint32_t key = row.key(i);
    if (!in(i, key)) return 0;
    const uint64_t w = weight(key, top, r);
    return (double)w >= least ? w : 0;
  };
  // ---- the kept weight, and the place where the running weight passes floor(u Z)
  const uint64_t z = row_sum(sh, n, kept_weight);
  if (z == 0) return none();  // min_p above 1
  const uint64_t kept = row_sum(sh, n, [&](int i) { return (uint64_t)(kept_weight(i) > 0); });
  const float u = a.u[rw];
  const uint64_t aim = u > 0.f ? min((uint64_t)((double)u * (double)z), z - 1) : 0;
  const int id = row_find(sh, n, aim, kept_weight);
  if (tid == 0) {
    a.id[rw] = id;
    if (a.kept) a.kept[rw] = (int32_t)kept;
    if (a.logprob) a.logprob[rw] = gap(row.key(id), top, r) - logf(__fdiv_rn((float)(double)z, kOne));
  }
  if (probs) {
    const float zf = (float)z;
    for (int i = tid; i < n; i += kSampleThreads) probs[i] = __fdiv_rn((float)kept_weight(i), zf);
  }
}

template <class T>
void launch_sample(const SampleArgs& a, int rows, cudaStream_t st) {
  sample_kernel<T><<<rows, kSampleThreads, 0, st>>>(a);
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
  if (rows < 0 || vocab < 1 || row_stride < vocab)
    return refuse(MLLM_ERR_ARG, "mllm_sample: negative rows, an empty vocabulary, or a row stride below it");
  if (vocab > 524288) return refuse(MLLM_ERR_UNSUPPORTED, "mllm_sample: vocab above 524,288");
  if (rows == 0) return MLLM_OK;
  if (!d_logits || !d_u || !d_id) return refuse(MLLM_ERR_ARG, "mllm_sample: null pointer");
  if ((uintptr_t)d_logits % esize(dtype)) return refuse(MLLM_ERR_ARG, "mllm_sample: misaligned logits");
  const SampleArgs a = {d_logits, row_stride, vocab, d_temperature, d_top_k, d_top_p, d_min_p, d_u, d_id, d_logprob,
                        d_kept, d_probs};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16)
    launch_sample<__half>(a, rows, st);
  else if (dtype == MLLM_DTYPE_BF16)
    launch_sample<__nv_bfloat16>(a, rows, st);
  else
    launch_sample<float>(a, rows, st);
  return launched("mllm_sample: launch failed");
}
