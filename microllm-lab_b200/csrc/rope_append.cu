// Position step of a paged cache (mllm_rope_append): per-head RMS norm of q and k, rotation by the
// token's position, q out, k and v into the token's page row, in one pass.
//
//   y = x / sqrt(mean x^2 + eps) * gain;   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// for the pairs (a, b) = (i, i + rope_dim / 2) or (2 i, 2 i + 1), c and s the table row of the position.
// A few operations per element: bound by the bytes read and written, or by launch latency for few rows.
// A lane holds 8 neighbouring elements of a head (one or two 16-byte accesses), as many lanes as the head
// needs share it, and a warp walks several heads of one token, so that the token's position, page and
// table row are looked up once.  The norm's sum is a shuffle among the lanes of the head.  Pairs (2 i,
// 2 i + 1) lie within a lane; pairs (i, i + rope_dim / 2) are exchanged by shuffles where rope_dim / 2 is
// whole lanes, through shared memory otherwise.
//
// B200: 24 prompts of 1,021 tokens, 15 + 2 x 5 heads of 64, f32 into bf16: 57 us (4.9 TB/s, 75 % of the measured
// copy; one element per lane and access: 258 us); one token, or 256: 7.5 us a call, most of it the caller's side.
#include <algorithm>

#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;

constexpr int kRopeWarps = 4;
enum RopePairs { kNoPairs, kAdjacent, kHalvesByLane, kAnyPairs };  // how a lane finds the partners of its elements

struct RopeArgs {
  void *k, *v;
  int64_t page_stride, head_stride, pos_stride;
  int n_pages, page_len, n_kv, dim;
  const void* qkv;
  int64_t row_stride;
  int n_tok, n_heads;
  const int32_t *seq, *pos, *table;
  int n_seq, table_stride;
  const float *q_gain, *k_gain;
  float eps;
  const float *cs, *sn;
  int n_pos, rope_dim, interleaved;
  int splits;  // warps of a token
  void* q;
  int64_t q_stride;
};

// Eight elements as they lie in memory.
template <class T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(reinterpret_cast<const T*>(u)[i]); }
};
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(e) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
}

// LANES: lanes of a head, a power of two with 8 LANES >= head_dim.
template <class A, class C, int LANES, RopePairs PAIRS>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_append_kernel(const RopeArgs a) {
  __shared__ float staged[PAIRS == kAnyPairs ? kRopeWarps : 1][PAIRS == kAnyPairs ? 256 : 1];
  constexpr int kHeads = 32 / LANES;  // heads of a warp at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kRopeWarps + warp;
  const int64_t t = unit / a.splits;
  if (t >= a.n_tok) return;
  const int seq = a.seq ? a.seq[t] : (int)t;
  const int pos = a.pos[t];
  const int per_tok = a.n_heads + 2 * a.n_kv, group = lane / LANES, d = lane % LANES * 8;
  const int step = a.splits * kHeads, h0 = (int)(unit - t * a.splits) * kHeads + group;
  const A* const x = static_cast<const A*>(a.qkv) + t * a.row_stride + d;
  A* const q = static_cast<A*>(a.q) + t * a.q_stride + d;
  const bool mine = d < a.dim;
  // the first heads' elements travel while the page is looked up, and each round's two rounds ahead
  Raw8<A> v0, v1;
  if (mine && h0 < per_tok && seq >= 0) v0.load(x + (int64_t)h0 * a.dim);
  if (mine && h0 + step < per_tok && seq >= 0) v1.load(x + (int64_t)(h0 + step) * a.dim);
  if (seq < 0) return;  // padding
  const int pg = pos / a.page_len;
  int page = -1;
  if (seq < a.n_seq && pos >= 0 && pg < a.table_stride && (pos < a.n_pos || a.rope_dim == 0))
    page = __ldg(a.table + (int64_t)seq * a.table_stride + pg);
  const bool good = (unsigned)page < (unsigned)a.n_pages;
  const int half = a.rope_dim >> 1;
  float c[8], s[8];  // of this lane's elements
  if constexpr (PAIRS == kAdjacent || PAIRS == kHalvesByLane) {
    if (good && d < a.rope_dim) {
      constexpr int N = PAIRS == kAdjacent ? 4 : 8;
      const int64_t at = (int64_t)pos * half + (PAIRS == kAdjacent ? d / 2 : (d < half ? d : d - half));
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        *reinterpret_cast<float4*>(c + i) = __ldg(reinterpret_cast<const float4*>(a.cs + at + i));
        *reinterpret_cast<float4*>(s + i) = __ldg(reinterpret_cast<const float4*>(a.sn + at + i));
      }
    }
  }
  const int64_t row = (int64_t)page * a.page_stride + (int64_t)(pos - pg * a.page_len) * a.pos_stride + d;
  for (int h = h0; h - group < per_tok; h += step) {
    const bool in = mine && h < per_tok;  // this lane has elements of a head
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = in ? v0.at(i) : 0.f;
    v0 = v1;
    if (mine && h + 2 * step < per_tok) v1.load(x + (int64_t)(h + 2 * step) * a.dim);
    if (a.q_gain) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (in && !is_v) {
        const float f = 1.f / sqrtf(ss / (float)a.dim + a.eps);
        const float* const gain = (is_q ? a.q_gain : a.k_gain) + d;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * f * __ldg(gain + i);
      }
    }
    if constexpr (PAIRS == kAdjacent) {
      if (!is_v && d < a.rope_dim) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float y0 = y[i], y1 = y[i + 1];
          y[i] = y0 * c[i / 2] - y1 * s[i / 2];
          y[i + 1] = y1 * c[i / 2] + y0 * s[i / 2];
        }
      }
    } else if constexpr (PAIRS == kHalvesByLane) {
      const int from = d < half ? lane + half / 8 : lane - half / 8;  // past rope_dim: some lane, unused
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __shfl_sync(0xffffffffu, y[i], from);
      if (!is_v && d < a.rope_dim) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = d < half ? y[i] * c[i] - p[i] * s[i] : y[i] * c[i] + p[i] * s[i];
      }
    } else if constexpr (PAIRS == kAnyPairs) {
      float* const st = staged[warp] + group * LANES * 8;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) st[d + i] = y[i];
      __syncwarp();
      if (good && !is_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = d + i;
          if (e >= a.rope_dim) continue;
          const bool second = a.interleaved ? e & 1 : e >= half;
          const int at = a.interleaved ? e >> 1 : (second ? e - half : e);
          const float p = st[a.interleaved ? e ^ 1 : (second ? e - half : e + half)];
          const float co = __ldg(a.cs + (int64_t)pos * half + at), si = __ldg(a.sn + (int64_t)pos * half + at);
          y[i] = second ? y[i] * co + p * si : y[i] * co - p * si;
        }
      }
    }
    if (!in) continue;
    if (is_q) {
      if (!good) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __int_as_float(0x7FC00000);
      }
      store8(q + (int64_t)h * a.dim, y);
    } else if (good) {
      C* const pool = static_cast<C*>(is_v ? a.v : a.k);
      store8(pool + row + (int64_t)(h - a.n_heads - (is_v ? a.n_kv : 0)) * a.head_stride, y);
    }
  }
}

template <class A, class C, int LANES>
void launch_rope(const RopeArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)(((int64_t)a.n_tok * a.splits + kRopeWarps - 1) / kRopeWarps)), block(kRopeWarps * 32);
  const int half = a.rope_dim / 2;
  // the tables' rows on 16-byte boundaries, and whole lanes on either side of every pair
  const bool rows = half % 4 == 0 && !((uintptr_t)a.cs & 15) && !((uintptr_t)a.sn & 15);
  if (a.rope_dim == 0)
    rope_append_kernel<A, C, LANES, kNoPairs><<<grid, block, 0, st>>>(a);
  else if (a.interleaved && rows)
    rope_append_kernel<A, C, LANES, kAdjacent><<<grid, block, 0, st>>>(a);
  else if (!a.interleaved && rows && half % 8 == 0)
    rope_append_kernel<A, C, LANES, kHalvesByLane><<<grid, block, 0, st>>>(a);
  else
    rope_append_kernel<A, C, LANES, kAnyPairs><<<grid, block, 0, st>>>(a);
}

template <class A, class C>
void launch_rope(RopeArgs a, cudaStream_t st) {
  const int lanes = a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : 32;
  // warps of a token: one round of heads each while there are few tokens, so that latency is not paid twice;
  // fewer, with the token's lookups shared, once there are warps enough to fill the device
  const int rounds = (a.n_heads + 2 * a.n_kv + 32 / lanes - 1) / (32 / lanes);
  a.splits = std::max(1, std::min<int>(rounds, 148 * 32 / a.n_tok));
  if (lanes == 8)
    launch_rope<A, C, 8>(a, st);
  else if (lanes == 16)
    launch_rope<A, C, 16>(a, st);
  else
    launch_rope<A, C, 32>(a, st);
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_rope_append(const mllm_paged_kv* kv, int dtype, const void* d_qkv, int64_t row_stride, int n_tok,
                                int n_heads, const int32_t* d_seq, const int32_t* d_pos, const int32_t* d_table,
                                int n_seq, int table_stride, const float* d_q_gain, const float* d_k_gain, float eps,
                                const float* d_cos, const float* d_sin, int n_pos, int rope_dim, int interleaved,
                                void* d_q, int64_t q_stride, void* stream) {
  using namespace mllm;
  using namespace mllm::paged;
  if (int rc = check_kv(kv)) return rc;
  if (!is_float_kind(dtype) || (dtype != MLLM_DTYPE_F32 && dtype != kv->dtype))
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_rope_append: activations must be f32 or of the cache's type");
  if (n_tok < 0 || n_heads < 1 || n_seq < 1 || table_stride < 1)
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: negative rows, or non-positive heads, sequences or table width");
  if (!d_qkv || !d_pos || !d_table || !d_q) return refuse(MLLM_ERR_ARG, "mllm_rope_append: null pointer");
  if (!d_q_gain != !d_k_gain) return refuse(MLLM_ERR_ARG, "mllm_rope_append: one gain without the other");
  if (rope_dim < 0 || rope_dim > kv->head_dim || rope_dim % 2)
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: rope_dim must be even, 0 to head_dim");
  if (rope_dim && (!d_cos || !d_sin || n_pos < 1)) return refuse(MLLM_ERR_ARG, "mllm_rope_append: no rotation tables");
  const int es = esize(dtype);
  const int64_t width = (int64_t)(n_heads + 2 * (int64_t)kv->n_kv_heads) * kv->head_dim;
  if (row_stride < width || q_stride < (int64_t)n_heads * kv->head_dim)
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: a row stride is shorter than a row");
  if (((uintptr_t)d_qkv & 15) || ((uintptr_t)d_q & 15) || row_stride * es % 16 || q_stride * es % 16)
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: rows must be 16-byte aligned");
  const int64_t row_heads = width / kv->head_dim;
  if (row_heads > (int64_t)1 << 30)  // a warp counts them in 31 bits, two rounds ahead
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: more than 2^30 heads in a row");
  if (n_tok * row_heads > (int64_t)1 << 31)
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: more than 2^31 heads in one call");
  if (n_tok == 0) return MLLM_OK;
  const RopeArgs a = {kv->k, kv->v, kv->page_stride, kv->head_stride, kv->pos_stride, kv->n_pages, kv->page_len,
                      kv->n_kv_heads, kv->head_dim, d_qkv, row_stride, n_tok, n_heads, d_seq, d_pos, d_table,
                      n_seq, table_stride, d_q_gain, d_k_gain, eps, d_cos, d_sin, n_pos, rope_dim,
                      interleaved != 0, 1, d_q, q_stride};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16)
    launch_rope<__half, __half>(a, st);
  else if (dtype == MLLM_DTYPE_BF16)
    launch_rope<__nv_bfloat16, __nv_bfloat16>(a, st);
  else if (kv->dtype == MLLM_DTYPE_F16)
    launch_rope<float, __half>(a, st);
  else if (kv->dtype == MLLM_DTYPE_BF16)
    launch_rope<float, __nv_bfloat16>(a, st);
  else
    launch_rope<float, float>(a, st);
  return launched("mllm_rope_append: launch failed");
}
