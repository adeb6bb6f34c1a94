// Attention of one new token per sequence over a paged K/V cache (mllm_paged_attn).
//
//   out = sum_p softmax_p(scale q . k_p) v_p,   lse = log sum_p exp(scale q . k_p)
//
// Two multiply-adds per cached element and query head of its group: bound by the bytes of the cache.
// One pass with the running maximum m and sum l of the softmax: a new score s turns (m, l, o) into
// (m', l e^(m - m') + e^(s - m'), o e^(m - m') + e^(s - m') v).  One CTA per query head; its warps take
// every fourth position and join their (m, l, o) at the end.
#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;

constexpr int kAttnWarps = 4;

struct AttnArgs {
  const void *k, *v;
  int64_t page_stride, head_stride, pos_stride;
  int n_pages, page_len, n_kv, dim;
  const void* q;
  int64_t q_stride;
  int n_seq, n_heads;
  const int32_t *len, *table;
  int table_stride;
  float scale;
  void* out;
  int64_t out_stride;
  float* lse;
};

template <class A, class C>
__global__ void __launch_bounds__(kAttnWarps * 32) paged_attn_kernel(const AttnArgs a) {
  __shared__ float sm[kAttnWarps], sl[kAttnWarps], so[kAttnWarps][256];
  __shared__ int bad;
  const int s = blockIdx.y, h = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = h / (a.n_heads / a.n_kv);
  const A* q = static_cast<const A*>(a.q) + s * a.q_stride + (int64_t)h * a.dim;
  const int len = max(a.len[s], 0);
  if (threadIdx.x == 0) bad = (int64_t)len > (int64_t)a.table_stride * a.page_len;
  __syncthreads();
  const int n = bad ? 0 : len;
  float qv[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    qv[i] = lane + 32 * i < a.dim ? to_f32(q[lane + 32 * i]) : 0.f;
    o[i] = 0.f;
  }
  for (int p = warp; p < n; p += kAttnWarps) {
    const int pg = p / a.page_len;
    const int page = a.table[(int64_t)s * a.table_stride + pg];
    if (page < 0 || page >= a.n_pages) {
      bad = 1;
      break;
    }
    const int64_t at = page * a.page_stride + hk * a.head_stride + (int64_t)(p - pg * a.page_len) * a.pos_stride;
    const C* kr = static_cast<const C*>(a.k) + at;
    const C* vr = static_cast<const C*>(a.v) + at;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) x = fmaf(qv[i], to_f32(kr[lane + 32 * i]), x);
    x = warp_sum(x) * a.scale;
    const float mn = fmaxf(m, x);
    const float keep = mn == -INFINITY ? 1.f : expf(m - mn), e = mn == -INFINITY ? 0.f : expf(x - mn);
    l = fmaf(l, keep, e);
    m = mn;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.dim) o[i] = fmaf(o[i], keep, e * to_f32(vr[lane + 32 * i]));
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, sm[w]);
  float f[kAttnWarps];
  for (int w = 0; w < kAttnWarps; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : expf(sm[w] - top);
    sum = fmaf(f[w], sl[w], sum);
  }
  const float nan = __int_as_float(0x7FC00000);
  A* out = static_cast<A*>(a.out) + s * a.out_stride + (int64_t)h * a.dim;
  for (int d = threadIdx.x; d < a.dim; d += kAttnWarps * 32) {
    float r = 0.f;
    for (int w = 0; w < kAttnWarps; ++w) r = fmaf(f[w], so[w][d], r);
    out[d] = from_f32<A>(bad ? nan : (sum > 0.f ? r / sum : r));
  }
  if (a.lse && threadIdx.x == 0) a.lse[(int64_t)s * a.n_heads + h] = bad ? nan : top + logf(sum);
}

template <class A, class C>
void launch_attn(const AttnArgs& a, cudaStream_t st) {
  paged_attn_kernel<A, C><<<dim3(a.n_heads, a.n_seq), kAttnWarps * 32, 0, st>>>(a);
}

}  // namespace
}  // namespace mllm

extern "C" size_t mllm_paged_attn_workspace(int n_seq, int n_heads, int head_dim) {
  if (n_seq < 1 || n_heads < 1 || head_dim < 8 || head_dim > 256) return 0;
  return 16;
}

extern "C" int mllm_paged_attn(const mllm_paged_kv* kv, int dtype, const void* d_q, int64_t q_stride, int n_seq,
                               int n_heads, const int32_t* d_len, const int32_t* d_table, int table_stride, float scale,
                               void* d_out, int64_t out_stride, float* d_lse, void* d_ws, size_t ws_bytes,
                               void* stream) {
  using namespace mllm;
  using namespace mllm::paged;
  if (int rc = check_kv(kv)) return rc;
  if (!is_float_kind(dtype) || (dtype != MLLM_DTYPE_F32 && dtype != kv->dtype))
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_paged_attn: queries must be f32 or of the cache's type");
  if (n_seq < 0 || n_seq > 65535 || n_heads < 1 || table_stride < 1)
    return refuse(MLLM_ERR_ARG, "mllm_paged_attn: sequences outside 0 to 65,535, or non-positive heads or table width");
  if (n_heads % kv->n_kv_heads || n_heads / kv->n_kv_heads > 64)
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_paged_attn: n_heads must be a multiple of the kv heads, at most 64 times");
  if (!d_q || !d_len || !d_table || !d_out) return refuse(MLLM_ERR_ARG, "mllm_paged_attn: null pointer");
  const int64_t row = (int64_t)n_heads * kv->head_dim;
  const int es = esize(dtype);
  if (q_stride < row || out_stride < row) return refuse(MLLM_ERR_ARG, "mllm_paged_attn: a row stride is shorter than a row");
  if (((uintptr_t)d_q & 15) || ((uintptr_t)d_out & 15) || q_stride * es % 16 || out_stride * es % 16)
    return refuse(MLLM_ERR_ARG, "mllm_paged_attn: rows must be 16-byte aligned");
  if (n_seq == 0) return MLLM_OK;
  if (!d_ws || ((uintptr_t)d_ws & 15) || ws_bytes < mllm_paged_attn_workspace(n_seq, n_heads, kv->head_dim))
    return refuse(MLLM_ERR_ARG, "mllm_paged_attn: workspace missing, misaligned or too small");
  const AttnArgs a = {kv->k, kv->v, kv->page_stride, kv->head_stride, kv->pos_stride, kv->n_pages, kv->page_len,
                      kv->n_kv_heads, kv->head_dim, d_q, q_stride, n_seq, n_heads, d_len, d_table, table_stride,
                      scale, d_out, out_stride, d_lse};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16)
    launch_attn<__half, __half>(a, st);
  else if (dtype == MLLM_DTYPE_BF16)
    launch_attn<__nv_bfloat16, __nv_bfloat16>(a, st);
  else if (kv->dtype == MLLM_DTYPE_F16)
    launch_attn<float, __half>(a, st);
  else if (kv->dtype == MLLM_DTYPE_BF16)
    launch_attn<float, __nv_bfloat16>(a, st);
  else
    launch_attn<float, float>(a, st);
  return launched("mllm_paged_attn: launch failed");
}
