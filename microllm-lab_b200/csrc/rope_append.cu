// Position step of a paged cache (mllm_rope_append): per-head RMS norm of q and k, rotation by the
// token's position, q out, k and v into the token's page row, in one pass.
//
//   y = x / sqrt(mean x^2 + eps) * gain;   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// for the pairs (a, b) = (i, i + rope_dim / 2) or (2 i, 2 i + 1), c and s the table row of the position.
// A few operations per element: bound by the bytes read and written, or by launch latency for few rows.
// One warp takes one head of one row: it normalises into shared memory, where each lane finds the
// partners of its elements whatever the layout and rope_dim.
#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;

constexpr int kRopeWarps = 4;

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
  void* q;
  int64_t q_stride;
};

template <class A, class C>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_append_kernel(const RopeArgs a) {
  __shared__ float y[kRopeWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kRopeWarps + warp;
  const int per_tok = a.n_heads + 2 * a.n_kv;
  const int64_t t = unit / per_tok;
  if (t >= a.n_tok) return;
  const int h = (int)(unit - t * per_tok);
  const int seq = a.seq ? a.seq[t] : (int)t;
  if (seq < 0) return;  // padding
  const int pos = a.pos[t];
  const int pg = pos / a.page_len;
  int page = -1;
  if (seq < a.n_seq && pos >= 0 && pg < a.table_stride && (pos < a.n_pos || a.rope_dim == 0))
    page = a.table[(int64_t)seq * a.table_stride + pg];
  const bool good = page >= 0 && page < a.n_pages;
  const A* x = static_cast<const A*>(a.qkv) + t * a.row_stride + (int64_t)h * a.dim;
  const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
  if (!good) {
    if (is_q) {
      A* out = static_cast<A*>(a.q) + t * a.q_stride + (int64_t)h * a.dim;
      for (int d = lane; d < a.dim; d += 32) out[d] = from_f32<A>(__int_as_float(0x7FC00000));
    }
    return;
  }
  const float* gain = is_q ? a.q_gain : (is_v ? nullptr : a.k_gain);
  float ss = 0.f;
  for (int d = lane; d < a.dim; d += 32) {
    const float f = to_f32(x[d]);
    y[warp][d] = f;
    ss = fmaf(f, f, ss);
  }
  if (gain) {
    const float r = sqrtf(warp_sum(ss) / (float)a.dim + a.eps);
    for (int d = lane; d < a.dim; d += 32) y[warp][d] = y[warp][d] / r * gain[d];
  }
  __syncwarp();
  C* kv = nullptr;
  if (!is_q) {
    const int hk = h - a.n_heads - (is_v ? a.n_kv : 0);
    kv = static_cast<C*>(is_v ? a.v : a.k) + page * a.page_stride + hk * a.head_stride +
         (int64_t)(pos - pg * a.page_len) * a.pos_stride;
  }
  A* out = static_cast<A*>(a.q) + t * a.q_stride + (int64_t)h * a.dim;
  const int half = a.rope_dim >> 1;
  for (int d = lane; d < a.dim; d += 32) {
    float f = y[warp][d];
    if (!is_v && d < a.rope_dim) {
      const int i = a.interleaved ? d >> 1 : (d < half ? d : d - half);
      const bool second = a.interleaved ? d & 1 : d >= half;
      const float p = y[warp][a.interleaved ? d ^ 1 : (second ? d - half : d + half)];
      const float c = a.cs[(int64_t)pos * half + i], s = a.sn[(int64_t)pos * half + i];
      f = second ? fmaf(f, c, p * s) : fmaf(f, c, -(p * s));
    }
    if (is_q)
      out[d] = from_f32<A>(f);
    else
      kv[d] = from_f32<C>(f);
  }
}

template <class A, class C>
void launch_rope(const RopeArgs& a, cudaStream_t st) {
  const int64_t units = (int64_t)a.n_tok * (a.n_heads + 2 * a.n_kv);
  rope_append_kernel<A, C><<<(unsigned)((units + kRopeWarps - 1) / kRopeWarps), kRopeWarps * 32, 0, st>>>(a);
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
  if ((int64_t)n_tok * (width / kv->head_dim) > (int64_t)1 << 31)
    return refuse(MLLM_ERR_ARG, "mllm_rope_append: more than 2^31 heads in one call");
  if (n_tok == 0) return MLLM_OK;
  const RopeArgs a = {kv->k, kv->v, kv->page_stride, kv->head_stride, kv->pos_stride, kv->n_pages, kv->page_len,
                      kv->n_kv_heads, kv->head_dim, d_qkv, row_stride, n_tok, n_heads, d_seq, d_pos, d_table,
                      n_seq, table_stride, d_q_gain, d_k_gain, eps, d_cos, d_sin, n_pos, rope_dim,
                      interleaved != 0, d_q, q_stride};
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
