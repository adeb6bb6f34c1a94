// Page copies of a paged cache (mllm_copy_pages): page dst[i] of every layer, k and v, becomes a copy of
// page src[i].  Nothing is computed: bound by HBM (each byte read and written once), or by launch
// latency for a few pages.  The page ids travel as kernel parameters, so a call needs no device copy of
// them, takes no workspace and may be captured.  A CTA copies up to 32 KB of a page, every thread's loads
// issued before its stores: large pages spread over the SMs, and few of them fill the device.
//
// B200: 1,500 pages of 20 KB in 30 layers, k and v: 561 us (6.6 TB/s, the measured copy); 6 pages of 786 KB in 30
// layers: 92 us (one CTA per page: 139 us); one page of 24 KB in 30 layers: 6.6 us a call (6.2 to 7.0).
#include <algorithm>
#include <new>
#include <vector>

#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;

constexpr int kCopyThreads = 256;
constexpr int kCopyEach = 8;                               // 16-byte units of a thread
constexpr int kCopyUnits = kCopyThreads * kCopyEach;       // of a CTA: 32 KB

template <int N>
struct CopyArgs {
  uint4 *k, *v;
  int64_t page_stride, layer_stride;  // 16-byte units
  int page_units, chunks;  // of a page, and CTAs that share it
  int32_t src[N], dst[N];
};

// grid: (moves x chunks, layers, k or v)
template <int N>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs<N> a) {
  const int move = blockIdx.x / a.chunks, chunk = blockIdx.x - move * a.chunks;
  uint4* pool = (blockIdx.z ? a.v : a.k) + (int64_t)blockIdx.y * a.layer_stride;
  const uint4* from = pool + (int64_t)a.src[move] * a.page_stride;
  uint4* to = pool + (int64_t)a.dst[move] * a.page_stride;
  const int first = chunk * kCopyUnits + threadIdx.x;
  uint4 u[kCopyEach];
#pragma unroll
  for (int i = 0; i < kCopyEach; ++i)
    if (first + i * kCopyThreads < a.page_units) u[i] = __ldcs(from + first + i * kCopyThreads);
#pragma unroll
  for (int i = 0; i < kCopyEach; ++i)
    if (first + i * kCopyThreads < a.page_units) to[first + i * kCopyThreads] = u[i];
}

template <int N>
void launch_copy(const mllm_paged_kv* kv, int layers, int64_t layer_stride, const int32_t* src, const int32_t* dst,
                 int n, cudaStream_t st) {
  const int per = 16 / esize(kv->dtype);
  CopyArgs<N> a;
  a.k = static_cast<uint4*>(kv->k);
  a.v = static_cast<uint4*>(kv->v);
  a.page_stride = kv->page_stride / per;
  a.layer_stride = layer_stride / per;
  a.page_units = kv->n_kv_heads * kv->page_len * (kv->head_dim / per);
  a.chunks = (a.page_units + kCopyUnits - 1) / kCopyUnits;
  std::copy(src, src + n, a.src);
  std::copy(dst, dst + n, a.dst);
  copy_pages_kernel<N><<<dim3((unsigned)n * a.chunks, layers, 2), kCopyThreads, 0, st>>>(a);
}

// Whether no destination is a source or another destination, for up to kSorted copies: by sorting them, so that a
// few copies cost the same in a pool of any size.  More are marked in one byte per page of the pool.
constexpr int kSorted = 64;
bool destinations_apart(const int32_t* src, const int32_t* dst, int n) {
  int64_t use[2 * kSorted];  // page id, and 1 for a destination
  for (int i = 0; i < n; ++i) {
    use[i] = 2 * (int64_t)src[i];
    use[n + i] = 2 * (int64_t)dst[i] + 1;
  }
  std::sort(use, use + 2 * n);
  for (int i = 1; i < 2 * n; ++i)
    if ((use[i] & 1) && use[i] / 2 == use[i - 1] / 2) return false;
  return true;
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_copy_pages(const mllm_paged_kv* kv, int n_layers, int64_t layer_stride, const int32_t* src,
                               const int32_t* dst, int n, void* stream) {
  using namespace mllm;
  using namespace mllm::paged;
  if (int rc = check_kv(kv)) return rc;
  if (n < 0 || n_layers < 1 || n_layers > 65535) return refuse(MLLM_ERR_ARG, "mllm_copy_pages: bad page or layer count");
  constexpr int64_t kMostOfPage = (int64_t)1 << 30;
  if ((int64_t)kv->n_kv_heads * kv->page_len > kMostOfPage / kv->head_dim)
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_copy_pages: pages above 2^30 elements");
  const int64_t page = (int64_t)kv->n_kv_heads * kv->page_len * kv->head_dim;
  const bool by_head = kv->pos_stride == kv->head_dim && kv->head_stride == (int64_t)kv->page_len * kv->head_dim;
  const bool by_pos = kv->head_stride == kv->head_dim && kv->pos_stride == (int64_t)kv->n_kv_heads * kv->head_dim;
  if (!(by_head || by_pos) || kv->page_stride < page)
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_copy_pages: pages must be contiguous");
  const int per = 16 / esize(kv->dtype);
  if (n_layers > 1 && (layer_stride < page || layer_stride % per))
    return refuse(MLLM_ERR_ARG, "mllm_copy_pages: layer_stride below a page, or not 16-byte aligned");
  // layers one after another, or side by side within a page's stride
  if (n_layers > 1 && layer_stride < (__int128)(kv->n_pages - 1) * kv->page_stride + page &&
      kv->page_stride < (__int128)(n_layers - 1) * layer_stride + page)
    return refuse(MLLM_ERR_ARG, "mllm_copy_pages: layers overlap");
  if (n == 0) return MLLM_OK;
  if (!src || !dst) return refuse(MLLM_ERR_ARG, "mllm_copy_pages: null page list");
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= kv->n_pages || dst[i] < 0 || dst[i] >= kv->n_pages)
      return refuse(MLLM_ERR_ARG, "mllm_copy_pages: page id outside the pool");
  bool apart = true;
  if (n <= kSorted) {
    apart = destinations_apart(src, dst, n);
  } else {
    try {
      std::vector<uint8_t> used(kv->n_pages, 0);
      for (int i = 0; i < n; ++i) used[src[i]] = 1;
      for (int i = 0; i < n; ++i) {
        apart &= !used[dst[i]];
        used[dst[i]] = 1;
      }
    } catch (const std::bad_alloc&) {
      return refuse(MLLM_ERR_OOM, "mllm_copy_pages: no host memory for one byte per page of the pool");
    }
  }
  if (!apart) return refuse(MLLM_ERR_ARG, "mllm_copy_pages: a page is written twice, or read and written");
  constexpr int kFew = 32, kMany = 2048;  // 16 KB of parameters
  for (int i = 0; i < n; i += kMany) {
    const int m = std::min(kMany, n - i);
    if (m <= kFew)
      launch_copy<kFew>(kv, n_layers, layer_stride, src + i, dst + i, m, (cudaStream_t)stream);
    else
      launch_copy<kMany>(kv, n_layers, layer_stride, src + i, dst + i, m, (cudaStream_t)stream);
    if (int rc = launched("mllm_copy_pages: launch failed")) return rc;
  }
  return MLLM_OK;
}
