// Attention of one new token per sequence over a paged K/V cache (mllm_paged_attn).
//
//   out = sum_p softmax_p(scale q . k_p) v_p,   lse = log sum_p exp(scale q . k_p)
//
// One pass with the running maximum m and sum l of the softmax: a block of scores with maximum m' turns
// (m, l, o) into (M, l e^(m - M) + sum e^(s - M), o e^(m - M) + sum e^(s - M) v), M = max(m, m').  Two
// multiply-adds per cached element and query head of its group: bound by the bytes of the cache.
//
// Work is cut into blocks of 32 positions of one (sequence, kv head, group of query heads), numbered in
// that order over the whole batch.  Every CTA takes an equal run of them, whatever the lengths: it sums
// the lengths itself, so that they may live on the device and the grid does not depend on them.  A run
// covers parts of a segment (a sequence's kv head) or several; the warps of a CTA take its blocks in turn
// and join their (m, l, o) in shared memory.  A segment that lies in one CTA is written at once; the
// others leave (m, l, o) in the workspace, and the CTA that counts itself last joins them in the order
// of their positions, so that the result does not depend on timing and no CTA waits for another.
#include <algorithm>
#include <atomic>

#include "device_common.cuh"
#include "paged.cuh"

namespace mllm {
namespace {

using namespace paged;

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kBlock = 32;       // positions per block: one per lane for the page lookups
constexpr int kMinBlocks = 4;    // a CTA's run is at least one block per warp
constexpr int kMaxCtas = 1024;   // partial slots in the workspace
constexpr int kMaxGroup = 16;    // query heads of a group
constexpr float kLog2e = 1.4426950408889634f;

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
  uint32_t* counter;  // [n_seq][n_kv][groups]
  float* part;        // [CTA][2][group][dim + 2]
  int rep, group_size, groups;  // query heads per kv head, of a group, groups of a kv head
};

// ---------------------------------------------------------------------------------------------
// Cached rows travel by asynchronous 16-byte copies into a ring in shared memory of which each lane reads
// back only what it asked for itself: many more bytes are under way than registers could take, and no
// barrier is needed, only the lane's own count of copies.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint4* to, const void* from, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 2^x for the softmax; x <= 0, or -inf.
__device__ __forceinline__ float pow2(float x) { return exp2f(x); }

// ---------------------------------------------------------------------------------------------
// A CTA's run of blocks.
// ---------------------------------------------------------------------------------------------
struct Run {
  int64_t q;          // blocks per CTA
  int64_t u, end;     // next block, end of the run
  int64_t before;     // blocks of the sequences before `seq`, per (kv head, group)
  int seq;
};

__device__ __forceinline__ int blocks_of(const AttnArgs& a, int s) {
  const int n = a.len[s];
  return n <= 0 || (int64_t)n > (int64_t)a.table_stride * a.page_len ? 0 : (n - 1) / kBlock + 1;
}

__device__ __forceinline__ Run find_run(const AttnArgs& a) {
  __shared__ int64_t wsum[kAttnWarps], s_before;
  __shared__ int s_seq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.n_seq + kAttnThreads - 1) / kAttnThreads;
  const int s0 = min(tid * per, a.n_seq), s1 = min(s0 + per, a.n_seq);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += blocks_of(a, s);
  int64_t run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) wsum[warp] = run;
  __syncthreads();
  int64_t total = 0, lead = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w == warp) lead = total;
    total += wsum[w];
  }
  const int64_t per_block = (int64_t)a.n_kv * a.groups;
  const int64_t all = total * per_block;
  Run r;
  r.q = max((int64_t)kMinBlocks, (all + gridDim.x - 1) / gridDim.x);
  r.u = blockIdx.x * r.q;
  r.end = min(r.u + r.q, all);
  r.seq = 0;
  r.before = 0;
  if (r.u >= all) return r;  // nothing (the same on every thread)
  int64_t b = lead + run - mine;  // blocks before this thread's sequences
  if (r.u >= b * per_block && r.u < (b + mine) * per_block) {
    int s = s0;
    for (;; ++s) {
      const int n = blocks_of(a, s);
      if (r.u < (b + n) * per_block) break;
      b += n;
    }
    s_seq = s;
    s_before = b;
  }
  __syncthreads();
  r.seq = s_seq;
  r.before = s_before;
  return r;
}

// The part of a run that lies in one segment.
struct Segment {
  int seq, kv, group, len;
  int b0, b1;          // blocks of the segment in this run
  int nb;              // blocks of the segment
  int64_t start;       // its first block in the batch's numbering
  int heads;           // query heads of the group
  int head0;           // the first of them
};

__device__ __forceinline__ bool next_segment(const AttnArgs& a, Run& r, Segment& g) {
  if (r.u >= r.end) return false;
  const int64_t per_block = (int64_t)a.n_kv * a.groups;
  int nb = blocks_of(a, r.seq);
  while (r.u >= (r.before + nb) * per_block) {
    r.before += nb;
    nb = blocks_of(a, ++r.seq);
  }
  const int64_t in = r.u - r.before * per_block;
  const int j = (int)(in / nb);
  g.seq = r.seq;
  g.nb = nb;
  g.len = a.len[r.seq];
  g.kv = j / a.groups;
  g.group = j - g.kv * a.groups;
  g.b0 = (int)(in - (int64_t)j * nb);
  g.b1 = (int)min((int64_t)nb, g.b0 + (r.end - r.u));
  g.start = r.u - g.b0;
  g.heads = min(a.rep - g.group * a.group_size, a.group_size);
  g.head0 = g.kv * a.rep + g.group * a.group_size;
  r.u += g.b1 - g.b0;
  return true;
}

// Element offset of this lane's position of a block, -1 when it is past the length or its page is bad.
__device__ __forceinline__ int64_t row_offset(const AttnArgs& a, const Segment& g, int block, int lane, int* bad) {
  const int p = block * kBlock + lane;
  if (block >= g.b1 || p >= g.len) return -1;
  const int pg = p / a.page_len;
  const int page = __ldg(a.table + (int64_t)g.seq * a.table_stride + pg);
  if ((unsigned)page >= (unsigned)a.n_pages) {
    *bad = 1;
    return -1;
  }
  return page * a.page_stride + g.kv * a.head_stride + (int64_t)(p - pg * a.page_len) * a.pos_stride;
}

// What the warps of a CTA leave for the join of a segment: m (in units of log 2) and l, and o, each warp's
// at the start of its ring.
struct Joint {
  float *m, *l;  // [warp][group]
  float* o;      // [warp] rings, each beginning with [group][DP]
  int ring;      // floats of a ring
};

template <class A>
__device__ __forceinline__ void write_out(const AttnArgs& a, const Segment& g, int h, int d, float o, float l) {
  static_cast<A*>(a.out)[g.seq * a.out_stride + (int64_t)(g.head0 + h) * a.dim + d] = from_f32<A>(l == 0.f ? 0.f : o / l);
}
__device__ __forceinline__ void write_lse(const AttnArgs& a, const Segment& g, int h, float m, float l) {
  if (a.lse) a.lse[(int64_t)g.seq * a.n_heads + g.head0 + h] = (m + log2f(l)) * (1.f / kLog2e);
}

// Joins the warps' (m, l, o); writes the segment's rows, or its part of them, and joins the parts when
// this CTA is the last to leave one.
template <class A, int DP>
__device__ void finish(const AttnArgs& a, const Run& r, const Segment& g, const Joint& w, int bad) {
  __shared__ int last;
  const int tid = threadIdx.x;
  const bool whole = g.b0 == 0 && g.b1 == g.nb;
  const size_t slot = (size_t)a.group_size * (a.dim + 2);
  float* part = a.part + ((size_t)blockIdx.x * 2 + (g.b0 == 0)) * slot;
  for (int i = tid; i < g.heads * a.dim; i += kAttnThreads) {
    const int h = i / a.dim, d = i - h * a.dim;
    float m = -INFINITY, l = 0.f, o = 0.f;
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) m = fmaxf(m, w.m[k * a.group_size + h]);
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) {
      const float mk = w.m[k * a.group_size + h];
      const float f = mk == -INFINITY ? 0.f : pow2(mk - m);
      l = fmaf(f, w.l[k * a.group_size + h], l);
      o = fmaf(f, w.o[k * w.ring + h * DP + d], o);
    }
    if (bad) l = __int_as_float(0x7FC00000);
    if (whole) {
      write_out<A>(a, g, h, d, o, l);
      if (d == 0) write_lse(a, g, h, m, l);
    } else {
      part[i] = o;
      if (d == 0) {
        part[a.group_size * a.dim + 2 * h] = m;
        part[a.group_size * a.dim + 2 * h + 1] = l;
      }
    }
  }
  if (whole) return;
  const int first = (int)(g.start / r.q), parts = (int)((g.start + g.nb - 1) / r.q) - first + 1;
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    uint32_t* c = a.counter + ((int64_t)g.seq * a.n_kv + g.kv) * a.groups + g.group;
    last = atomicAdd(c, 1u) == (uint32_t)parts - 1;
    if (last) *c = 0;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int i = tid; i < g.heads * a.dim; i += kAttnThreads) {
    const int h = i / a.dim;
    float m = -INFINITY, l = 0.f, o = 0.f;
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      const float* p = a.part + ((size_t)(first + k) * 2 + (k == 0)) * slot;
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + a.group_size * a.dim) + h);
      const float ok = __ldcg(p + i), mn = fmaxf(m, ml.x);
      const float f0 = m == -INFINITY ? 0.f : pow2(m - mn), f1 = ml.x == -INFINITY ? 0.f : pow2(ml.x - mn);
      l = l * f0 + ml.y * f1;
      o = o * f0 + ok * f1;
      m = mn;
    }
    write_out<A>(a, g, h, i - h * a.dim, o, l);
    if (i == h * a.dim) write_lse(a, g, h, m, l);
  }
}

// Sequences without positions, and those whose length the table cannot hold.
template <class A>
__device__ void finish_empty(const AttnArgs& a) {
  for (int s = blockIdx.x; s < a.n_seq; s += gridDim.x) {
    if (blocks_of(a, s)) continue;
    const float v = a.len[s] > 0 ? __int_as_float(0x7FC00000) : 0.f;
    A* out = static_cast<A*>(a.out) + s * a.out_stride;
    for (int i = threadIdx.x; i < a.n_heads * a.dim; i += kAttnThreads) out[i] = from_f32<A>(v);
    if (a.lse)
      for (int h = threadIdx.x; h < a.n_heads; h += kAttnThreads) a.lse[(int64_t)s * a.n_heads + h] = v == 0.f ? -INFINITY : v;
  }
}

// ---------------------------------------------------------------------------------------------
// Caches of 16 bits: both products on the tensor cores, m16n8k16 with positions (then head_dim) as the
// 16 rows and 8 query heads as the columns, so that a group of few heads wastes little.  The order of the
// summed index is free as long as both operands share it, so the 16-byte pieces of cached rows that a lane
// copies are its operands as they are: for the scores its 8 neighbouring elements of a key row serve two
// steps; for the output, pairs of value rows are woven by byte permutes.  The scores' accumulators, packed
// and transposed by movmatrix, are the second product's operand.
//
// The cached values are exact operands, and so are queries of their type.  f32 queries and weights are
// split into as many 16-bit terms as f32 needs (3 in bf16, 2 in f16, where queries are first scaled by a
// power of two to at most 1).  With queries of 16 bits the weights get two terms: one alone would add an
// error of the size of the output's own rounding (bf16 2.1e-3 of the result against 1.7e-3).
// ---------------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The terms of a pair: each is the rounding of what the ones before it left.
template <class T, int TERMS>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&w)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    w[i] = pack2<T>(a, b);
    if (i + 1 < TERMS) {
      const T* e = reinterpret_cast<const T*>(&w[i]);
      a -= to_f32(e[0]);
      b -= to_f32(e[1]);
    }
  }
}
template <class T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <class T, class A>
constexpr int terms_of() { return sizeof(A) == 2 ? 1 : (__is_same(T, __half) ? 2 : 3); }

template <class T, class A, int DP, int NT>
constexpr size_t mma_query_bytes() { return (size_t)(DP / 32) * terms_of<T, A>() * NT * 512; }

// Ring stages of 16 positions, and CTAs per SM: about 190 KB of copies under way on each SM.
template <int DP>
constexpr int mma_stages() { return DP == 64 ? 4 : 3; }
template <int DP>
constexpr int mma_ctas() { return DP == 64 ? 3 : DP == 128 ? 2 : 1; }
template <int DP>
constexpr int mma_ring_bytes() { return mma_stages<DP>() * 16 * 2 * DP * 2; }  // of a warp

template <class T, class A, int DP, int NT>
__global__ void __launch_bounds__(kAttnThreads, mma_ctas<DP>()) attn_mma_kernel(const AttnArgs a) {
  constexpr int C = DP / 32, V = DP / 64, S = mma_stages<DP>(), TERMS = terms_of<T, A>(), WT = TERMS == 1 ? 2 : TERMS;
  constexpr int PIECES = 2 * C + 4 * V;  // 16-byte pieces of a stage per lane
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float qscale[8 * NT];
  __shared__ int bad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = lane >> 2, quad = lane & 3;
  uint4* const ring = reinterpret_cast<uint4*>(smem + warp * mma_ring_bytes<DP>()) + lane;  // piece i of stage s: [(s PIECES + i) 32]
  uint4* const qs = reinterpret_cast<uint4*>(smem + kAttnWarps * mma_ring_bytes<DP>());      // [C][TERMS][NT][32]: operand words
  Joint joint;
  joint.o = reinterpret_cast<float*>(smem);
  joint.ring = mma_ring_bytes<DP>() / 4;
  joint.m = reinterpret_cast<float*>(qs + C * TERMS * NT * 32);
  joint.l = joint.m + kAttnWarps * a.group_size;
  const T* const kp = static_cast<const T*>(a.k);
  const T* const vp = static_cast<const T*>(a.v);

  Run run = find_run(a);
  Segment g;
  while (next_segment(a, run, g)) {
    __syncthreads();  // the last segment's queries and join are done with
    if (tid == 0) bad = 0;
    __syncthreads();
    // ---- this warp's stages: both halves of blocks b0 + warp, b0 + warp + 4, ...
    const int mine = g.b1 - g.b0 > warp ? (g.b1 - g.b0 - warp - 1) / kAttnWarps + 1 : 0;
    int n = 2 * mine;
    if (n && (g.b0 + warp + (mine - 1) * kAttnWarps) * kBlock + 16 >= g.len) --n;  // the last half is past the length
    int64_t off = row_offset(a, g, g.b0 + warp, lane, &bad);
    int64_t off_next = row_offset(a, g, g.b0 + warp + kAttnWarps, lane, &bad);
    auto issue = [&](int i) {
      if (i < n) {
        uint4* const to = ring + (i % S) * PIECES * 32;
        const int half = (i & 1) * 16;
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // key rows row, row + 8
          const int64_t at = __shfl_sync(0xffffffffu, off, half + row + 8 * e);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const int d = c * 32 + quad * 8;
            const bool ok = at >= 0 && d < a.dim;
            copy16(to + (2 * c + e) * 32, kp + (ok ? at + d : 0), ok);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // value rows 2 quad, 2 quad + 1, 2 quad + 8, 2 quad + 9
          const int64_t at = __shfl_sync(0xffffffffu, off, half + (e >> 1) * 8 + quad * 2 + (e & 1));
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const int d = v * 64 + row * 8;
            const bool ok = at >= 0 && d < a.dim;
            copy16(to + (2 * C + 4 * v + e) * 32, vp + (ok ? at + d : 0), ok);
          }
        }
        if (i & 1) {
          off = off_next;
          off_next = row_offset(a, g, g.b0 + warp + ((i >> 1) + 2) * kAttnWarps, lane, &bad);
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
    // ---- the group's queries as operand words, every head's rows of 8 * NT columns (0 past the group)
    const A* const q = static_cast<const A*>(a.q) + g.seq * a.q_stride + (int64_t)g.head0 * a.dim;
    if constexpr (TERMS == 2) {  // f32 queries as f16 terms: scaled to at most 1
      for (int h = warp; h < 8 * NT; h += kAttnWarps) {
        float m = 0.f;
        for (int d = lane; h < g.heads && d < a.dim; d += 32) m = fmaxf(m, fabsf(to_f32(q[h * a.dim + d])));
        m = warp_max(m);
        int e = 0;
        if (m > 0.f && m < INFINITY) (void)frexpf(m, &e);
        if (lane == 0) qscale[h] = ldexpf(1.f, max(min(e, 126), -126));
      }
      __syncthreads();
    }
    for (int i = tid; i < C * NT * 32; i += kAttnThreads) {
      const int l = i & 31, nt = (i >> 5) % NT, c = (i >> 5) / NT;
      const int h = nt * 8 + (l >> 2), d = c * 32 + (l & 3) * 8;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = h < g.heads && d < a.dim ? to_f32(q[h * a.dim + d + e]) : 0.f;
      if constexpr (TERMS == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] /= qscale[h];
      }
      uint32_t w[4][TERMS];
#pragma unroll
      for (int e = 0; e < 4; ++e) split2<T, TERMS>(x[2 * e], x[2 * e + 1], w[e]);
#pragma unroll
      for (int s = 0; s < TERMS; ++s) qs[((c * TERMS + s) * NT + nt) * 32 + l] = make_uint4(w[0][s], w[1][s], w[2][s], w[3][s]);
    }
    __syncthreads();
    float sc[NT][2];  // score factors of this lane's two columns, for base-2 exponents
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[nt][e] = a.scale * kLog2e;
        if constexpr (TERMS == 2) sc[nt][e] = a.scale * qscale[nt * 8 + quad * 2 + e] * kLog2e;
      }

    float m[NT][2], l[NT][2], o[V][4][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[v][i][nt][e] = 0.f;
    }
    for (int i = 0; i < n; ++i) {
      copies_wait<S - 2>();
      issue(i + S - 1);  // into the stage that the last round read
      const uint4* const st = ring + (i % S) * PIECES * 32;
      const int p0 = (g.b0 + warp + (i >> 1) * kAttnWarps) * kBlock + (i & 1) * 16 + row;
      // ---- scores: 16 positions x heads
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
      auto score = [&](float (&f)[4], const uint4& k0, const uint4& k1, const uint4& b) {
        mma<T>(f, k0.x, k1.x, k0.y, k1.y, b.x, b.y);
        mma<T>(f, k0.z, k1.z, k0.w, k1.w, b.z, b.w);
      };
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint4 k0 = st[(2 * c) * 32], k1 = st[(2 * c + 1) * 32];
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) score(s[nt], k0, k1, qs[((c * TERMS + t) * NT + nt) * 32 + lane]);
      }
      if constexpr (TERMS > 1) {
        // A key of +-inf times a later term of a query (of any sign, or 0) is NaN: there the first
        // term alone gives the score that f32 products would.
        bool odd = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= s[nt][e] != s[nt][e];
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C; ++c) score(f, st[(2 * c) * 32], st[(2 * c + 1) * 32], qs[(c * TERMS * NT + nt) * 32 + lane]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (s[nt][e] != s[nt][e]) s[nt][e] = f[e];
          }
        }
      }
      // ---- running maximum and sum of this lane's two heads, weights as the second operand
      uint32_t p[NT][WT][2];
      float keep[NT][2];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x0 = p0 < g.len ? s[nt][e] * sc[nt][e] : -INFINITY;
          float x1 = p0 + 8 < g.len ? s[nt][2 + e] * sc[nt][e] : -INFINITY;
          float top = fmaxf(m[nt][e], fmaxf(x0, x1));
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
          moved |= top != m[nt][e];
          const float base = top == -INFINITY ? 0.f : top;
          keep[nt][e] = pow2(m[nt][e] - base);  // 0 while there was nothing
          m[nt][e] = top;
          x0 = pow2(x0 - base);
          x1 = pow2(x1 - base);
          l[nt][e] = fmaf(l[nt][e], keep[nt][e], x0 + x1);
          s[nt][e] = x0;
          s[nt][2 + e] = x1;
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t w[WT];
          split2<T, WT>(s[nt][2 * k], s[nt][2 * k + 1], w);
#pragma unroll
          for (int t = 0; t < WT; ++t) p[nt][t][k] = transpose8x8(w[t]);
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[v][k][nt][e] *= keep[nt][e & 1];
      }
      // ---- output: head_dim x heads, the value rows woven in pairs of positions
#pragma unroll
      for (int v = 0; v < V; ++v) {
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = st[(2 * C + 4 * v + e) * 32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = __byte_perm(word(x[0], k), word(x[1], k), 0x5410), a1 = __byte_perm(word(x[0], k), word(x[1], k), 0x7632);
          const uint32_t a2 = __byte_perm(word(x[2], k), word(x[3], k), 0x5410), a3 = __byte_perm(word(x[2], k), word(x[3], k), 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int t = 0; t < WT; ++t) mma<T>(o[v][k][nt], a0, a1, a2, a3, p[nt][t][0], p[nt][t][1]);
        }
      }
    }
    copies_wait<0>();
    // ---- leave (m, l, o) for the join
    float* const jo = joint.o + warp * joint.ring;
    __syncwarp();  // every lane has read the ring
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], b);
        const int h = nt * 8 + quad * 2 + e;
        if (h < g.heads) {
          if (row == 0) {
            joint.m[warp * a.group_size + h] = m[nt][e];
            joint.l[warp * a.group_size + h] = l[nt][e];
          }
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<float2*>(jo + h * DP + v * 64 + row * 8 + 2 * k) = make_float2(o[v][k][nt][e], o[v][k][nt][2 + e]);
        }
      }
    __syncthreads();
    finish<A, DP>(a, run, g, joint, bad);
  }
  finish_empty<A>(a);
}

// ---------------------------------------------------------------------------------------------
// f32 caches: the products on the CUDA cores, at most 8 query heads for every cached element.  Four lanes
// share a key row for the scores; for the output a row's elements are spread over the lanes in pieces of
// four, the weights passing through shared memory.
// ---------------------------------------------------------------------------------------------
// Key rows of a stage that a lane shares (stages of 8 R positions), ring stages, CTAs per SM.
template <int DP>
constexpr int f32_rows() { return DP == 256 ? 1 : 2; }
template <int DP>
constexpr int f32_stages() { return DP == 64 ? 3 : 2; }
template <int DP>
constexpr int f32_ctas() { return DP == 64 ? 2 : 1; }
template <int DP>
constexpr int f32_ring_bytes() { return f32_stages<DP>() * 8 * f32_rows<DP>() * 2 * DP * 4; }  // of a warp
template <int DP, int G>
constexpr size_t f32_query_bytes() { return (size_t)G * DP * 4 + (size_t)kAttnWarps * 8 * f32_rows<DP>() * G * 4; }

template <int DP, int G>
__global__ void __launch_bounds__(kAttnThreads, f32_ctas<DP>()) attn_f32_kernel(const AttnArgs a) {
  constexpr int R = f32_rows<DP>(), P = 8 * R, S = f32_stages<DP>(), PARTS = kBlock / P;  // stages of a block
  constexpr int C = DP / 16, PER = DP / 4 < 32 ? DP / 4 : 32, ROWS = 32 / PER, V = DP / 4 / PER;
  constexpr int PIECES = R * C + P / ROWS * V;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int bad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = lane >> 2, quad = lane & 3;
  uint4* const ring = reinterpret_cast<uint4*>(smem + warp * f32_ring_bytes<DP>()) + lane;
  float* const qs = reinterpret_cast<float*>(smem + kAttnWarps * f32_ring_bytes<DP>());  // [G][DP]
  float* const pw = qs + G * DP + warp * P * G;                                            // [position][G]
  Joint joint;
  joint.o = reinterpret_cast<float*>(smem);
  joint.ring = f32_ring_bytes<DP>() / 4;
  joint.m = qs + G * DP + kAttnWarps * P * G;
  joint.l = joint.m + kAttnWarps * a.group_size;
  const float* const kp = static_cast<const float*>(a.k);
  const float* const vp = static_cast<const float*>(a.v);
  const float sc = a.scale * kLog2e;

  Run run = find_run(a);
  Segment g;
  while (next_segment(a, run, g)) {
    __syncthreads();
    if (tid == 0) bad = 0;
    __syncthreads();
    const int mine = g.b1 - g.b0 > warp ? (g.b1 - g.b0 - warp - 1) / kAttnWarps + 1 : 0;
    int n = PARTS * mine;
    while (n && (g.b0 + warp + (mine - 1) * kAttnWarps) * kBlock + ((n - 1) % PARTS) * P >= g.len) --n;
    int64_t off = row_offset(a, g, g.b0 + warp, lane, &bad);
    int64_t off_next = row_offset(a, g, g.b0 + warp + kAttnWarps, lane, &bad);
    auto issue = [&](int i) {
      if (i < n) {
        uint4* const to = ring + (i % S) * PIECES * 32;
        const int part = (i % PARTS) * P;
#pragma unroll
        for (int e = 0; e < R; ++e) {
          const int64_t at = __shfl_sync(0xffffffffu, off, part + row + 8 * e);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const int d = c * 16 + quad * 4;
            const bool ok = at >= 0 && d < a.dim;
            copy16(to + (c * R + e) * 32, kp + (ok ? at + d : 0), ok);
          }
        }
#pragma unroll
        for (int p = 0; p < P / ROWS; ++p) {
          const int64_t at = __shfl_sync(0xffffffffu, off, part + p * ROWS + lane / PER);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const int d = (v * PER + lane % PER) * 4;
            const bool ok = at >= 0 && d < a.dim;
            copy16(to + (R * C + p * V + v) * 32, vp + (ok ? at + d : 0), ok);
          }
        }
        if (i % PARTS == PARTS - 1) {
          off = off_next;
          off_next = row_offset(a, g, g.b0 + warp + (i / PARTS + 2) * kAttnWarps, lane, &bad);
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
    const float* const q = static_cast<const float*>(a.q) + g.seq * a.q_stride + (int64_t)g.head0 * a.dim;
    for (int i = tid; i < G * DP; i += kAttnThreads) {
      const int h = i / DP, d = i - h * DP;
      qs[i] = h < g.heads && d < a.dim ? q[h * a.dim + d] : 0.f;
    }
    __syncthreads();
    float m[G], l[G];  // of every head: m the same on every lane, l of this lane's positions
    float o[V][G][4];
#pragma unroll
    for (int h = 0; h < G; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[v][h][e] = 0.f;
    }
    for (int i = 0; i < n; ++i) {
      copies_wait<S - 2>();
      issue(i + S - 1);
      const float4* const st = reinterpret_cast<const float4*>(ring + (i % S) * PIECES * 32);
      const int p0 = (g.b0 + warp + (i / PARTS) * kAttnWarps) * kBlock + (i % PARTS) * P + row;
      // ---- scores of rows row, row + 8, ...
      float s[R][G];
#pragma unroll
      for (int e = 0; e < R; ++e)
#pragma unroll
        for (int h = 0; h < G; ++h) s[e][h] = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float4 k[R];
#pragma unroll
        for (int e = 0; e < R; ++e) k[e] = st[(c * R + e) * 32];
#pragma unroll
        for (int h = 0; h < G; ++h) {
          const float4 x = *reinterpret_cast<const float4*>(qs + h * DP + c * 16 + quad * 4);
#pragma unroll
          for (int e = 0; e < R; ++e)
            s[e][h] = fmaf(k[e].x, x.x, fmaf(k[e].y, x.y, fmaf(k[e].z, x.z, fmaf(k[e].w, x.w, s[e][h]))));
        }
      }
      bool moved = false;
      float keep[G];
      __syncwarp();  // the last round's weights are read
#pragma unroll
      for (int h = 0; h < G; ++h) {
        float top = m[h];
#pragma unroll
        for (int e = 0; e < R; ++e) {
          float x = s[e][h];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          s[e][h] = p0 + 8 * e < g.len ? x * sc : -INFINITY;
          top = fmaxf(top, s[e][h]);
        }
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
        moved |= top != m[h];
        const float base = top == -INFINITY ? 0.f : top;
        keep[h] = pow2(m[h] - base);
        m[h] = top;
        l[h] *= keep[h];
        if (quad < R) {  // lane e of a row's four holds the weight of row + 8 e
          const float w = pow2((R == 1 || quad == 0 ? s[0][h] : s[R - 1][h]) - base);
          l[h] += w;
          pw[(row + 8 * quad) * G + h] = w;
        }
      }
      __syncwarp();
      if (moved) {  // the maxima are the same on every lane
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int h = 0; h < G; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[v][h][e] *= keep[h];
      }
      // ---- output: ROWS value rows at a time
#pragma unroll
      for (int p = 0; p < P / ROWS; ++p) {
        float w[G];
#pragma unroll
        for (int h = 0; h < G; h += 4)
          *reinterpret_cast<float4*>(w + h) = *reinterpret_cast<const float4*>(pw + (p * ROWS + lane / PER) * G + h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float4 x = st[(R * C + p * V + v) * 32];
#pragma unroll
          for (int h = 0; h < G; ++h) {
            o[v][h][0] = fmaf(w[h], x.x, o[v][h][0]);
            o[v][h][1] = fmaf(w[h], x.y, o[v][h][1]);
            o[v][h][2] = fmaf(w[h], x.z, o[v][h][2]);
            o[v][h][3] = fmaf(w[h], x.w, o[v][h][3]);
          }
        }
      }
    }
    copies_wait<0>();
    float* const jo = joint.o + warp * joint.ring;
    __syncwarp();  // every lane has read the ring
#pragma unroll
    for (int h = 0; h < G; ++h) {
      l[h] = warp_sum(l[h]);
      if (h < g.heads) {
        if (lane == 0) {
          joint.m[warp * a.group_size + h] = m[h];
          joint.l[warp * a.group_size + h] = l[h];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int b = PER; b < 32; b <<= 1) o[v][h][e] += __shfl_xor_sync(0xffffffffu, o[v][h][e], b);
          }
          if (lane < PER)
            *reinterpret_cast<float4*>(jo + h * DP + (v * PER + lane) * 4) = make_float4(o[v][h][0], o[v][h][1], o[v][h][2], o[v][h][3]);
        }
      }
    }
    __syncthreads();
    finish<float, DP>(a, run, g, joint, bad);
  }
  finish_empty<float>(a);
}

// ---------------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------------
size_t counter_bytes(int n_seq, int n_heads) { return (((size_t)n_seq * n_heads * 4 + 255) / 256) * 256; }

// Opt in to more than 48 KB of shared memory, once per kernel and device.
template <auto KERNEL>
bool allow_smem(int dev, size_t smem) {
  static std::atomic<uint64_t> done{0};
  if (smem <= 48 * 1024 || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

template <auto KERNEL>
int launch(const AttnArgs& a, int per_sm, size_t smem, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return refuse(MLLM_ERR_CUDA, "mllm_paged_attn: no current CUDA device");
  smem += (size_t)2 * kAttnWarps * a.group_size * 4;  // m and l of the join
  if (!allow_smem<KERNEL>(dev, smem)) return refuse(MLLM_ERR_CUDA, "mllm_paged_attn: not enough shared memory");
  // no more CTAs than runs of the shortest length over the whole table
  const int64_t blocks = ((int64_t)a.table_stride * a.page_len + kBlock - 1) / kBlock;
  const int64_t most = (blocks + kMinBlocks - 1) / kMinBlocks * a.n_seq * a.n_kv * a.groups;
  const int grid = (int)std::min<int64_t>(most, std::min(kMaxCtas, sms * per_sm));
  KERNEL<<<grid, kAttnThreads, smem, st>>>(a);
  return launched("mllm_paged_attn: launch failed");
}

template <class T, class A, int DP, int NT>
int launch_mma(const AttnArgs& a, cudaStream_t st) {
  return launch<attn_mma_kernel<T, A, DP, NT>>(a, mma_ctas<DP>(), kAttnWarps * mma_ring_bytes<DP>() + mma_query_bytes<T, A, DP, NT>(), st);
}
template <class T, class A>
int run_mma(AttnArgs& a, cudaStream_t st) {
  a.group_size = std::min(a.rep, kMaxGroup);
  a.groups = (a.rep + a.group_size - 1) / a.group_size;
  const bool one = a.group_size <= 8;
  if (a.dim <= 64) return one ? launch_mma<T, A, 64, 1>(a, st) : launch_mma<T, A, 64, 2>(a, st);
  if (a.dim <= 128) return one ? launch_mma<T, A, 128, 1>(a, st) : launch_mma<T, A, 128, 2>(a, st);
  return one ? launch_mma<T, A, 256, 1>(a, st) : launch_mma<T, A, 256, 2>(a, st);
}
template <int DP, int G>
int launch_f32(const AttnArgs& a, cudaStream_t st) {
  return launch<attn_f32_kernel<DP, G>>(a, f32_ctas<DP>(), kAttnWarps * f32_ring_bytes<DP>() + f32_query_bytes<DP, G>(), st);
}
int run_f32(AttnArgs& a, cudaStream_t st) {
  a.group_size = std::min(a.rep, 8);
  a.groups = (a.rep + a.group_size - 1) / a.group_size;
  const bool four = a.group_size <= 4;
  if (a.dim <= 64) return four ? launch_f32<64, 4>(a, st) : launch_f32<64, 8>(a, st);
  if (a.dim <= 128) return four ? launch_f32<128, 4>(a, st) : launch_f32<128, 8>(a, st);
  return four ? launch_f32<256, 4>(a, st) : launch_f32<256, 8>(a, st);
}

}  // namespace
}  // namespace mllm

extern "C" size_t mllm_paged_attn_workspace(int n_seq, int n_heads, int head_dim) {
  using namespace mllm;
  if (n_seq < 1 || n_heads < 1 || head_dim < 8 || head_dim > 256) return 0;
  return counter_bytes(n_seq, n_heads) + (size_t)kMaxCtas * 2 * std::min(n_heads, kMaxGroup) * (head_dim + 2) * 4;
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
  AttnArgs a = {kv->k, kv->v, kv->page_stride, kv->head_stride, kv->pos_stride, kv->n_pages, kv->page_len,
                kv->n_kv_heads, kv->head_dim, d_q, q_stride, n_seq, n_heads, d_len, d_table, table_stride,
                scale, d_out, out_stride, d_lse};
  a.rep = n_heads / kv->n_kv_heads;
  a.counter = static_cast<uint32_t*>(d_ws);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d_ws) + counter_bytes(n_seq, n_heads));
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16) return run_mma<__half, __half>(a, st);
  if (dtype == MLLM_DTYPE_BF16) return run_mma<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (kv->dtype == MLLM_DTYPE_F16) return run_mma<__half, float>(a, st);
  if (kv->dtype == MLLM_DTYPE_BF16) return run_mma<__nv_bfloat16, float>(a, st);
  return run_f32(a, st);
}
