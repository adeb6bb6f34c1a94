// Attention of one new token per sequence over a paged K/V cache (mllm_paged_attn).
//
//   out = sum_p softmax_p(scale q . k_p) v_p,   lse = log sum_p exp(scale q . k_p)
//
// One pass with the running maximum m and sum l of the softmax: a block of scores with maximum m' turns
// (m, l, o) into (M, l e^(m - M) + sum e^(s - M), o e^(m - M) + sum e^(s - M) v), M = max(m, m').  Two
// multiply-adds per cached element and query head of its group: bound by the bytes of the cache.
//
// Work is cut into blocks of 32 positions of one segment (a sequence's kv head and group of query heads),
// numbered segment by segment over the whole batch.  Every CTA takes an equal run of blocks, whatever the
// lengths, and so does every warp within it: a warp walks its run on its own, through the ends of segments.
// The CTAs sum the lengths themselves, so that these may live on the device and the grid does not depend
// on them.  A segment that lies in one warp's run is written at once; the parts of the others are joined
// by the CTA in shared memory, and what spans CTAs through the workspace by the CTA that counts itself
// last, always in the order of positions: the result does not depend on timing, and no CTA waits for
// another.  Where every segment is short and can have a CTA of its own, it gets one, which saves the
// second join.
//
// B200: 3 sequences to 100,003 positions, 32 heads over 8 of 128, f16: 155 us (5.7 TB/s, 87 % of the measured
// copy); 256 sequences of 0 to 384, 9 heads over 3 of 64, bf16: 22.1 us, of which the copies need 7.2 (the rest
// is the latency of finding the runs, the first rows and the joins); 1 of 191, f32: 12.3 us.
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
constexpr int kWholeBlocks = 16; // segments up to this long get a CTA of their own where there are enough CTAs
constexpr int kFan = 16;         // a segment in more than twice as many parts is joined by so many of them first
constexpr int kMaxCtas = 1024;   // partial slots in the workspace
// Query heads of a group, at most (8 for f32 caches and for head_dim above 128, by registers).  Each group of a kv head
// walks the segment on its own, so that more heads than that read the cache several times (16 sequences to 32,768,
// 2 kv heads of 128, f32: 170 us for 8 heads each, 304 for 16; bf16: 91 us for 16, 146 for 32).
constexpr int kMaxGroup = 16;
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
  uint32_t* counter;  // [CTA]: of the segment that begins in it and ends in another
  uint32_t* counter2; // [CTA][2]
  float2* top;        // [CTA][2][kMaxGroup]: (m, l) of joined parts
  float* part;        // [CTA][2]: o [group][dim], (m, l) [group]
  int rep, group_size, groups;  // query heads per kv head, of a group, groups of a kv head
  int max_len;                  // positions that a row of the table can hold
  uint64_t page_mult;           // p / page_len = (p page_mult) >> page_shift for 0 <= p < 2^31
  int page_shift;
};

// ---------------------------------------------------------------------------------------------
// Cached rows travel by asynchronous 16-byte copies into a warp's own ring in shared memory: many more bytes
// are under way than registers could take, and no barrier is needed, only the lanes' counts of copies and the
// warp in step.  Eight lanes copy 128 neighbouring bytes of a row into one 128-byte line: where either side
// was split further, L2 sent lines twice (3 sequences to 100,003 f16: 206 us), and where the copies passed
// through L1 they waited for room in what shared memory leaves of it (188 us).  Within a line the
// 16-byte pieces are exchanged by an exclusive or of the row's number, so that no reads meet in a bank.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(ok ? 16 : 0) : "memory");
}
// The same for rows that are known to be there; further pieces of a row at constant distances.
template <int TO, int FROM>
__device__ __forceinline__ void copy16_at(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(to), "l"(from), "n"(TO), "n"(FROM) : "memory");
}
// N pieces of a row, FROM bytes apart, to places TO bytes apart from the AT-th byte on.
template <int AT, int TO, int FROM, int N, int I = 0>
__device__ __forceinline__ void copy_rows(uint32_t to, const void* from) {
  copy16_at<AT + I * TO, I * FROM>(to, from);
  if constexpr (I + 1 < N) copy_rows<AT, TO, FROM, N, I + 1>(to, from);
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 2^x for the softmax; x <= 0, or -inf.
__device__ __forceinline__ float pow2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---------------------------------------------------------------------------------------------
// Runs of blocks.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int blocks_of_len(const AttnArgs& a, int n) {
  return n <= 0 || n > a.max_len ? 0 : (n - 1) / kBlock + 1;
}
__device__ __forceinline__ int blocks_of(const AttnArgs& a, int s) { return blocks_of_len(a, __ldg(a.len + s)); }

// A place in the batch: block b of segment (seq, kv head, group).  Block numbers fit 31 bits (checked on the host
// for the longest lengths that the table can hold).
struct Place {
  int seq, kv, group, b, nb, len;
  __device__ __forceinline__ void at_seq(const AttnArgs& a, int s) {
    seq = s;
    len = __ldg(a.len + s);
    nb = blocks_of_len(a, len);
  }
  // To the next block; only called while more blocks follow.  True where another segment begins.
  __device__ __forceinline__ bool next(const AttnArgs& a) {
    if (++b < nb) return false;
    b = 0;
    if (++group == a.groups) {
      group = 0;
      if (++kv == a.n_kv) {
        kv = 0;
        do at_seq(a, seq + 1);
        while (!nb);
      }
    }
    return true;
  }
};

// What a CTA knows of the partition, and this warp's run.
struct Run {
  uint32_t q;     // blocks of a CTA's run
  uint32_t u0;    // the first of them
  int n;          // blocks of this warp's run (0: none)
  Place from;
};

// Every warp on its own: lanes sum the lengths of neighbouring sequences.
__device__ __forceinline__ Run find_run(const AttnArgs& a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = ((a.n_seq + 31) / 32 + 3) & ~3, s0 = min(lane * per, a.n_seq), s1 = min(s0 + per, a.n_seq);
  uint32_t mine = 0, longest = 0;
  auto add = [&](int len) {
    const uint32_t nb = blocks_of_len(a, len);
    mine += nb;
    longest = max(longest, nb);
  };
  int s4 = s0;
  if (((uintptr_t)a.len & 15) == 0) {  // four lengths at a time
#pragma unroll 2
    for (; s4 + 4 <= s1; s4 += 4) {
      const int4 v = __ldg(reinterpret_cast<const int4*>(a.len + s4));
      add(v.x), add(v.y), add(v.z), add(v.w);
    }
  }
#pragma unroll 4
  for (; s4 < s1; ++s4) add(__ldg(a.len + s4));
  longest = __reduce_max_sync(0xffffffffu, longest);
  const uint32_t per_seq = a.n_kv * a.groups;
  Run r;
  r.n = 0;
  if (longest <= kWholeBlocks && (uint64_t)a.n_seq * per_seq <= gridDim.x) {  // one segment, its blocks shared by the warps
    r.q = r.u0 = 0;
    const uint32_t seq = blockIdx.x / per_seq, j = blockIdx.x - seq * per_seq;
    if (seq >= a.n_seq) return r;
    r.from.at_seq(a, seq);
    r.from.kv = j / a.groups;
    r.from.group = j - r.from.kv * a.groups;
    const int share = (r.from.nb + kAttnWarps - 1) / kAttnWarps;
    r.from.b = warp * share;
    r.n = max(min(share, r.from.nb - r.from.b), 0);
    return r;
  }
  uint32_t upto = mine;  // this lane's sequences and those before them
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  const uint32_t all = __shfl_sync(0xffffffffu, upto, 31) * per_seq;
  r.q = max((all + gridDim.x - 1) / gridDim.x, (uint32_t)kMinBlocks);
  r.u0 = blockIdx.x * r.q;
  if ((uint64_t)blockIdx.x * r.q >= all) return r;
  const uint32_t end = min(r.u0 + r.q, all), each = (end - r.u0 + kAttnWarps - 1) / kAttnWarps, u = r.u0 + warp * each;
  if (u >= end) return r;
  r.n = min(each, end - u);
  // the lane whose sequences hold block u, then the one of them, 32 at a time
  const int who = __ffs(__ballot_sync(0xffffffffu, u < upto * per_seq)) - 1;
  uint32_t before = __shfl_sync(0xffffffffu, upto - mine, who) * per_seq;
  for (int s = who * per;; s += 32) {
    const int len = s + lane < a.n_seq ? __ldg(a.len + s + lane) : 0;
    const uint32_t nb = blocks_of_len(a, len);
    uint32_t sum = nb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, u < before + sum * per_seq);
    if (past) {
      const int at = __ffs(past) - 1;
      r.from.seq = s + at;
      r.from.nb = __shfl_sync(0xffffffffu, nb, at);
      r.from.len = __shfl_sync(0xffffffffu, len, at);
      before += __shfl_sync(0xffffffffu, sum - nb, at) * per_seq;
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31) * per_seq;
  }
  const uint32_t j = (u - before) / r.from.nb;
  r.from.b = u - before - j * r.from.nb;
  r.from.kv = j / a.groups;
  r.from.group = j - r.from.kv * a.groups;
  return r;
}

// Element offset of this lane's position of a block, -1 when it is past the length or its page is bad
// (noted in bit ord of `bad`).
__device__ __forceinline__ int64_t row_offset(const AttnArgs& a, const Place& c, int lane, uint32_t& bad, int ord) {
  const int p = c.b * kBlock + lane;
  if (p >= c.len) return -1;
  const int pg = (int)((uint64_t)p * a.page_mult >> a.page_shift);
  const int page = __ldg(a.table + (int64_t)c.seq * a.table_stride + pg);
  if ((unsigned)page >= (unsigned)a.n_pages) {
    bad |= 1u << (ord & 31);
    return -1;
  }
  return page * a.page_stride + c.kv * a.head_stride + (int64_t)(p - pg * a.page_len) * a.pos_stride;
}
// A part of a segment: what one run holds of it.
struct Part {
  int seq, kv, group, b0, blocks, nb;  // blocks 0: none
  __device__ __forceinline__ int first_head(const AttnArgs& a) const { return kv * a.rep + group * a.group_size; }
  __device__ __forceinline__ int heads(const AttnArgs& a) const { return min(a.rep - group * a.group_size, a.group_size); }
};

// The parts that a CTA's warps leave for the join: of a run's first segment (slot 0) and of its last (slot
// 1).  m is in units of log 2.  A page id outside the pool makes l, and with it the result, NaN.
struct Joint {
  Part* part;           // [warp][2]
  float *m, *l;         // [warp][2][group]
  float *first, *ring;  // o [group][DP]: slot 0 in `first`, slot 1 at the start of the warp's ring
  int ring_floats;
  template <int DP>
  __device__ __forceinline__ float* o(const AttnArgs& a, int warp, int slot) const {
    return slot ? ring + warp * ring_floats : first + warp * a.group_size * DP;
  }
};

__device__ __forceinline__ float4 rows4(const float4& v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }
__device__ __forceinline__ float4 fma4(float f, const float4& x, const float4& y) {
  return make_float4(fmaf(f, x.x, y.x), fmaf(f, x.y, y.y), fmaf(f, x.z, y.z), fmaf(f, x.w, y.w));
}
template <class A>
__device__ __forceinline__ void store4(A* p, const float4& v) {  // p on a 4-element boundary
  if constexpr (sizeof(A) == 4) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    A e[4] = {from_f32<A>(v.x), from_f32<A>(v.y), from_f32<A>(v.z), from_f32<A>(v.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
  }
}
// Four elements of a finished row of head h of the group; l == 0: no position had a weight.
template <class A>
__device__ __forceinline__ void write_out(const AttnArgs& a, const Part& p, int h, int d, const float4& o, float l) {
  A* out = static_cast<A*>(a.out) + p.seq * a.out_stride + (int64_t)(p.first_head(a) + h) * a.dim + d;
  store4(out, rows4(o, l == 0.f ? 0.f : 1.f / l));
}
__device__ __forceinline__ void write_lse(const AttnArgs& a, const Part& p, int h, float m, float l) {
  if (a.lse) a.lse[(int64_t)p.seq * a.n_heads + p.first_head(a) + h] = (m + log2f(l)) * (1.f / kLog2e);
}
// (m, l, o) joined with another.
__device__ __forceinline__ void join2(float& m, float& l, float4& o, float m1, float l1, const float4& o1) {
  const float top = fmaxf(m, m1);
  const float f0 = m == -INFINITY ? 0.f : pow2(m - top), f1 = m1 == -INFINITY ? 0.f : pow2(m1 - top);
  l = l * f0 + l1 * f1;
  o = fma4(f1, o1, rows4(o, f0));
  m = top;
}

// Joins the parts that the warps left, each segment by the warp that has its first part here.  A segment that
// spans CTAs is joined by the last of them to come; of one that spans more than 2 kFan, every kFan neighbours
// first, each time by the last to come, so that no CTA reads more than some dozens of parts (one sequence of
// 100,000 positions and 9 heads over one kv head, bf16: 29 us; joined by one CTA from at most 64 parts, 54 us).
template <class A, int DP>
__device__ __forceinline__ void join(const AttnArgs& a, const Run& r, const Joint& w) {
  struct Open {  // parts that this CTA joins: `parts` of them (0: none), `stride` CTAs apart from CTA `first` on
    Part p;
    int begin, first, parts, stride, groups;  // begin: the segment's first CTA; groups > 0: of so many such joins
  };
  __shared__ Open open[2];  // of a segment that began before this CTA, of one that began in it
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quads = a.dim / 4;
  const size_t slot = (size_t)a.group_size * (a.dim + 4);  // o, then m and l; 16-byte aligned for any group
  auto arrive = [](uint32_t* c, int n) {  // true for the last of n, which leaves the counter at 0
    const bool last = atomicAdd(c, 1u) == (uint32_t)n - 1;
    if (last) *c = 0;
    return last;
  };
  if (tid < 2) open[tid].parts = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = 2 * warp; i < 2 * warp + 2; ++i) {
    const Part p = w.part[i];
    if (!p.blocks || (i && p.b0)) continue;  // none, or it goes on from another warp's
    int have = p.blocks, end = i + 1;        // parts i .. end - 1 are of this segment
    for (; end < 2 * kAttnWarps; ++end) {
      const int more = w.part[end].blocks;
      if (!more) continue;
      if (w.part[end].b0 == 0) break;  // another segment
      have += more;
    }
    const bool done = have == p.nb;
    const int side = p.b0 == 0, items = p.heads(a) * quads;
    float* const out = a.part + ((size_t)blockIdx.x * 2 + side) * slot;
#pragma unroll 1
    for (int x = lane; x < items; x += 32) {
      const int h = x / quads, d = (x - h * quads) * 4;
      float m = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = i; k < end; ++k)
        if (w.part[k].blocks)
          join2(m, l, o, w.m[k * a.group_size + h], w.l[k * a.group_size + h],
                *reinterpret_cast<const float4*>(w.o<DP>(a, k >> 1, k & 1) + h * DP + d));
      if (done) {
        write_out<A>(a, p, h, d, o, l);
        if (d == 0) write_lse(a, p, h, m, l);
      } else {
        *reinterpret_cast<float4*>(out + h * a.dim + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(out + a.group_size * a.dim + 2 * h) = make_float2(m, l);
      }
    }
    if (done) continue;
    __threadfence();
    __syncwarp();
    if (lane == 0) {
      // which CTAs have a part, by the segment's first block: one that began in this run goes on to its end
      const uint32_t start = side ? r.u0 + r.q - have : r.u0 - p.b0, begin = start / r.q;
      const int parts = (int)((start + p.nb - 1) / r.q - begin) + 1;
      if (parts <= 2 * kFan) {
        if (arrive(a.counter + begin, parts)) open[side] = Open{p, (int)begin, (int)begin, parts, 1, 0};
      } else {
        const int k = (blockIdx.x - begin) / kFan * kFan, n = min(kFan, parts - k);
        if (arrive(a.counter2 + (begin + k) * 2 + (k == 0), n))
          open[side] = Open{p, (int)begin, (int)begin + k, n, 1, (parts + kFan - 1) / kFan};
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
#pragma unroll 1
    while (open[side].parts) {
      const Open s = open[side];
      __threadfence();
      const int items = s.p.heads(a) * quads;
      // (m, l) of a part: beside it, or of parts that were joined (their o is at the first one's place)
      auto ml = [&](int c, int h) {
        return s.stride == 1 ? reinterpret_cast<const float2*>(a.part + ((size_t)c * 2 + (c == s.begin)) * slot + a.group_size * a.dim) + h
                             : a.top + (c * 2 + (c == s.begin)) * kMaxGroup + h;
      };
#pragma unroll 1
      for (int x = tid; x < items; x += kAttnThreads) {
        const int h = x / quads, d = (x - h * quads) * 4;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < s.parts; ++k) {
          const int c = s.first + k * s.stride;
          const float2 mk = __ldcg(ml(c, h));
          join2(m, l, o, mk.x, mk.y,
                __ldcg(reinterpret_cast<const float4*>(a.part + ((size_t)c * 2 + (c == s.begin)) * slot + h * a.dim + d)));
        }
        if (s.groups == 0) {
          write_out<A>(a, s.p, h, d, o, l);
          if (d == 0) write_lse(a, s.p, h, m, l);
        } else {  // nobody else reads this element of o any more; (m, l) of the parts are still in use
          const int c = s.first * 2 + (s.first == s.begin);
          *reinterpret_cast<float4*>(a.part + c * slot + h * a.dim + d) = o;
          if (d == 0) a.top[c * kMaxGroup + h] = make_float2(m, l);
        }
      }
      if (s.groups) __threadfence();
      __syncthreads();
      if (tid == 0) {
        open[side].parts = 0;
        if (s.groups && arrive(a.counter + s.begin, s.groups)) open[side] = Open{s.p, s.begin, s.begin, s.groups, kFan, 0};
      }
      __syncthreads();
    }
  }
}

// Sequences without positions, and those whose length the table cannot hold.
template <class A>
__device__ __forceinline__ void finish_empty(const AttnArgs& a) {
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
// reads are its operands as they are: for the scores its 8 neighbouring elements of a key row serve two
// steps; for the output, pairs of value rows are woven by byte permutes.  The scores' accumulators, packed
// and transposed by movmatrix, are the second product's operand.
//
// The cached values are exact operands, and so are queries of their type.  f32 queries and weights are
// split into 3 terms in bf16 (24 bits) or 2 in f16 (23 bits; queries are first scaled by a power of two to below
// 2^15, so that an element is good to 2^-39 of the row's largest, or better).  With queries of 16 bits the
// weights get two terms: one alone would add an error of the size of the output's own rounding (bf16 2.1e-3 of
// the result against 1.7e-3).  f16 ends at 2^-24, so its weights are scaled to at most 2^15 before they are
// split, and the output's sums back at the end: a weight is good to 2^-40 of the largest of its run, not to
// 2^-25 (which loses all of 32 positions 18 nats below one other).
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
// An element too small for f16 keeps its sign in the first term, as the smallest number there is, and the second
// takes that off again: with an infinite key the first term alone decides (below).
template <int TERMS>
__device__ __forceinline__ void signed_zero(uint32_t (&w)[TERMS], float v, int at) {
  if (v == 0.f || (w[0] >> at & 0x7FFFu)) return;
  const uint32_t sign = v < 0.f ? 0x8000u : 0u;
  w[0] = (w[0] & ~(0xFFFFu << at)) | (sign | 1u) << at;
  w[1] = (w[1] & ~(0xFFFFu << at)) | ((sign ^ 0x8000u) | 1u) << at;
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

template <class T>
constexpr float weight_scale() { return __is_same(T, __half) ? 32768.f : 1.f; }
template <class T, class A>
constexpr int terms_of() { return sizeof(A) == 2 ? 1 : (__is_same(T, __half) ? 2 : 3); }

// Ring stages of 16 positions, and CTAs per SM: the copies under way (100 KB on an SM) need few stages, the chain
// of dependent steps from scores to output many warps.
template <int DP, int NT>
constexpr int mma_ctas() { return DP == 64 ? (NT == 1 ? 4 : 3) : DP == 128 ? (NT == 1 ? 3 : 2) : 1; }
constexpr int kMmaStages = 2;
template <int DP>
constexpr int mma_ring_bytes() { return kMmaStages * 16 * 2 * DP * 2; }  // of a warp
// Operand words of the queries of a warp's segment: in registers where they are few.
template <class T, class A, int DP, int NT>
constexpr int mma_query_words() { return (DP / 32) * terms_of<T, A>() * NT; }  // uint4 of a lane
template <class T, class A, int DP, int NT>
constexpr bool mma_query_regs() { return mma_query_words<T, A, DP, NT>() <= 6; }
template <class T, class A, int DP, int NT>
constexpr int mma_query_bytes() { return mma_query_regs<T, A, DP, NT>() ? 0 : mma_query_words<T, A, DP, NT>() * 512; }  // of a warp

template <class T, class A, int DP, int NT>
__global__ void __launch_bounds__(kAttnThreads, mma_ctas<DP, NT>()) attn_mma_kernel(const AttnArgs a) {
  constexpr int C = DP / 32, V = DP / 64, S = kMmaStages, TERMS = terms_of<T, A>(), WT = TERMS == 1 ? 2 : TERMS;
  constexpr int PIECES = 2 * C + 4 * V;  // 16-byte pieces of a stage per lane
  constexpr bool QREG = mma_query_regs<T, A, DP, NT>();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Part parts[2 * kAttnWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, quad = lane & 3;
  const uint4* const ring = reinterpret_cast<const uint4*>(smem + warp * mma_ring_bytes<DP>());  // piece i of stage s: [(s PIECES + i) 32]
  uint4* const qs = reinterpret_cast<uint4*>(smem + kAttnWarps * mma_ring_bytes<DP>() + warp * mma_query_bytes<T, A, DP, NT>()) + lane;
  Joint joint;
  joint.part = parts;
  joint.ring = reinterpret_cast<float*>(smem);
  joint.ring_floats = mma_ring_bytes<DP>() / 4;
  joint.first = reinterpret_cast<float*>(smem + kAttnWarps * (mma_ring_bytes<DP>() + mma_query_bytes<T, A, DP, NT>()));
  joint.m = joint.first + kAttnWarps * a.group_size * DP;
  joint.l = joint.m + 2 * kAttnWarps * a.group_size;
  const T* const kp = static_cast<const T*>(a.k);
  const T* const vp = static_cast<const T*>(a.v);

  const Run run = find_run(a);
  if (lane == 0) parts[2 * warp].blocks = parts[2 * warp + 1].blocks = 0;
  const int n = run.n;  // blocks; two stages each
  if (n) {
    Place ahead = run.from, c = run.from;
    uint32_t bad = 0;  // by segment, numbered along the run: this lane has met a page outside the pool
    int ahead_ord = 0, ord = 0;
    int64_t off = row_offset(a, ahead, lane, bad, ahead_ord), off_next = -1;
    auto look = [&](int k) {  // the rows of block k of the run
      if (k < n) {
        ahead_ord += ahead.next(a);
        off_next = row_offset(a, ahead, lane, bad, ahead_ord);
      }
    };
    look(1);
    // A stage: keys, then values, each [64-element chunk][16 rows][8 pieces]; piece c of row p at c ^ 4 (p & 1) (keys),
    // at c ^ (p & 6) (values).  This lane copies piece `chunk` of rows 4 x + part.
    const int part = lane >> 3, chunk = lane & 7;
    const uint32_t ring32 = smem_u32(smem + warp * mma_ring_bytes<DP>());
    const uint32_t k_to = part * 128 + (chunk ^ (part & 1) * 4) * 16;
    const uint32_t v_even = V * 2048 + part * 128 + (chunk ^ (part & 2)) * 16, v_odd = V * 2048 + part * 128 + (chunk ^ (part & 2) ^ 4) * 16;
    auto issue = [&](int i) {
      if (i < 2 * n) {
        const uint32_t to = ring32 + (i % S) * PIECES * 512;
        const bool whole = a.dim == DP && __all_sync(0xffffffffu, off >= 0);  // every row of the block
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int64_t at = __shfl_sync(0xffffffffu, off, (i & 1) * 16 + 4 * x + part);
          const T* const kr = kp + at + chunk * 8;
          const T* const vr = vp + at + chunk * 8;
          const uint32_t kt = to + k_to + x * 512, vt = to + (x & 1 ? v_odd : v_even) + x * 512;
          if (whole) {
            copy_rows<0, 2048, 128, V>(kt, kr);
            copy_rows<0, 2048, 128, V>(vt, vr);
          } else {
#pragma unroll
            for (int y = 0; y < V; ++y) {
              const bool ok = at >= 0 && y * 64 + chunk * 8 < a.dim;
              copy16(kt + y * 2048, ok ? kr + y * 64 : kp, ok);
              copy16(vt + y * 2048, ok ? vr + y * 64 : vp, ok);
            }
          }
        }
        if (i & 1) {
          off = off_next;
          look((i >> 1) + 2);
        }
      }
      copies_commit();
    };
#pragma unroll 1
    for (int i = 0; i < S - 1; ++i) issue(i);

    uint4 qr[QREG ? C : 1][QREG ? TERMS : 1][QREG ? NT : 1] = {};
    auto query = [&](int x, int t, int nt) -> uint4 {
      if constexpr (QREG)
        return qr[x][t][nt];
      else
        return qs[((x * TERMS + t) * NT + nt) * 32];
    };
    float sc[NT][2];  // score factors of this lane's two heads, for base-2 exponents
    float m[NT][2], l[NT][2], o[V][4][NT][4];
    int b0 = 0;
    for (int k = 0; k < n; ++k) {
      if (k == 0 || c.b == 0) {  // a segment begins: its queries, every head's row of 8 * NT (0 past the group)
        b0 = c.b;
        const Part p = {c.seq, c.kv, c.group};
        const int heads = p.heads(a);
        const A* const q = static_cast<const A*>(a.q) + c.seq * a.q_stride + (int64_t)p.first_head(a) * a.dim;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int h = nt * 8 + row;
          if constexpr (TERMS == 1) {
#pragma unroll
            for (int x = 0; x < C; ++x) {
              const int d = x * 32 + quad * 8;
              uint4 w = make_uint4(0u, 0u, 0u, 0u);
              if (h < heads && d < a.dim) w = __ldg(reinterpret_cast<const uint4*>(q + h * a.dim + d));
              if constexpr (QREG)
                qr[x][0][nt] = w;
              else
                qs[(x * NT + nt) * 32] = w;
            }
            sc[nt][0] = sc[nt][1] = a.scale * kLog2e;
          } else {
            float f[C][8], top = 0.f, low = INFINITY;
#pragma unroll
            for (int x = 0; x < C; ++x) {
              const int d = x * 32 + quad * 8;
              float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
              if (h < heads && d < a.dim) {
                u = __ldg(reinterpret_cast<const float4*>(q + h * a.dim + d));
                v = __ldg(reinterpret_cast<const float4*>(q + h * a.dim + d) + 1);
              }
              f[x][0] = u.x, f[x][1] = u.y, f[x][2] = u.z, f[x][3] = u.w;
              f[x][4] = v.x, f[x][5] = v.y, f[x][6] = v.z, f[x][7] = v.w;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                top = fmaxf(top, fabsf(f[x][e]));
                if constexpr (TERMS == 2) low = fminf(low, fabsf(f[x][e]));
              }
            }
            float up = 1.f, down = 1.f;
            if constexpr (TERMS == 2) {  // f16 terms: scaled to below 2^15
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
              int e = 15;
              if (top > 0.f && top < INFINITY) (void)frexpf(top, &e);
              e = max(e - 15, -126);  // at most 113
              up = ldexpf(1.f, e);
              down = ldexpf(1.f, -e);
            }
            const bool tiny = h < heads && low * down < 0x1p-24f;  // some element is 0 in f16, as few are
            sc[nt][0] = a.scale * __shfl_sync(0xffffffffu, up, quad * 8) * kLog2e;
            sc[nt][1] = a.scale * __shfl_sync(0xffffffffu, up, quad * 8 + 4) * kLog2e;
#pragma unroll
            for (int x = 0; x < C; ++x) {
              uint32_t w[4][TERMS];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                split2<T, TERMS>(f[x][2 * e] * down, f[x][2 * e + 1] * down, w[e]);
                if (TERMS == 2 && tiny) {
                  signed_zero(w[e], f[x][2 * e], 0);
                  signed_zero(w[e], f[x][2 * e + 1], 16);
                }
              }
#pragma unroll
              for (int t = 0; t < TERMS; ++t) {
                const uint4 v = make_uint4(w[0][t], w[1][t], w[2][t], w[3][t]);
                if constexpr (QREG)
                  qr[x][t][nt] = v;
                else
                  qs[((x * TERMS + t) * NT + nt) * 32] = v;
              }
            }
          }
          m[nt][0] = m[nt][1] = -INFINITY;
          l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[v][x][nt][e] = 0.f;
        }
      }
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int i = 2 * k + half;
        copies_wait<S - 2>();
        __syncwarp();      // all lanes' copies are there, and all have read the last round's stage
        issue(i + S - 1);  // into that one
        if (c.b * kBlock + half * 16 >= c.len) continue;
        const uint4* const sk = ring + (i % S) * PIECES * 32 + row * 8 + (quad ^ (row & 1) * 4);           // this lane's key pieces
        const uint4* const sk2 = ring + (i % S) * PIECES * 32 + row * 8 + ((quad + 4) ^ (row & 1) * 4);    // of odd 32-element steps
        const uint4* const sv = ring + ((i % S) * PIECES + 2 * C) * 32 + quad * 16 + (row ^ quad * 2);     // and value pieces
        const int p0 = c.b * kBlock + half * 16 + row;
        // ---- scores: 16 positions x heads
        float s[NT][4], s2[NT][4];  // two sums, so that the products' latencies overlap
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
        auto score = [&](float (&f)[4], float (&f2)[4], const uint4& k0, const uint4& k1, const uint4& b) {
          mma<T>(f, k0.x, k1.x, k0.y, k1.y, b.x, b.y);
          mma<T>(f2, k0.z, k1.z, k0.w, k1.w, b.z, b.w);
        };
#pragma unroll
        for (int x = 0; x < C; ++x) {
          const uint4 k0 = (x & 1 ? sk2 : sk)[(x >> 1) * 128], k1 = (x & 1 ? sk2 : sk)[(x >> 1) * 128 + 64];
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) score(s[nt], s2[nt], k0, k1, query(x, t, nt));
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
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
              for (int x = 0; x < C; ++x) score(f, f, (x & 1 ? sk2 : sk)[(x >> 1) * 128], (x & 1 ? sk2 : sk)[(x >> 1) * 128 + 64], query(x, 0, nt));
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
            float x0 = p0 < c.len ? s[nt][e] * sc[nt][e] : -INFINITY;
            float x1 = p0 + 8 < c.len ? s[nt][2 + e] * sc[nt][e] : -INFINITY;
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
          for (int x = 0; x < 2; ++x) {
            uint32_t w[WT];
            split2<T, WT>(s[nt][2 * x] * weight_scale<T>(), s[nt][2 * x + 1] * weight_scale<T>(), w);
#pragma unroll
            for (int t = 0; t < WT; ++t) p[nt][t][x] = transpose8x8(w[t]);
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[v][x][nt][e] *= keep[nt][e & 1];
        }
        // ---- output: head_dim x heads, the value rows woven in pairs of positions
#pragma unroll
        for (int v = 0; v < V; ++v) {
          uint4 x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = sv[v * 128 + (e >> 1) * 64 + (e & 1) * 8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t a0 = __byte_perm(word(x[0], y), word(x[1], y), 0x5410), a1 = __byte_perm(word(x[0], y), word(x[1], y), 0x7632);
            const uint32_t a2 = __byte_perm(word(x[2], y), word(x[3], y), 0x5410), a3 = __byte_perm(word(x[2], y), word(x[3], y), 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int t = 0; t < WT; ++t) mma<T>(o[v][y][nt], a0, a1, a2, a3, p[nt][t][0], p[nt][t][1]);
          }
        }
      }
      const bool ends = c.b + 1 == c.nb;
      if (ends || k + 1 == n) {  // all that this run has of the segment
        const bool done = ends && b0 == 0;
        const int slot = k + 1 - (c.b + 1 - b0) == 0 ? 0 : 1;
        const Part mine = {c.seq, c.kv, c.group, b0, c.b + 1 - b0, c.nb};
        const int heads = mine.heads(a);
        const bool nan = __any_sync(0xffffffffu, bad >> (ord & 31) & 1u);
        bad &= ~(1u << (ord & 31));
        if (slot == 1 && !done) {  // the run's end: the ring is free
          copies_wait<0>();
          __syncwarp();
        }
        float* const jo = joint.o<DP>(a, warp, slot);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float sum = l[nt][e];
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, b);
            if (nan) sum = __int_as_float(0x7FC00000);
            const int h = nt * 8 + quad * 2 + e;
            if (h >= heads) continue;
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const int d = v * 64 + row * 8;
              if (d >= a.dim) continue;
              constexpr float back = 1.f / weight_scale<T>();
              const float4 lo = rows4(make_float4(o[v][0][nt][e], o[v][0][nt][2 + e], o[v][1][nt][e], o[v][1][nt][2 + e]), back);
              const float4 hi = rows4(make_float4(o[v][2][nt][e], o[v][2][nt][2 + e], o[v][3][nt][e], o[v][3][nt][2 + e]), back);
              if (done) {
                write_out<A>(a, mine, h, d, lo, sum);
                write_out<A>(a, mine, h, d + 4, hi, sum);
              } else {
                *reinterpret_cast<float4*>(jo + h * DP + d) = lo;
                *reinterpret_cast<float4*>(jo + h * DP + d + 4) = hi;
              }
            }
            if (row == 0) {
              if (done) {
                write_lse(a, mine, h, m[nt][e], sum);
              } else {
                joint.m[(2 * warp + slot) * a.group_size + h] = m[nt][e];
                joint.l[(2 * warp + slot) * a.group_size + h] = sum;
              }
            }
          }
        if (!done && lane == 0) parts[2 * warp + slot] = mine;
        ++ord;
      }
      if (k + 1 < n) c.next(a);
    }
    copies_wait<0>();
  }
  join<A, DP>(a, run, joint);
  finish_empty<A>(a);
}

// ---------------------------------------------------------------------------------------------
// f32 caches: the products on the CUDA cores, at most 8 query heads for every cached element.  Four lanes
// share a key row for the scores; for the output a row's elements are spread over the lanes in pieces of
// four, the weights passing through shared memory.
// ---------------------------------------------------------------------------------------------
// Key rows of a stage that a lane shares (stages of 8 R positions), ring stages, CTAs per SM.
template <int DP>
constexpr int f32_rows() { return DP == 64 ? 2 : 1; }
constexpr int kF32Stages = 2;
template <int DP, int G>
constexpr int f32_ctas() { return DP == 256 ? 1 : G == 4 ? 3 : 2; }
template <int DP>
constexpr int f32_ring_bytes() { return kF32Stages * 8 * f32_rows<DP>() * 2 * DP * 4; }  // of a warp
template <int DP, int G>
constexpr int f32_query_bytes() { return G * DP * 4 + 8 * f32_rows<DP>() * G * 4; }  // of a warp: queries and weights

template <int DP, int G>
__global__ void __launch_bounds__(kAttnThreads, f32_ctas<DP, G>()) attn_f32_kernel(const AttnArgs a) {
  constexpr int R = f32_rows<DP>(), P = 8 * R, S = kF32Stages, PARTS = kBlock / P;  // stages of a block
  constexpr int C = DP / 16, PER = DP / 4 < 32 ? DP / 4 : 32, ROWS = 32 / PER, V = DP / 4 / PER;
  constexpr int PIECES = R * C + P / ROWS * V;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Part parts[2 * kAttnWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, quad = lane & 3;
  const float4* const ring = reinterpret_cast<const float4*>(smem + warp * f32_ring_bytes<DP>());
  float* const qs = reinterpret_cast<float*>(smem + kAttnWarps * f32_ring_bytes<DP>() + warp * f32_query_bytes<DP, G>());  // [G][DP]
  float* const pw = qs + G * DP;                                                                                            // [position][G]
  Joint joint;
  joint.part = parts;
  joint.ring = reinterpret_cast<float*>(smem);
  joint.ring_floats = f32_ring_bytes<DP>() / 4;
  joint.first = reinterpret_cast<float*>(smem + kAttnWarps * (f32_ring_bytes<DP>() + f32_query_bytes<DP, G>()));
  joint.m = joint.first + kAttnWarps * a.group_size * DP;
  joint.l = joint.m + 2 * kAttnWarps * a.group_size;
  const float* const kp = static_cast<const float*>(a.k);
  const float* const vp = static_cast<const float*>(a.v);
  const float sc = a.scale * kLog2e;

  const Run run = find_run(a);
  if (lane == 0) parts[2 * warp].blocks = parts[2 * warp + 1].blocks = 0;
  const int n = run.n;  // blocks
  if (n) {
    Place ahead = run.from, c = run.from;
    uint32_t bad = 0;
    int ahead_ord = 0, ord = 0;
    int64_t off = row_offset(a, ahead, lane, bad, ahead_ord), off_next = -1;
    auto look = [&](int k) {
      if (k < n) {
        ahead_ord += ahead.next(a);
        off_next = row_offset(a, ahead, lane, bad, ahead_ord);
      }
    };
    look(1);
    const int part = lane >> 3, chunk = lane & 7;  // of the key copies: rows 4 i + part, 32-element chunks of 8 pieces
    const uint32_t ring32 = smem_u32(smem + warp * f32_ring_bytes<DP>());
    const uint32_t k_to = part * 128 + (chunk ^ (part & 1) * 4) * 16;  // as above
    auto issue = [&](int i) {
      if (i < PARTS * n) {
        const uint32_t to = ring32 + (i % S) * PIECES * 512;
        const int first = (i % PARTS) * P;
        const bool whole = a.dim == DP && __all_sync(0xffffffffu, off >= 0);  // every row of the block
#pragma unroll
        for (int x = 0; x < 2 * R; ++x) {
          const int64_t at = __shfl_sync(0xffffffffu, off, first + 4 * x + part);
          const float* const kr = kp + at + chunk * 4;
          const uint32_t kt = to + k_to + x * 512;
          if (whole) {
            copy_rows<0, P * 128, 128, C / 2>(kt, kr);
          } else {
#pragma unroll 1
            for (int y = 0; y < C / 2; ++y) {
              const bool ok = at >= 0 && y * 32 + chunk * 4 < a.dim;
              copy16(kt + y * P * 128, ok ? kr + y * 32 : kp, ok);
            }
          }
        }
#pragma unroll
        for (int p = 0; p < P / ROWS; ++p) {
          const int64_t at = __shfl_sync(0xffffffffu, off, first + p * ROWS + lane / PER);
          const float* const from = vp + at + lane % PER * 4;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const bool ok = whole || (at >= 0 && (v * PER + lane % PER) * 4 < a.dim);
            copy16(to + (R * C + p * V + v) * 512 + lane * 16, ok ? from + v * PER * 4 : vp, ok);
          }
        }
        if (i % PARTS == PARTS - 1) {
          off = off_next;
          look(i / PARTS + 2);
        }
      }
      copies_commit();
    };
#pragma unroll 1
    for (int i = 0; i < S - 1; ++i) issue(i);
    float m[G], l[G];  // of every head: m the same on every lane, l of this lane's positions
    float o[V][G][4];
    int b0 = 0;
    for (int k = 0; k < n; ++k) {
      if (k == 0 || c.b == 0) {
        b0 = c.b;
        const Part p = {c.seq, c.kv, c.group};
        const int heads = p.heads(a);
        const float* const q = static_cast<const float*>(a.q) + c.seq * a.q_stride + (int64_t)p.first_head(a) * a.dim;
        __syncwarp();  // the last segment's queries are read
#pragma unroll
        for (int x = 0; x < G * DP / 128; ++x) {
          const int e = (x * 32 + lane) * 4, h = e / DP, d = e % DP;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (h < heads && d < a.dim) v = __ldg(reinterpret_cast<const float4*>(q + h * a.dim + d));
          *reinterpret_cast<float4*>(qs + e) = v;
        }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < G; ++h) {
          m[h] = -INFINITY;
          l[h] = 0.f;
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[v][h][e] = 0.f;
        }
      }
#pragma unroll 1
      for (int turn = 0; turn < PARTS; ++turn) {
        const int i = PARTS * k + turn;
        copies_wait<S - 2>();
        __syncwarp();  // all lanes' copies are there, and all have read the last round's stage
        issue(i + S - 1);
        if (c.b * kBlock + turn * P >= c.len) continue;
        const float4* const st = ring + (i % S) * PIECES * 32;
        const int p0 = c.b * kBlock + turn * P + row;
        // ---- scores of rows row, row + 8, ...
        float s[R][G];
#pragma unroll
        for (int e = 0; e < R; ++e)
#pragma unroll
          for (int h = 0; h < G; ++h) s[e][h] = 0.f;
#pragma unroll
        for (int x = 0; x < C; ++x) {
          float4 key[R];
#pragma unroll
          for (int e = 0; e < R; ++e) key[e] = st[((x >> 1) * P + row + 8 * e) * 8 + (((x & 1) * 4 + quad) ^ (row & 1) * 4)];
#pragma unroll
          for (int h = 0; h < G; ++h) {
            const float4 q = *reinterpret_cast<const float4*>(qs + h * DP + x * 16 + quad * 4);
#pragma unroll
            for (int e = 0; e < R; ++e)
              s[e][h] = fmaf(key[e].x, q.x, fmaf(key[e].y, q.y, fmaf(key[e].z, q.z, fmaf(key[e].w, q.w, s[e][h]))));
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
            s[e][h] = p0 + 8 * e < c.len ? x * sc : -INFINITY;
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
            const float4 x = st[(R * C + p * V + v) * 32 + lane];
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
      const bool ends = c.b + 1 == c.nb;
      if (ends || k + 1 == n) {  // all that this run has of the segment
        const bool done = ends && b0 == 0;
        const int slot = k + 1 - (c.b + 1 - b0) == 0 ? 0 : 1;
        const Part mine = {c.seq, c.kv, c.group, b0, c.b + 1 - b0, c.nb};
        const int heads = mine.heads(a);
        const bool nan = __any_sync(0xffffffffu, bad >> (ord & 31) & 1u);
        bad &= ~(1u << (ord & 31));
        if (slot == 1 && !done) {  // the run's end: the ring is free
          copies_wait<0>();
          __syncwarp();
        }
        float* const jo = joint.o<DP>(a, warp, slot);
#pragma unroll
        for (int h = 0; h < G; ++h) {
          float sum = warp_sum(l[h]);
          if (nan) sum = __int_as_float(0x7FC00000);
          if (h >= heads) continue;
#pragma unroll
          for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
              for (int b = PER; b < 32; b <<= 1) o[v][h][e] += __shfl_xor_sync(0xffffffffu, o[v][h][e], b);
            }
            const int d = (v * PER + lane) * 4;
            if (lane >= PER || d >= a.dim) continue;
            const float4 x = make_float4(o[v][h][0], o[v][h][1], o[v][h][2], o[v][h][3]);
            if (done)
              write_out<float>(a, mine, h, d, x, sum);
            else
              *reinterpret_cast<float4*>(jo + h * DP + d) = x;
          }
          if (lane == 0) {
            if (done) {
              write_lse(a, mine, h, m[h], sum);
            } else {
              joint.m[(2 * warp + slot) * a.group_size + h] = m[h];
              joint.l[(2 * warp + slot) * a.group_size + h] = sum;
            }
          }
        }
        if (!done && lane == 0) parts[2 * warp + slot] = mine;
        ++ord;
      }
      if (k + 1 < n) c.next(a);
    }
    copies_wait<0>();
  }
  join<float, DP>(a, run, joint);
  finish_empty<float>(a);
}

// ---------------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------------
// The workspace: counters of segments, then of groups of parts, (m, l) of joined parts, parts.  A segment's counter
// is that of the CTA it begins in: a run ends once, so no more than one segment begins in it and goes on.  What
// lies before the parts thus has the same place in every call, whatever its sequences, heads and head_dim, and no
// call's data lies where another's counters are.
constexpr size_t kCounterBytes = (size_t)kMaxCtas * 4;
constexpr size_t kCounter2Bytes = (size_t)kMaxCtas * 2 * 4, kTopBytes = (size_t)kMaxCtas * 2 * kMaxGroup * 8;

// Opt in to more than 48 KB of shared memory, once per kernel and device, whatever the call needs: what the
// kernel has statically counts too, so that 48 KB is not the limit of the dynamic part.
template <auto KERNEL>
bool allow_smem(int dev) {
  static std::atomic<uint64_t> done{0};
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

// `smem`: what the warps need; the parts of the join come on top.
template <auto KERNEL>
int launch(const AttnArgs& a, int dp, int per_sm, size_t smem, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return refuse(MLLM_ERR_CUDA, "mllm_paged_attn: no current CUDA device");
  smem += (size_t)kAttnWarps * a.group_size * (dp + 4) * 4;
  if (!allow_smem<KERNEL>(dev)) return refuse(MLLM_ERR_CUDA, "mllm_paged_attn: not enough shared memory");
  per_sm = std::min(per_sm, (int)(228 * 1024 / (smem + 1024 + 512)));
  // no more CTAs than runs of the shortest length over the whole table
  const int64_t blocks = ((int64_t)a.table_stride * a.page_len + kBlock - 1) / kBlock;
  if ((double)blocks * a.n_seq * a.n_kv * a.groups > 2147483648.0 - 65536.0)
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_paged_attn: the table can hold 2^31 blocks of 32 positions, over all kv heads");
  const int64_t most = (blocks + kMinBlocks - 1) / kMinBlocks * a.n_seq * a.n_kv * a.groups;
  const int grid = (int)std::min<int64_t>(most, std::min(kMaxCtas, sms * per_sm));
  KERNEL<<<grid, kAttnThreads, smem, st>>>(a);
  return launched("mllm_paged_attn: launch failed");
}

template <class T, class A, int DP, int NT>
int launch_mma(const AttnArgs& a, cudaStream_t st) {
  return launch<attn_mma_kernel<T, A, DP, NT>>(a, DP, mma_ctas<DP, NT>(), kAttnWarps * (mma_ring_bytes<DP>() + mma_query_bytes<T, A, DP, NT>()), st);
}
template <class T, class A>
int run_mma(AttnArgs& a, cudaStream_t st) {
  a.group_size = std::min(a.rep, a.dim <= 128 ? kMaxGroup : 8);
  a.groups = (a.rep + a.group_size - 1) / a.group_size;
  const bool one = a.group_size <= 8;
  if (a.dim <= 64) return one ? launch_mma<T, A, 64, 1>(a, st) : launch_mma<T, A, 64, 2>(a, st);
  if (a.dim <= 128) return one ? launch_mma<T, A, 128, 1>(a, st) : launch_mma<T, A, 128, 2>(a, st);
  return launch_mma<T, A, 256, 1>(a, st);
}
template <int DP, int G>
int launch_f32(const AttnArgs& a, cudaStream_t st) {
  return launch<attn_f32_kernel<DP, G>>(a, DP, f32_ctas<DP, G>(), kAttnWarps * (f32_ring_bytes<DP>() + f32_query_bytes<DP, G>()), st);
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
  return kCounterBytes + kCounter2Bytes + kTopBytes + (size_t)kMaxCtas * 2 * std::min(n_heads, kMaxGroup) * (head_dim + 4) * 4;
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
  if (row > (int64_t)1 << 30)  // empty sequences count a row's elements in 31 bits
    return refuse(MLLM_ERR_UNSUPPORTED, "mllm_paged_attn: more than 2^30 elements in a row");
  if (((uintptr_t)d_q & 15) || ((uintptr_t)d_out & 15) || q_stride * es % 16 || out_stride * es % 16)
    return refuse(MLLM_ERR_ARG, "mllm_paged_attn: rows must be 16-byte aligned");
  if (n_seq == 0) return MLLM_OK;
  if (!d_ws || ((uintptr_t)d_ws & 15) || ws_bytes < mllm_paged_attn_workspace(n_seq, n_heads, kv->head_dim))
    return refuse(MLLM_ERR_ARG, "mllm_paged_attn: workspace missing, misaligned or too small");
  AttnArgs a = {kv->k, kv->v, kv->page_stride, kv->head_stride, kv->pos_stride, kv->n_pages, kv->page_len,
                kv->n_kv_heads, kv->head_dim, d_q, q_stride, n_seq, n_heads, d_len, d_table, table_stride,
                scale, d_out, out_stride, d_lse};
  a.rep = n_heads / kv->n_kv_heads;
  int bits = 0;  // ceil(log2 page_len)
  while (((int64_t)1 << bits) < kv->page_len) ++bits;
  a.max_len = (int)std::min<int64_t>((int64_t)table_stride * kv->page_len, 0x7FFFFFFF);
  a.page_shift = 31 + bits;
  a.page_mult = ((uint64_t)1 << a.page_shift) / kv->page_len + 1;
  a.counter = static_cast<uint32_t*>(d_ws);
  uint8_t* at = static_cast<uint8_t*>(d_ws) + kCounterBytes;
  a.counter2 = reinterpret_cast<uint32_t*>(at);
  a.top = reinterpret_cast<float2*>(at + kCounter2Bytes);
  a.part = reinterpret_cast<float*>(at + kCounter2Bytes + kTopBytes);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MLLM_DTYPE_F16) return run_mma<__half, __half>(a, st);
  if (dtype == MLLM_DTYPE_BF16) return run_mma<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (kv->dtype == MLLM_DTYPE_F16) return run_mma<__half, float>(a, st);
  if (kv->dtype == MLLM_DTYPE_BF16) return run_mma<__nv_bfloat16, float>(a, st);
  return run_f32(a, st);
}
