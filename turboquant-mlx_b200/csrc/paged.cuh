// Paged caches: argument blocks, and how the decode kernels share out their work.
//
// A pool holds pages of `page` positions for every kv head; page_table[b][i] names the pool page of
// positions [i * page, (i + 1) * page) of sequence b.  Pages may be anywhere in the pool and may be shared
// between sequences (forks), so nothing here assumes an order.
//
// The unit of decode work is a tile: 32 or 64 consecutive positions (the kernel's choice) of one (sequence, kv head,
// group of up to 8 query heads), which lies in one page, or in two of 32 positions (page sizes are powers of two, 32
// at least).  A sequence has only the tiles that its newest token sees: all of them, or with a sliding window the tiles of the first
// `sinks` positions and those from position len - window on.  The tiles of a launch, numbered sequence by
// sequence, group by group, are cut into runs of equal cost, one per CTA, whatever the lengths of the
// sequences: a ragged batch loads every SM alike, and a single long sequence is split as finely as it needs.
// Starting and finishing a group costs a CTA time too, so each group counts group_cost tiles more than it has
// (a run that begins inside that lead begins at the group's first tile).  When there is a CTA for every group and
// splitting would not save two rounds of a CTA's warps, each group gets one CTA instead (16 windowed streams on 8 kv
// heads: 29 us, split over all SMs 36).  A CTA that holds all tiles of a
// group writes its output; otherwise it leaves a partial state (m, l, acc) in one of its two slots of the
// workspace and counts itself in, and the CTA that completes the count joins the states and writes the output.
// No CTA waits for another.
#pragma once

#include "common.cuh"

namespace tq {

constexpr int kMinPage = 32;         // positions of the smallest page
constexpr int kPagedRows = 8;        // query heads per group
constexpr int kMaxCtas = 256;        // of a decode launch (one per SM)
constexpr int kPlanEntries = 256;    // prefix entries of a CTA's plan (each covers ceil(batch / 256) sequences)
constexpr float kPagedLog2e = 1.4426950408889634f;

struct PagedHalf {                   // the K or the V half of a pool
  int format, bits, dtype;           // tq_kv_format; code width; element type of dense rows
  void* data;                        // packed words or dense rows, rows of one (page, head) contiguous
  float* norms;                      // packed rows only
  int64_t page_stride, head_stride;              // in 32-bit words (packed) or elements (dense)
  int64_t norm_page_stride, norm_head_stride;
  Table16 cent;
  SignMask signs;
};

struct PageView {
  const int* table;
  int64_t table_stride;
  int table_width, page_shift;
  int64_t n_pages;
  int* status;                       // set when a page id lies outside the pool

  __device__ __forceinline__ int capacity() const {
    const int64_t c = (int64_t)table_width << page_shift;
    return c > 0x7fff0000 ? 0x7fff0000 : (int)c;         // room for a tile behind the last position
  }
  __device__ __forceinline__ int entry(int b, int pos) const { return __ldg(table + b * table_stride + (pos >> page_shift)); }
  // Pool page of position `pos` of sequence b, -1 when the table names none in the pool.
  __device__ __forceinline__ int page_of(int b, int pos) const {
    const int id = entry(b, pos);
    return id >= 0 && id < n_pages ? id : -1;
  }
};

struct PagedDecodeArgs {
  PagedHalf k, v;
  PageView view;
  int batch, n_q_heads, n_kv_heads, n_rep, groups;     // groups = n_kv_heads * ceil(n_rep / 8)
  const int* lens;
  int window, sinks;                 // window 0: every position is visible
  int tile_shift;                    // tiles have 1 << tile_shift positions
  const void* q;
  int q_dtype, out_dtype;
  int64_t q_batch_stride, q_head_stride;
  void* out;
  int64_t out_batch_stride, out_head_stride;
  float scale_log2;                  // attn_scale * log2(e)
  uint32_t k_page_bytes, v_page_bytes, kn_page_bytes, vn_page_bytes;   // tensor-core kernel: page distances
  int* counters;                     // [kMaxCtas], zero between calls: CTAs of the split group that begins in CTA c
  float* part;                       // [2 * ctas][8][dim + 4]: acc (rotated domain), m (log2 domain), l, two unused
  int ctas, min_tiles, group_cost;   // grid of the main kernel; fewest tiles worth a CTA; what a group costs besides, in tiles
};

#ifdef __CUDACC__
// What the newest token of a sequence sees.
struct SeqSpan {
  int n;        // positions
  int lo;       // positions below lo are visible only as sinks
  int st, wt;   // tiles of the sinks; first tile behind them
  int tiles;
  __device__ __forceinline__ int tile_at(int j) const { return j < st ? j : j - st + wt; }
  __device__ __forceinline__ bool sees(int pos, int sinks) const { return pos < n && (pos >= lo || pos < sinks); }
};

__device__ __forceinline__ SeqSpan span_of(const PagedDecodeArgs& a, int b) {
  SeqSpan s;
  s.n = min(max(__ldg(a.lens + b), 0), a.view.capacity());
  s.lo = a.window > 0 ? max(0, s.n - a.window) : 0;
  const int full = (int)(((int64_t)s.n + (1 << a.tile_shift) - 1) >> a.tile_shift);
  s.st = s.lo > 0 ? (int)min(((int64_t)a.sinks + (1 << a.tile_shift) - 1) >> a.tile_shift, (int64_t)full) : 0;
  s.wt = max(s.lo >> a.tile_shift, s.st);
  s.tiles = s.st + full - s.wt;
  return s;
}

// What one group of a sequence costs in the plan.
__device__ __forceinline__ int cost_of(const PagedDecodeArgs& a, const SeqSpan& s) { return s.tiles > 0 ? s.tiles + a.group_cost : 0; }

__device__ __forceinline__ int plan_stride(const PagedDecodeArgs& a) { return (a.batch + kPlanEntries - 1) / kPlanEntries; }
__device__ __forceinline__ int plan_entries(const PagedDecodeArgs& a) { const int per = plan_stride(a); return (a.batch + per - 1) / per; }

// prefix[e] = cost of one group in the sequences in front of entry e, prefix[n] = of all sequences; behind them the
// largest cost of an entry and the number of entries that have any.  Called by every thread of the block; `prefix`
// holds kPlanInts ints.
constexpr int kPlanInts = kPlanEntries + 3;
// `early`: this thread's cost_early(), asked for ahead so that its load is on its way.
__device__ __forceinline__ int cost_early(const PagedDecodeArgs& a) {
  return (int)threadIdx.x < a.batch && plan_stride(a) == 1 ? cost_of(a, span_of(a, threadIdx.x)) : 0;
}
__device__ __forceinline__ void plan_costs(const PagedDecodeArgs& a, int* prefix, int early) {
  const int per = plan_stride(a), n = plan_entries(a);
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    int t = early;
    if (per != 1 || e != (int)threadIdx.x) {
      t = 0;
      for (int b = e * per; b < min(a.batch, (e + 1) * per); ++b) t += cost_of(a, span_of(a, b));
    }
    prefix[e + 1] = t;
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    int carry = 0, most = 0, some = 0;
    for (int e0 = 1; e0 <= n; e0 += 32) {
      const int e = e0 + threadIdx.x;
      int t = e <= n ? prefix[e] : 0;
      most = max(most, t);
      some += t != 0;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, t, k);
        if ((int)threadIdx.x >= k) t += o;
      }
      t += carry;
      if (e <= n) prefix[e] = t;
      carry = __shfl_sync(0xffffffffu, t, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    some = __reduce_add_sync(0xffffffffu, some);
    if (threadIdx.x == 0) {
      prefix[kPlanEntries + 1] = most;
      prefix[kPlanEntries + 2] = some;
    }
  }
  __syncthreads();
}

struct Plan {
  int64_t total, q;    // cost of the launch; cost of a run (the first `r` runs have one more)
  int ctas, r;
  bool whole;          // CTA c takes the c-th group that has tiles, whole
  __device__ __forceinline__ int64_t begin(int cta) const { return cta * q + min(cta, r); }
  // the CTA whose run holds point t of the numbering
  __device__ __forceinline__ int owner(int64_t t) const {
    const int64_t head = r * (q + 1);
    return t < head ? (int)(t / (q + 1)) : r + (int)((t - head) / q);
  }
};
__device__ __forceinline__ Plan make_paged_plan(const PagedDecodeArgs& a, const int* prefix) {
  Plan p;
  p.total = (int64_t)prefix[plan_entries(a)] * a.groups;
  const int most = prefix[kPlanEntries + 1] - a.group_cost, some = prefix[kPlanEntries + 2];
  if (plan_stride(a) == 1 && (int64_t)some * a.groups <= a.ctas) {
    // rounds of min_tiles tiles: the longest group alone, and an equal share of all
    const int64_t tiles = p.total - (int64_t)some * a.groups * a.group_cost;
    const int64_t share = (tiles + (int64_t)a.ctas * a.min_tiles - 1) / ((int64_t)a.ctas * a.min_tiles);
    p.whole = (most + a.min_tiles - 1) / a.min_tiles <= share + 1;
  } else {
    p.whole = false;
  }
  if (p.whole) {
    p.ctas = max(1, some * a.groups);
    p.q = p.r = 0;
    return p;
  }
  p.ctas = p.total >= (int64_t)a.ctas * a.min_tiles ? a.ctas : max(1, (int)(p.total + a.min_tiles - 1) / a.min_tiles);
  if (p.total < (1ll << 31)) {           // 32-bit division is a tenth of the 64-bit one
    p.q = (uint32_t)p.total / (uint32_t)p.ctas;
    p.r = (int)((uint32_t)p.total - (uint32_t)p.q * (uint32_t)p.ctas);
  } else {
    p.q = p.total / p.ctas;
    p.r = (int)(p.total - p.q * p.ctas);
  }
  return p;
}
// A tile of the numbering: sequence, (kv head, row group), tile inside the group.
struct Cursor {
  int b, group, j;
  SeqSpan span;        // of sequence b
  // the first tile at or behind point t; (batch, 0, 0) behind the last
  __device__ __forceinline__ void seek(const PagedDecodeArgs& a, const int* prefix, int64_t t) {
    const int per = plan_stride(a);
    int lo = 0, hi = plan_entries(a) - 1;
    if (t >= (int64_t)prefix[hi + 1] * a.groups) {
      b = a.batch;
      group = j = 0;
      span.tiles = 0;
      return;
    }
    while (lo < hi) {                            // last entry that does not begin behind t
      const int mid = (lo + hi + 1) / 2;
      if ((int64_t)prefix[mid] * a.groups <= t) lo = mid;
      else hi = mid - 1;
    }
    int64_t rest = t - (int64_t)prefix[lo] * a.groups;
    b = lo * per;
    span = span_of(a, b);
    int cost = cost_of(a, span);
    while (rest >= (int64_t)cost * a.groups) {
      rest -= (int64_t)cost * a.groups;
      span = span_of(a, ++b);
      cost = cost_of(a, span);
    }
    if (rest < (1ll << 31)) {
      group = (int)((uint32_t)rest / (uint32_t)cost);
      j = (int)((uint32_t)rest - (uint32_t)group * (uint32_t)cost);
    } else {
      group = (int)(rest / cost);
      j = (int)(rest - (int64_t)group * cost);
    }
    j = max(0, j - a.group_cost);
  }
  // both ends of CTA `cta`'s run (one warp)
  __device__ __forceinline__ void seek_run(const PagedDecodeArgs& a, const int* prefix, const Plan& plan, int cta, bool behind,
                                           int lane) {
    if (!plan.whole) {
      seek(a, prefix, plan.begin(cta + behind));
      return;
    }
    int k = cta / a.groups;                      // the k-th sequence that has tiles
    for (int b0 = 0;; b0 += 32) {
      const uint32_t some = __ballot_sync(0xffffffffu, b0 + lane < a.batch && prefix[b0 + lane + 1] != prefix[b0 + lane]);
      if (k < __popc(some)) {
        b = b0 + (int)__fns(some, 0, k + 1);
        break;
      }
      k -= __popc(some);
    }
    group = cta % a.groups;
    j = 0;
    span = span_of(a, b);
    if (behind) next_group(a);
  }
  // tiles from here to the end of the group, at most to `end`
  __device__ __forceinline__ int count_to(const Cursor& end) const {
    return (b == end.b && group == end.group ? end.j : span.tiles) - j;
  }
  __device__ __forceinline__ bool at(const Cursor& end) const { return b == end.b && group == end.group && j == end.j; }
  // to the first tile of the next group that has any
  __device__ __forceinline__ void next_group(const PagedDecodeArgs& a) {
    j = 0;
    if (++group < a.groups) return;
    group = 0;
    do {
      if (++b >= a.batch) {
        span.tiles = 0;
        return;
      }
      span = span_of(a, b);
    } while (span.tiles == 0);
  }
};

__device__ __forceinline__ float paged_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float load_elem(const void* base, int dtype, int64_t i) {
  return dtype == TQ_F32 ? reinterpret_cast<const float*>(base)[i]
         : dtype == TQ_F16 ? __half2float(reinterpret_cast<const __half*>(base)[i])
                           : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
}
__device__ __forceinline__ void store_elem(void* base, int dtype, int64_t i, float x) {
  if (dtype == TQ_F32) reinterpret_cast<float*>(base)[i] = x;
  else if (dtype == TQ_F16) reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// Output row of one query head, held by one warp (lane = EPL consecutive elements of the rotated
// accumulator): signs * butterfly(acc) / dim / l.  A row that saw nothing (l == 0) is zero.
template <int EPL>
__device__ __forceinline__ void finish_row(const PagedDecodeArgs& a, int b, int head, float (&v)[EPL], float l, int lane) {
  warp_butterfly<EPL>(v, lane);
  const float inv = l == 0.f ? 0.f : 1.0f / (l * (EPL * 32));
  const int64_t off = b * a.out_batch_stride + head * a.out_head_stride + lane * EPL;
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    store_elem(a.out, a.out_dtype, off + j, l == 0.f ? 0.f : v[j] * sign_at(a.v.signs, lane * EPL + j) * inv);
}
// Sequences without a tile get zeros, from the CTAs in turn.
__device__ __forceinline__ void zero_empty(const PagedDecodeArgs& a, int dim) {
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (span_of(a, b).tiles != 0) continue;
    for (int i = threadIdx.x; i < a.n_q_heads * dim; i += blockDim.x)
      store_elem(a.out, a.out_dtype, b * a.out_batch_stride + i / dim * a.out_head_stride + i % dim, 0.f);
  }
}

// Slot of CTA c's part of a group that begins in CTA c0: its tail piece (1) or its head piece (0).
__device__ __forceinline__ float* part_of(const PagedDecodeArgs& a, int c, int c0, int row, int dim) {
  return a.part + ((int64_t)(2 * c + (c == c0)) * kPagedRows + row) * (dim + 4);
}

// The CTA has stored its part of a split group and its threads have met: counts it in and says whether it was the last
// (release: everything before the meeting is visible to whoever sees the count; acquire: the others' parts are).  One
// thread.
__device__ __forceinline__ bool last_part(const PagedDecodeArgs& a, int c0, int c1) {
  int before;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + c0) : "memory");
  if (before != c1 - c0) return false;
  a.counters[c0] = 0;                // nobody else touches it before the next call
  return true;
}

// Joins one row of the parts c0 .. c1 of a group: m = max m_i, l = sum l_i 2^(m_i - m), acc likewise; one warp.  The
// first rows are on their way while the weights are worked out.
template <int EPL>
__device__ __forceinline__ void join_row(const PagedDecodeArgs& a, int c0, int c1, int row, int b, int head, int lane) {
  constexpr int DIM = EPL * 32;
  constexpr int kBatch = EPL <= 4 ? 16 : 8;          // parts whose rows a lane has in flight
  constexpr int kOwn = kMaxCtas / 32;                // lane i keeps the states of parts i, i + 32, ...
  const int n = c1 - c0 + 1;
  float x[kBatch][EPL], m[kOwn], w[kOwn];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float* p = part_of(a, c0 + min(i0 + k, n - 1), c0, row, DIM) + lane * EPL;
      if (EPL == 4) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(p));
        x[k][0] = f.x; x[k][EPL > 1 ? 1 : 0] = f.y; x[k][EPL > 2 ? 2 : 0] = f.z; x[k][EPL > 3 ? 3 : 0] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[k][j] = __ldcg(p + j);
      }
    }
  };
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    m[o] = -INFINITY;
    w[o] = 0.f;
    if (32 * o < n && 32 * o + lane < n) {
      const float2 f = __ldcg(reinterpret_cast<const float2*>(part_of(a, c0 + 32 * o + lane, c0, row, DIM) + DIM));
      m[o] = f.x;
      w[o] = f.y;
    }
  }
  load(0);
  float mx = -INFINITY, l = 0.f, v[EPL];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) mx = fmaxf(mx, m[o]);
  mx = warp_max(mx);
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const float f = m[o] == -INFINITY ? 1.f : paged_ex2(m[o] - mx);        // m = -inf: l is 0, or NaN (a missing page)
    l += w[o] * f;
    w[o] = f;
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) v[j] = 0.f;
#pragma unroll
  for (int o = 0; o < kOwn; ++o)
    for (int i0 = 32 * o; i0 < min(n, 32 * o + 32); i0 += kBatch) {
      if (i0 > 0) load(i0);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float f = __shfl_sync(0xffffffffu, w[o], (i0 + k) & 31);
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (i0 + k < n) v[j] += x[k][j] * f;
      }
    }
  finish_row<EPL>(a, b, head, v, warp_sum(l), lane);
}
#endif  // __CUDACC__

bool paged_mma_supported(const PagedDecodeArgs& a, int dim);
int launch_paged_mma(PagedDecodeArgs a, cudaStream_t st, bool* taken);

}  // namespace tq
