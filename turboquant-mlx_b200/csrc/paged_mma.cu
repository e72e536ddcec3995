// Decode attention over pages on tensor cores: head_dim 128, 3 / 4-bit values, 16-bit dense or 3 / 4-bit keys.
//
// A CTA owns an equal run of the launch's tiles (paged.cuh), W consumer warps that share nothing but tables while they
// stream it, and a producer warp.  Consumer w takes the tiles w, w + W, ... of a group from a ring of its own, S tiles
// deep; lane w of the producer fills it with bulk copies (key rows, key norms, value rows, value norms of a tile: 32
// positions with 16-bit keys, 64 with packed ones, of one page or of two pages of 32) and runs ahead into the next group
// while this one is finished.  The page id of a ring's next tile is already on its way when a copy is issued, so the
// indirection costs no waiting.  Per tile, in one pass:
//   scores : mma m16n8k16, A = query (rows 0-7 the 16-bit high parts of 8 heads, rows 8-15 their residuals), B = K^T.
//            Codes become 16-bit centroids two at a time through a table in shared memory, one copy per lane
//            (entry * 256 + lane * 4): conflict free, and for 4-bit codes one byte permute makes the address.
//   softmax: log2 domain, running maximum of score + log2(value norm) per head, so the 16-bit weights stay below 2^8
//            whatever the norms are; the sum counts the weights without the norm, in 32 bits.
//   values : out^T += V^T P.  The codes of two neighbouring positions are interleaved bit by bit field first, so that one
//            table entry is the pair of values the MMA wants side by side and nothing is permuted afterwards.
// At the end of a group the warps meet in shared memory; a group that lies in one CTA is finished there (butterfly,
// signs, / dim / l), otherwise its partial state goes to the workspace and the CTA that is last joins the states.
//
// Measured at 32 sequences of 8192 tokens, 32 / 8 heads, pages of 64: 16-bit keys + 3-bit values 109 us = 5.9 TB/s (0.91 of
// the copy peak: HBM-bound), 4 + 3 bits 93 us = 2.8 TB/s, 4 + 4 bits 82 us = 3.4 TB/s, 3 + 3 bits 90 us = 2.6 TB/s.  Packed
// halves are bound by latency inside the SM: two warps per scheduler (253 registers a thread) issue in 43 % of the cycles
// (integer pipe 38 %, shared-memory loads 44 to 51 %, tensor pipe 24 %), and what lies between is a lookup behind its
// address, a product behind its lookup, an exponential behind its product.  One sequence of 433
// tokens: 10 us, of 32768 with 16-bit keys: 18 us, where starting (2.6 us), the warps' meeting (1.5 us) and the join of
// the parts (5 us) are what is left beside the stream.
//
// Positions of a tile are dealt to MMA columns so that thread t of a quad owns 8 consecutive ones of each 32: norms come
// in 16-byte loads, and the rows that the threads of a warp read together lie in different banks where they can.
#include <cuda_fp16.h>
#include <string.h>

#include "paged.cuh"
#include "paged_host.cuh"
#include "scaled_book.cuh"

namespace tq {
namespace {

constexpr int kDim = 128;
constexpr uint32_t kSpin = 1u << 22;
constexpr float kRescale = 8.0f;        // log2 units a maximum may grow before the accumulators are rescaled
enum : int { KF_F16 = 0, KF_BF16 = 1, KF_P3 = 3, KF_P4 = 4 };
__host__ __device__ constexpr bool dense(int kf) { return kf == KF_F16 || kf == KF_BF16; }
__host__ __device__ constexpr int k_row_bytes(int kf) { return dense(kf) ? 256 : kf == KF_P3 ? 52 : 64; }
__host__ __device__ constexpr int v_row_bytes(int vb) { return vb == 3 ? 52 : 64; }

struct MmaTables {
  uint16_t k_c16[16], v_c16[16];   // centroids times a common factor beta, as f16 bits
  float k_post, v_post;            // what scores and accumulators are multiplied with: ... / beta
};

// Shared memory of one CTA, by address in the shared window (kBase: where dynamic memory begins when a kernel has no
// static arrays).  The pair tables lie at a multiple of their own size, so that a lookup's address is put together from
// bits alone: one byte permute, or a shift and one logic operation, and no add.
constexpr uint32_t kBase = 1024;
constexpr uint32_t kEnd = 228 * 1024;
constexpr uint32_t up16(uint32_t x) { return (x + 15) & ~15u; }
template <int KF, int VB, int W, int S, int H>
struct Layout {
  static constexpr uint32_t entry = dense(KF) ? 128 : 256;              // bytes between table entries (K and V side by side)
  static constexpr uint32_t v_entry = dense(KF) ? 0 : 128;
  static constexpr uint32_t entries = (KF == KF_P4 || VB == 4) ? 256 : 64;
  static constexpr uint32_t table_bytes = entries * entry;
  static constexpr uint32_t table = table_bytes > 16384 ? table_bytes : 16384, table_end = table + table_bytes;
  static constexpr uint32_t k_off = 0;
  static constexpr uint32_t tile = 32 * H;                              // positions of a tile
  static constexpr uint32_t kn_off = tile * k_row_bytes(KF);
  static constexpr uint32_t v_off = kn_off + (dense(KF) ? 0 : tile * 4);
  static constexpr uint32_t vn_off = v_off + tile * v_row_bytes(VB);
  static constexpr uint32_t stage = vn_off + tile * 4;
  // below the table: barriers, scalars, the plan; what does not fit goes behind the table, ring stages fill both sides
  static constexpr uint32_t full = kBase, empty = full + W * S * 8;     // mbarriers of the ring stages
  static constexpr uint32_t info = empty + W * S * 8;                   // per stage: first position of its tile | flags
  static constexpr uint32_t q_post = up16(info + W * S * 4);            // 8 floats
  static constexpr uint32_t ml = q_post + 32;                           // m, l of the warps that hand over rows: [2][W][8]
  static constexpr uint32_t flag = ml + 2 * W * 32;
  static constexpr uint32_t ends = flag + 16;                               // both ends of the CTA's run: [2] Cursor
  static constexpr uint32_t prefix = ends + 2 * sizeof(Cursor);
  static constexpr uint32_t norms = up16(prefix + kPlanInts * 4);   // per warp: key norms, log2 value norms, value norms
  static constexpr uint32_t q = norms + W * 3 * 32 * H * 4;                 // query fragments [k-step][lane][4]
  static constexpr uint32_t small_end = q + 8 * 32 * 16;
  static constexpr int xch_warps = (W + 1) / 2;
  static constexpr uint32_t xch_row = kDim + 4;                         // padded: conflict-free stores
  static constexpr uint32_t xch_bytes = xch_warps * 34 * 32 * 4;        // [xch_warps][34][32] or [xch_warps][8][xch_row]
  static constexpr bool xch_low = small_end + xch_bytes <= table;
  static constexpr uint32_t xch = xch_low ? small_end : table_end;
  static constexpr uint32_t low = xch_low ? xch + xch_bytes : small_end;       // ring stages 0 .. low_stages - 1
  static constexpr uint32_t high = xch_low ? table_end : xch + xch_bytes;      // the others
  static constexpr int low_fit = (int)((table - low) / stage);
  static constexpr int low_stages = low_fit < W * S ? low_fit : W * S;
  static constexpr uint32_t end = high + (W * S - low_stages) * stage;
  static_assert(small_end <= table, "the small arrays fit below the table");
  static_assert(xch_warps * 8 * xch_row * 4 <= xch_bytes, "row exchange fits");
  static_assert(low % 16 == 0 && high % 16 == 0 && stage % 16 == 0 && q % 16 == 0 && norms % 16 == 0, "alignment");
  static_assert(end <= kEnd, "shared memory of an SM");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t it = 0; it < kSpin; ++it)
    if (mbar_try(bar, parity)) return true;
  return false;
}
template <int W>
__device__ __forceinline__ void consumer_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(W * 32) : "memory");
}
// Two 32-bit floats at once.
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return r;
}
__device__ __forceinline__ void bulk_g2s(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Pure functions of their operands (not volatile), so that the compiler may interleave independent chains.
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a pair of floats as 16-bit high parts and residuals
template <bool BF>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}

// Which MMA slot the query element pair (e, e + 1), e even, goes to: k-step, quad thread, upper half of the k range.
// The assignment is free as long as keys use the same one; each thread's slots are consecutive bytes of a key row.
template <int KF>
__device__ __forceinline__ void query_slot(int e, int& ks, int& t, int& up) {
  if (dense(KF)) {
    t = (e >> 3) & 3;
    ks = 2 * (e >> 5) + ((e >> 2) & 1);
    up = (e >> 1) & 1;
  } else if (KF == KF_P4) {
    t = e >> 5;
    ks = (e >> 2) & 7;
    up = (e >> 1) & 1;
  } else {                       // 15 pairs in the words 3 t .. 3 t + 2, one in word 12
    const int pi = e < 120 ? (e % 30) / 2 : 15;
    t = e < 120 ? e / 30 : (e - 120) / 2;
    ks = pi >> 1;
    up = pi & 1;
  }
}
// Where the accumulators hold element e of a row: thread group g, slot s = 2 * (MMA tile) + (upper half of its rows).
// 4-bit values: 16 consecutive codes per g; 3-bit: word g, half of word 8 + g / 2, one code of word 12.
template <int VB>
__device__ __forceinline__ void value_slot(int e, int& g, int& s) {
  if (VB == 4) {
    g = e >> 4;
    s = e & 15;
  } else if (e < 80) {
    g = e / 10;
    s = e % 10;
  } else if (e < 120) {
    g = (e - 80) / 5;
    s = 10 + (e - 80) % 5;
  } else {
    g = e - 120;
    s = 15;
  }
}

// Table entries never change once built, so the loads are not volatile; OFF: a constant part of the address.
template <uint32_t OFF>
__device__ __forceinline__ uint32_t lut(uint32_t addr) {
  uint32_t v;
  asm("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(addr), "n"(OFF));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t addr) { return __uint_as_float(lds32(addr)); }
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void sts_f32(uint32_t addr, float v) { sts32(addr, __float_as_uint(v)); }

template <int KF, int VB, int W, int S, int H>
__global__ void __launch_bounds__((W + 1) * 32, 1)
paged_mma_kernel(const __grid_constant__ PagedDecodeArgs a, const __grid_constant__ MmaTables tb) {
  using L = Layout<KF, VB, W, S, H>;
  extern __shared__ __align__(1024) uint8_t smem[];       // shared address kBase
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t lane4 = lane * 4;
  int* prefix = reinterpret_cast<int*>(smem + L::prefix - kBase);
  if (smem_u32(smem) != kBase) {         // the layout above would not hold (the launcher has checked that it does)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0) atomicExch(a.view.status, 4);
    return;
  }
  auto stage_addr = [&](int w, int s) {
    const int k = w * S + s;
    return k < L::low_stages ? L::low + k * L::stage : L::high + (k - L::low_stages) * L::stage;
  };
  if (threadIdx.x == 0) sts32(L::flag, 0);
  if (threadIdx.x < W * S) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(L::full + 8 * threadIdx.x) : "memory");
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(L::empty + 8 * threadIdx.x), "n"(1) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Everything above overlaps the end of the kernel in front; everything below may read what that kernel wrote.  (The
  // tables could be built above, but while a kernel of this size runs in front there is no room on its SM to begin.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int early = cost_early(a);       // a length is on its way while the tables are built
  // pair tables, one copy per lane: K entry = (code of the lower element | code of the upper << bits), V entry =
  // (code of the lower position | code of the upper << bits)
  for (uint32_t i = threadIdx.x; i < L::entries * 32; i += (W + 1) * 32) {
    const uint32_t e = i >> 5, at = L::table + e * L::entry + lane4;
    if (!dense(KF)) {
      constexpr int KB = KF == KF_P4 ? 4 : 3;
      if (e < (1u << (2 * KB))) sts32(at, (uint32_t)tb.k_c16[e & ((1 << KB) - 1)] | ((uint32_t)tb.k_c16[e >> KB] << 16));
    }
    if (e < (1u << (2 * VB))) sts32(at + L::v_entry, (uint32_t)tb.v_c16[e & ((1 << VB) - 1)] | ((uint32_t)tb.v_c16[e >> VB] << 16));
  }
  plan_costs(a, prefix, early);   // also the barrier behind the tables
  zero_empty(a, kDim);
  const Plan plan = make_paged_plan(a, prefix);
  const int cta = blockIdx.x;
  if (plan.total == 0 || cta >= plan.ctas) return;
  const int rg_per_head = a.groups / a.n_kv_heads;
  // both ends of the run, found by a warp each
  Cursor* ends = reinterpret_cast<Cursor*>(smem + L::ends - kBase);
  if (warp < 2) {
    Cursor c;
    c.seek_run(a, prefix, plan, cta, warp == 1, lane);
    if (lane == 0) ends[warp] = c;
  }
  __syncthreads();
  Cursor cur = ends[0];
  const Cursor end = ends[1];
  if (cur.at(end)) return;

  // ---------------- producer: lane r fetches for ring r ----------------
  // Each lane walks its ring's tiles on its own; the warp executes that walk once for all of them.
  if (warp == W) {
    const bool polar = !dense(KF);
    const int row_mask = (1 << a.view.page_shift) - 1;
    Cursor fc = cur;                  // the piece the lane's next tile is in
    int i = lane, cnt = lane < W ? cur.count_to(end) : 0;       // cnt 0: the lane has no tile left
    int page[H];
    const bool small_page = H == 2 && a.view.page_shift == 5;
    const uint8_t *kb = nullptr, *vb = nullptr, *kn = nullptr, *vn = nullptr;      // the group's head in page 0
    auto bases = [&]() {
      const int head = rg_per_head == 1 ? fc.group : fc.group / rg_per_head;
      kb = reinterpret_cast<const uint8_t*>(a.k.data) + head * a.k.head_stride * (polar ? 4 : 2);
      vb = reinterpret_cast<const uint8_t*>(a.v.data) + head * a.v.head_stride * 4;
      kn = reinterpret_cast<const uint8_t*>(a.k.norms) + head * a.k.norm_head_stride * 4;
      vn = reinterpret_cast<const uint8_t*>(a.v.norms) + head * a.v.norm_head_stride * 4;
    };
    auto settle = [&]() {             // to the lane's next tile; its page id is on its way when this returns
      while (cnt != 0 && i >= cnt) {
        if (fc.j + cnt < fc.span.tiles) {      // the run ends inside this group
          cnt = 0;
          break;
        }
        i -= cnt;
        fc.next_group(a);
        cnt = fc.at(end) ? 0 : fc.count_to(end);
        if (cnt != 0) bases();
      }
      if (cnt != 0) {
        const int pos = fc.span.tile_at(fc.j + i) * L::tile;
        const int* entry = a.view.table + fc.b * a.view.table_stride + (pos >> a.view.page_shift);
        page[0] = __ldg(entry);
        // pages of 32 under tiles of 64: the second half has an entry of its own, if the sequence reaches it
        if (H == 2 && small_page) page[H - 1] = pos + 32 < fc.span.n ? __ldg(entry + 1) : -1;
      }
    };
    bases();
    settle();
    int s = 0, issued = 0;
    uint32_t phase = 1, idle = 0;     // a fresh stage counts as released
    while (__any_sync(0xffffffffu, cnt != 0)) {
      const bool go = cnt != 0 && mbar_try(L::empty + 8 * (lane * S + s), phase);
      if (go) {
        const int pos = fc.span.tile_at(fc.j + i) * L::tile;
        const uint32_t bar = L::full + 8 * (lane * S + s), st = stage_addr(lane, s);
        // copies `n` positions from row `row` of page `pg` behind position `at` of the stage
        auto copy = [&](uint32_t pg, uint32_t row, uint32_t at, uint32_t n) {
          bulk_g2s(st + L::k_off + at * k_row_bytes(KF), kb + (uint64_t)pg * a.k_page_bytes + row * k_row_bytes(KF), n * k_row_bytes(KF), bar);
          if (polar) bulk_g2s(st + L::kn_off + at * 4, kn + (uint64_t)pg * a.kn_page_bytes + row * 4, n * 4, bar);
          bulk_g2s(st + L::v_off + at * v_row_bytes(VB), vb + (uint64_t)pg * a.v_page_bytes + row * v_row_bytes(VB), n * v_row_bytes(VB), bar);
          bulk_g2s(st + L::vn_off + at * 4, vn + (uint64_t)pg * a.vn_page_bytes + row * 4, n * 4, bar);
        };
        const bool full = pos + (int)L::tile <= fc.span.n && (pos >= fc.span.lo || pos + (int)L::tile <= a.sinks);
        if (!small_page) {
          const bool ok = page[0] >= 0 && page[0] < a.view.n_pages;
          sts32(L::info + 4 * (lane * S + s), (uint32_t)pos | (ok ? (full ? 1u : 0u) : 6u));
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(ok ? L::stage : 0u) : "memory");
          if (ok) copy(page[0], pos & row_mask, 0, L::tile);
          else atomicExch(a.view.status, 1);
        } else {
          // a half that the token does not see needs no page; one that it sees and that has none is missing
          uint32_t flags = full ? 1u : 0u, have = 0;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const int p = pos + 32 * h;
            const bool seen = p < fc.span.n && (p + 32 > fc.span.lo || p < a.sinks);
            const bool ok = page[h] >= 0 && page[h] < a.view.n_pages;
            if (seen && ok) have |= 1u << h;
            if (seen && !ok) flags = (flags & ~1u) | (2u << h);
          }
          if (flags & 6u) atomicExch(a.view.status, 1);
          sts32(L::info + 4 * (lane * S + s), (uint32_t)pos | flags);
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                       "r"((uint32_t)__popc(have) * (L::stage / H)) : "memory");
#pragma unroll
          for (int h = 0; h < H; ++h)
            if ((have >> h) & 1u) copy(page[h], 0, 32 * h, 32);
        }
        ++issued;
        if (++s == S) {
          s = 0;
          phase ^= 1u;
        }
        i += W;
        settle();
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, go)) {
        idle = 0;
      } else {
        if (lds32(L::flag) != 0) break;
        if (++idle == kSpin) {
          sts32(L::flag, 1);
          if (lane == 0) atomicExch(a.view.status, 3);
          break;
        }
        __nanosleep(100);
      }
    }
    // every copy has landed before the CTA may end (bounded; the consumers have seen to it in all but the failed case)
    for (int n = max(0, issued - S); n < issued; ++n) mbar_wait(L::full + 8 * (lane * S + n % S), (n / S) & 1);
    return;
  }

  // Which position of a block of 32 column 2 t + c of n-group ng stands for: 8 t + (kNg ng + kC c), the places of two
  // neighbouring positions exchanged for odd t with kSwap.  3-bit rows are 13 words long: with c 4 rows apart the key
  // words of a load lie in 32 different banks; with 64-byte value rows the exchange halves the conflicts.
  constexpr bool kSwap = VB == 4;
  constexpr int kNg = KF == KF_P3 && VB == 3 ? 1 : 2, kC = KF == KF_P3 && VB == 3 ? 4 : 1;
  const int k_row0 = 8 * (g >> 1) + kC * ((g & 1) ^ (kSwap ? (g >> 1) & 1 : 0));
  const int v_row0 = 8 * t4 + kC * (kSwap ? t4 & 1 : 0), v_row1 = 8 * t4 + kC * (1 - (kSwap ? t4 & 1 : 0));
  const uint32_t nrm = L::norms + warp * 3 * 128 * H;          // [3][32 H]
  const uint32_t nrm_at = nrm + 4 * (kSwap ? lane ^ ((lane >> 3) & 1) : lane);      // the place of position `lane` in that order
  uint32_t lut_lane;                                     // table address of entry 0 in this lane's copy; opaque, so that
  asm("add.u32 %0, %1, %2;" : "=r"(lut_lane) : "r"(lane4), "n"(L::table));   // an address stays one logic operation
  auto k_lut = [&](uint32_t at) { return lut<0>(at); };
  auto v_lut = [&](uint32_t at) { return lut<L::v_entry>(at); };
  // byte j of a word (a pair of 4-bit codes) as a table address
  auto byte_at = [&](uint32_t w, int j) {
    return L::entry == 256 ? __byte_perm(w, lut_lane, 0x7604 | (j << 4))
                           : ((j == 0 ? w << 7 : w >> (8 * j - 7)) & 0x7F80u) | lut_lane;
  };
  // 6-bit field i of a word as a table address
  auto field_at = [&](uint32_t w, int i) {
    constexpr int sh = L::entry == 256 ? 8 : 7;
    return ((6 * i >= sh ? w >> (6 * i - sh) : w << (sh - 6 * i)) & (0x3Fu << sh)) | lut_lane;
  };

  uint32_t st = stage_addr(warp, 0);
  int us = 0;                        // stage of the tile consumed next
  uint32_t phase = 0;
  int i = warp;
  // the group's query rows, four elements of rows warp, warp + W per lane: fetched a group ahead
  constexpr int kRpw = (kPagedRows + W - 1) / W;
  auto load_query = [&](const Cursor& c, float (&x)[kRpw][4]) {
    const int kvh = rg_per_head == 1 ? c.group : c.group / rg_per_head;
#pragma unroll
    for (int k = 0; k < kRpw; ++k) {
      const int r = warp + k * W, rr = (c.group - kvh * rg_per_head) * kPagedRows + r;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[k][j] = r < kPagedRows && rr < a.n_rep
                      ? load_elem(a.q, a.q_dtype, c.b * a.q_batch_stride + (kvh * a.n_rep + rr) * a.q_head_stride + lane * 4 + j) : 0.f;
    }
  };
  float xq[kRpw][4];
  load_query(cur, xq);
  bool gave_up = false;              // a bounded wait failed: no more tiles, NaN for every group still to come
  while (true) {
    const int cnt = cur.count_to(end);
    const int b = cur.b, kvh = rg_per_head == 1 ? cur.group : cur.group / rg_per_head;
    const int r0 = (cur.group - kvh * rg_per_head) * kPagedRows;
    const int nr = min(kPagedRows, a.n_rep - r0), h0 = kvh * a.n_rep + r0;
    // ---------------- query fragments ----------------
#pragma unroll
    for (int k = 0; k < kRpw; ++k) {
      const int r = warp + k * W;
      if (r >= kPagedRows) break;
      float x[4] = {xq[k][0], xq[k][1], xq[k][2], xq[k][3]};
      if (!dense(KF)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] *= sign_at(a.k.signs, lane * 4 + j);
        warp_butterfly<4>(x, lane);
      }
      // scaled by a power of two to a maximum in [256, 512): any query fits the 16-bit pairs
      const float top = warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
      const int ex = top > 0.f && top < INFINITY ? 9 - (((__float_as_int(top) >> 23) & 255) - 126) : 0;
      const int up1 = ex / 2, up2 = ex - up1;           // two steps: each factor is a normal number
      const float f1 = __int_as_float((127 + up1) << 23), f2 = __int_as_float((127 + up2) << 23);
      if (lane == 0)
        sts_f32(L::q_post + 4 * r, tb.k_post * __int_as_float((127 - up1) << 23) * __int_as_float((127 - up2) << 23));
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        uint32_t hi, lo;
        split_pair<KF == KF_BF16>(x[j] * f1 * f2, x[j + 1] * f1 * f2, hi, lo);
        int ks, t, up;
        query_slot<KF>(lane * 4 + j, ks, t, up);
        const uint32_t at = L::q + ((ks * 32 + r * 4 + t) * 4 + 2 * up) * 4;
        sts32(at, hi);
        sts32(at + 4, lo);
      }
    }
    consumer_barrier<W>();
    uint32_t aq[8][4];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      const uint4 w = lds128(L::q + (ks * 32 + lane) * 16);
      aq[ks][0] = w.x; aq[ks][1] = w.y; aq[ks][2] = w.z; aq[ks][3] = w.w;
    }
    const float post = lds_f32(L::q_post + 4 * g);
    const bool last = cur.j + cnt < cur.span.tiles;       // the run ends inside this group
    Cursor nx = cur;
    if (!last) nx.next_group(a);
    const bool more = !last && !nx.at(end);
    if (more) load_query(nx, xq);

    float o[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    for (; i < cnt && !gave_up; i += W) {
      if (!mbar_wait(L::full + 8 * (warp * S + us), phase)) {      // gave up: everything this CTA produces from here on is NaN
        if (lane == 0) {
          sts32(L::flag, 1);
          atomicExch(a.view.status, 3);
        }
        break;
      }
      const uint32_t info = lds32(L::info + 4 * (warp * S + us));
      const int p0 = (int)(info & ~31u);
      const bool full = info & 1u;
#pragma unroll
      for (int h = 0; h < H; ++h) {   // norms: lane = position
        const bool seen = full || cur.span.sees(p0 + 32 * h + lane, a.sinks);
        const float vn = seen ? lds_f32(st + L::vn_off + lane4 + 128 * h) : 0.f;
        if (!dense(KF)) sts32(nrm_at + 128 * h, lds32(st + L::kn_off + lane4 + 128 * h));
        sts_f32(nrm_at + 128 * (H + h), lg2(fmaxf(vn, 1e-26f)));
        sts_f32(nrm_at + 128 * (2 * H + h), vn);
      }
      __syncwarp();
      // ---------------- scores ----------------
      float sc[4 * H][4];
#pragma unroll
      for (int ng = 0; ng < 4 * H; ++ng) {
        sc[ng][0] = sc[ng][1] = sc[ng][2] = sc[ng][3] = 0.f;
        const uint32_t row = st + L::k_off + (32 * (ng >> 2) + k_row0 + kNg * (ng & 3)) * k_row_bytes(KF);
        if (dense(KF)) {
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const uint4 w = lds128(row + t4 * 16 + it * 64);
            mma<KF == KF_BF16>(sc[ng], aq[2 * it], w.x, w.y);
            mma<KF == KF_BF16>(sc[ng], aq[2 * it + 1], w.z, w.w);
          }
        } else if (KF == KF_P4) {
          const uint4 w4 = lds128(row + t4 * 16);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma<false>(sc[ng], aq[2 * k], k_lut(byte_at(w[k], 0)), k_lut(byte_at(w[k], 1)));
            mma<false>(sc[ng], aq[2 * k + 1], k_lut(byte_at(w[k], 2)), k_lut(byte_at(w[k], 3)));
          }
        } else {
          uint32_t w[3];
#pragma unroll
          for (int k = 0; k < 3; ++k) w[k] = lds32(row + 12 * t4 + 4 * k);
          const uint32_t w12 = lds32(row + 48) >> (6 * t4);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const int p = 2 * ks, p1 = 2 * ks + 1;
            mma<false>(sc[ng], aq[ks], k_lut(field_at(w[p / 5], p % 5)),
                       p1 < 15 ? k_lut(field_at(w[p1 < 15 ? p1 / 5 : 0], p1 % 5)) : k_lut(field_at(w12, 0)));
          }
        }
      }
      // value fragments of one k-step (two position pairs per thread)
      auto load_values = [&](int step, uint32_t (&af)[8][4]) {
        uint32_t off[2][16];          // table addresses of the 16 slots, for the two position pairs of this k-step
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int vrow = 32 * (step >> 1) + kNg * (2 * (step & 1) + p);
          const uint32_t r0p = st + L::v_off + (v_row0 + vrow) * v_row_bytes(VB);
          const uint32_t r1p = st + L::v_off + (v_row1 + vrow) * v_row_bytes(VB);
          if (VB == 4) {
            const uint2 x = lds64(r0p + 8 * g), y = lds64(r1p + 8 * g);
            const uint32_t xs[2] = {x.x, x.y}, ys[2] = {y.x, y.y};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t ev = (xs[w] & 0x0F0F0F0Fu) | ((ys[w] << 4) & 0xF0F0F0F0u);     // even elements
              const uint32_t od = ((xs[w] >> 4) & 0x0F0F0F0Fu) | (ys[w] & 0xF0F0F0F0u);     // odd elements
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                off[p][8 * w + 2 * k] = byte_at(ev, k);
                off[p][8 * w + 2 * k + 1] = byte_at(od, k);
              }
            }
          } else {
            constexpr uint32_t kEven = 0707070707u;             // codes 0, 2, 4, 6, 8 of a word
            const int shb = 15 * (g & 1), shc = 3 * g;
            const uint32_t wb = 32 + 4 * (g >> 1);
            const uint32_t xa = lds32(r0p + 4 * g), ya = lds32(r1p + 4 * g), xb = lds32(r0p + wb) >> shb,
                           yb = lds32(r1p + wb) >> shb, xc = lds32(r0p + 48) >> shc, yc = lds32(r1p + 48) >> shc;
            // complementary masks (one logic operation); bits behind the fields are cut off by field_at
            const uint32_t ea = (xa & kEven) | ((ya << 3) & ~kEven), oa = ((xa >> 3) & kEven) | (ya & ~kEven);
            const uint32_t eb = (xb & kEven) | ((yb << 3) & ~kEven), ob = ((xb >> 3) & kEven) | (yb & ~kEven);
            const uint32_t ec = (xc & kEven) | ((yc << 3) & ~kEven);
#pragma unroll
            for (int k = 0; k < 5; ++k) {
              off[p][2 * k] = field_at(ea, k);
              off[p][2 * k + 1] = field_at(oa, k);
            }
            off[p][10] = field_at(eb, 0);
            off[p][11] = field_at(ob, 0);
            off[p][12] = field_at(eb, 1);
            off[p][13] = field_at(ob, 1);
            off[p][14] = field_at(eb, 2);
            off[p][15] = field_at(ec, 0);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          af[j][0] = v_lut(off[0][2 * j]);
          af[j][1] = v_lut(off[0][2 * j + 1]);
          af[j][2] = v_lut(off[1][2 * j]);
          af[j][3] = v_lut(off[1][2 * j + 1]);
        }
      };
      // the first step's lookups wait for nothing: they fill the time the score products and the softmax take
      // ---------------- softmax: head g ----------------
      float s2[8 * H], vn[8 * H], top = -INFINITY;       // [4 h + n-group][c]
      const float2 post2 = make_float2(post, post);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        // norms of this thread's 8 positions of the block, in the order of the tile
        float kn[8], lv[8], vo[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t at = nrm + 128 * h + 32 * t4 + 16 * q;
          const uint4 x = dense(KF) ? make_uint4(0, 0, 0, 0) : lds128(at), y = lds128(at + 128 * H), z = lds128(at + 256 * H);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            kn[4 * q + k] = __uint_as_float(xs[k]);
            lv[4 * q + k] = __uint_as_float(ys[k]);
            vo[4 * q + k] = __uint_as_float(zs[k]);
          }
        }
#pragma unroll
        for (int ng = 0; ng < 4; ++ng) {     // high part and residual of the query, scale, key norm
          const int i0 = kNg * ng, i1 = kNg * ng + kC, to = 8 * h + 2 * ng;
          const float (&c)[4] = sc[4 * h + ng];
          float2 v = mul2(add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])), post2);
          if (!dense(KF)) v = mul2(v, make_float2(kn[i0], kn[i1]));
          if (!full) {
            const int pos = p0 + 32 * h + kNg * ng;
            const bool missing = (info >> (1 + h)) & 1u;
            if (!cur.span.sees(pos + v_row0, a.sinks)) v.x = -INFINITY;
            if (!cur.span.sees(pos + v_row1, a.sinks)) v.y = -INFINITY;
            if (missing) v.x = v.y = __int_as_float(0x7fc00000);
          }
          s2[to] = v.x;
          s2[to + 1] = v.y;
          vn[to] = vo[i0];
          vn[to + 1] = vo[i1];
          const float2 u = add2(v, make_float2(lv[i0], lv[i1]));
          top = fmaxf(top, fmaxf(u.x, u.y));
        }
      }
      if (__any_sync(0xffffffffu, top > m_run + kRescale)) {       // also for the first visible tile
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool grow = top > m_run + kRescale;
        const float alpha = grow ? (m_run == -INFINITY ? 0.f : paged_ex2(m_run - top)) : 1.f;
        if (grow) m_run = top;
        l_run *= alpha;
        const float al0 = __shfl_sync(0xffffffffu, alpha, 8 * t4);      // heads 2 t4 and 2 t4 + 1
        const float al1 = __shfl_sync(0xffffffffu, alpha, 8 * t4 + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j][0] *= al0; o[j][1] *= al1; o[j][2] *= al0; o[j][3] *= al1;
        }
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
      uint32_t pb[4 * H];
#pragma unroll
      for (int ng = 0; ng < 4 * H; ++ng) {
        const float2 d = add2(make_float2(s2[2 * ng], s2[2 * ng + 1]), make_float2(-m_use, -m_use));
        const float2 e = make_float2(paged_ex2(d.x), paged_ex2(d.y));
        l_run += e.x + e.y;
        const float2 w = mul2(e, make_float2(vn[2 * ng], vn[2 * ng + 1]));
        const __half2 h = __floats2half2_rn(w.x, w.y);
        pb[ng] = *reinterpret_cast<const uint32_t*>(&h);
      }
      // ---------------- values ----------------
#pragma unroll
      for (int step = 0; step < 2 * H; ++step) {
        uint32_t af0[8][4];
        load_values(step, af0);
#pragma unroll
        for (int j = 0; j < 8; ++j) mma<false>(o[j], af0[j], pb[2 * step], pb[2 * step + 1]);
      }
      __syncwarp();            // every lane is done with the stage (and with the norms)
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(L::empty + 8 * (warp * S + us)) : "memory");
      if (++us == S) {
        us = 0;
        phase ^= 1u;
      }
      st = stage_addr(warp, us);
    }
    i -= cnt;                  // the warp's first tile of the next group

    // ---------------- the warps meet ----------------
    // the upper half of the warps hands its state to the lower half, which hands rows to one warp per head
    constexpr int HW = L::xch_warps;
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (warp >= HW) {
      const uint32_t to = L::xch + (warp - HW) * 34 * 128 + lane4;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) sts_f32(to + (4 * j + c) * 128, o[j][c]);
      sts_f32(to + 32 * 128, m_run);
      sts_f32(to + 33 * 128, l_run);
    }
    consumer_barrier<W>();
    if (warp < HW && warp + HW < W) {
      const uint32_t from = L::xch + warp * 34 * 128 + lane4;
      const float m2 = lds_f32(from + 32 * 128), l2 = lds_f32(from + 33 * 128);
      const float mx = fmaxf(m_run, m2);
      // a state that saw nothing has m = -inf; one that met a missing page then has l = NaN, which must live on
      const float fa = m_run == -INFINITY ? 1.f : paged_ex2(m_run - mx), fb = m2 == -INFINITY ? 1.f : paged_ex2(m2 - mx);
      l_run = l_run * fa + l2 * fb;
      m_run = mx;
      const float fa0 = __shfl_sync(0xffffffffu, fa, 8 * t4), fa1 = __shfl_sync(0xffffffffu, fa, 8 * t4 + 4);
      const float fb0 = __shfl_sync(0xffffffffu, fb, 8 * t4), fb1 = __shfl_sync(0xffffffffu, fb, 8 * t4 + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          o[j][c] = o[j][c] * ((c & 1) ? fa1 : fa0) + lds_f32(from + (4 * j + c) * 128) * ((c & 1) ? fb1 : fb0);
    }
    consumer_barrier<W>();
    if (warp < HW) {
      const uint32_t to = L::xch + warp * kPagedRows * L::xch_row * 4;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) sts_f32(to + ((2 * t4 + (c & 1)) * L::xch_row + (2 * j + (c >> 1)) * 8 + g) * 4, o[j][c]);
      if (t4 == 0) {
        sts_f32(L::ml + (warp * 8 + g) * 4, m_run);
        sts_f32(L::ml + ((W + warp) * 8 + g) * 4, l_run);
      }
    }
    consumer_barrier<W>();
    // Behind a barrier that every consumer has passed.  The producer, which also sets the flag, does not join it, so the
    // warps may see its failure in this group or in the next: until then a warp waits (bounded) for tiles that do not come.
    gave_up = lds32(L::flag) != 0;
    for (int r = warp; r < nr; r += W) {
      float mx = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t at[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int gg, sl;
        value_slot<VB>(lane * 4 + j, gg, sl);
        at[j] = L::xch + (r * L::xch_row + sl * 8 + gg) * 4;
      }
#pragma unroll
      for (int w = 0; w < HW; ++w) mx = fmaxf(mx, lds_f32(L::ml + (w * 8 + r) * 4));
#pragma unroll
      for (int w = 0; w < HW; ++w) {
        const float mw = lds_f32(L::ml + (w * 8 + r) * 4);
        const float fw = mw == -INFINITY ? 1.f : paged_ex2(mw - mx);
        l += lds_f32(L::ml + ((W + w) * 8 + r) * 4) * fw;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += lds_f32(at[j] + w * kPagedRows * L::xch_row * 4) * fw;
      }
      if (gave_up) l = __int_as_float(0x7fc00000);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= tb.v_post;
      if (cnt == cur.span.tiles) {
        finish_row<4>(a, b, h0 + r, v, l, lane);
      } else {
        float* part = part_of(a, cta, cur.j == 0 ? cta : -1, r, kDim);
        *reinterpret_cast<float4*>(part + lane * 4) = make_float4(v[0], v[1], v[2], v[3]);
        if (lane == 0) {
          part[kDim] = mx;
          part[kDim + 1] = l;
        }
      }
    }
    if (cnt != cur.span.tiles) {
      // where the group begins in the plan's numbering: from the end of this run, or from its beginning
      const int64_t first = cur.j == 0 ? plan.begin(cta + 1) - end.j : plan.begin(cta) - cur.j;
      const int c0 = plan.owner(first), c1 = plan.owner(first + cur.span.tiles - 1);
      consumer_barrier<W>();           // the whole part is on its way
      if (threadIdx.x == 0) sts32(L::flag + 4, last_part(a, c0, c1));
      consumer_barrier<W>();
      if (lds32(L::flag + 4))
        for (int r = warp; r < nr; r += W) join_row<4>(a, c0, c1, r, b, h0 + r, lane);
    }
    if (!more) return;
    cur = nx;
    // the next group's first stores to q, xch and ml come behind a barrier that every reader above has passed
  }
}

// ---- host side ---------------------------------------------------------------------------------------------
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int KF, int VB, int W, int S, int H>
int launch(PagedDecodeArgs& a, const MmaTables& tb, cudaStream_t st) {
  using L = Layout<KF, VB, W, S, H>;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_mma_kernel<KF, VB, W, S, H>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(L::end - kBase));
    if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  a.tile_shift = H == 2 ? 6 : 5;
  a.min_tiles = W;
  a.group_cost = W;              // a round of the warps; 32 sequences of 0 to 8192 tokens 62 us (0: 74 us, 2 W: 62 us)
  return launch_dependent("tq_paged_decode", paged_mma_kernel<KF, VB, W, S, H>, dim3(a.ctas), (W + 1) * 32, L::end - kBase, st, a, tb);
}

}  // namespace

// The layout of shared memory counts on where dynamic memory begins.
bool base_holds() {
  static int known[64] = {0};          // 1: holds, 2: does not
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!known[dev]) {
    int v = 0;
    known[dev] = cudaDeviceGetAttribute(&v, cudaDevAttrReservedSharedMemoryPerBlock, dev) == cudaSuccess && v == (int)kBase ? 1 : 2;
  }
  return known[dev] == 1;
}

// Queries in 32 bits ask for 32-bit weights and take the general kernel.
bool paged_mma_supported(const PagedDecodeArgs& a, int dim) {
  if (dim != kDim || a.q_dtype == TQ_F32 || a.v.format != TQ_KV_POLAR || (a.v.bits != 3 && a.v.bits != 4)) return false;
  if (!base_holds()) return false;
  if (!aligned16(a.v.data) || a.v.page_stride % 4 || a.v.head_stride % 4) return false;
  if (!aligned16(a.v.norms) || a.v.norm_page_stride % 4 || a.v.norm_head_stride % 4) return false;
  if (!aligned16(a.k.data)) return false;
  // page distances travel as 32-bit byte counts
  if (a.k.page_stride >= (1ll << 30) || a.v.page_stride >= (1ll << 30) || a.k.norm_page_stride >= (1ll << 30) ||
      a.v.norm_page_stride >= (1ll << 30))
    return false;
  if (a.k.format == TQ_KV_DENSE) return a.k.dtype != TQ_F32 && a.k.page_stride % 8 == 0 && a.k.head_stride % 8 == 0;
  return (a.k.bits == 3 || a.k.bits == 4) && a.k.page_stride % 4 == 0 && a.k.head_stride % 4 == 0 && aligned16(a.k.norms) &&
         a.k.norm_page_stride % 4 == 0 && a.k.norm_head_stride % 4 == 0;
}

// *taken: whether the kernel takes the call (its codebooks may not fit 16 bits).
int launch_paged_mma(PagedDecodeArgs a, cudaStream_t st, bool* taken) {
  MmaTables tb;
  memset(&tb, 0, sizeof(tb));
  const ScaledBook vb = scaled_book(a.v.cent.v, 1 << a.v.bits);
  *taken = vb.good;
  if (!*taken) return TQ_OK;
  memcpy(tb.v_c16, vb.c16, sizeof(tb.v_c16));
  tb.v_post = 1.0f / vb.beta;
  tb.k_post = a.scale_log2;
  a.k_page_bytes = (uint32_t)(a.k.page_stride * (a.k.format == TQ_KV_DENSE ? 2 : 4));
  a.v_page_bytes = (uint32_t)(a.v.page_stride * 4);
  a.kn_page_bytes = (uint32_t)(a.k.norm_page_stride * 4);
  a.vn_page_bytes = (uint32_t)(a.v.norm_page_stride * 4);
  if (a.k.format == TQ_KV_POLAR) {
    const ScaledBook kb = scaled_book(a.k.cent.v, 1 << a.k.bits);
    *taken = kb.good;
    if (!*taken) return TQ_OK;
    memcpy(tb.k_c16, kb.c16, sizeof(tb.k_c16));
    tb.k_post = a.scale_log2 / ((float)kDim * kb.beta);
  }
  const bool v3 = a.v.bits == 3;
  // Warps, ring stages and blocks of 32 positions per tile, by format; us for 32 sequences of 8192 tokens, 32 / 8 heads.
  // 16-bit keys: as many bytes in flight as fit; 8 warps x 2 stages 110 (7 x 2: 111, 8 x 1: 150, 11 x 1: 130).
  // Packed keys: a tile of two blocks gives a warp two independent chains; 4 + 3 bits 7 warps x 2 blocks 94 (8 x 1: 116,
  // 11 x 1: 108), 4 + 4 bits 84 (113, 104), 3 + 4 bits 88 (116, 108).  The small tables of 3 + 3 bits leave room for 11
  // warps: 91 (7 x 2 blocks: 100, 11 x 1: 110, 14 x 1: 111).
  if (a.k.format == TQ_KV_DENSE) {
    if (a.k.dtype == TQ_BF16) return v3 ? launch<KF_BF16, 3, 8, 2, 1>(a, tb, st) : launch<KF_BF16, 4, 8, 2, 1>(a, tb, st);
    return v3 ? launch<KF_F16, 3, 8, 2, 1>(a, tb, st) : launch<KF_F16, 4, 8, 2, 1>(a, tb, st);
  }
  if (a.k.bits == 3) return v3 ? launch<KF_P3, 3, 11, 2, 2>(a, tb, st) : launch<KF_P3, 4, 7, 2, 2>(a, tb, st);
  return v3 ? launch<KF_P4, 3, 7, 2, 2>(a, tb, st) : launch<KF_P4, 4, 7, 2, 2>(a, tb, st);
}

}  // namespace tq
