// Decode attention over pages on tensor cores: head_dim 128, 3 / 4-bit values, 16-bit dense or 3 / 4-bit keys.
//
// A CTA owns an equal run of the launch's tiles (paged.cuh) and W warps that share nothing but tables while they
// stream it: warp w takes the tiles w, w + W, ... of a group, fetches each with four bulk copies (key rows, key norms,
// value rows, value norms of 32 positions of one page) into a ring of its own, S tiles deep, and runs ahead into the
// next group while it finishes this one.  The page id of the tile after next is already on its way when a copy is
// issued, so the indirection costs no waiting.  Per tile, in one pass:
//   scores : mma m16n8k16, A = query (rows 0-7 the 16-bit high parts of 8 heads, rows 8-15 their residuals), B = K^T.
//            Codes become 16-bit centroids two at a time through a table in shared memory, one copy per lane
//            (entry * 256 + lane * 4): conflict free, and for 4-bit codes one byte permute makes the address.
//   softmax: log2 domain, running maximum of score + log2(value norm) per head, so the 16-bit weights stay below 2^8
//            whatever the norms are; the sum counts the weights without the norm, in 32 bits.
//   values : out^T += V^T P.  The codes of two neighbouring positions are interleaved bit by bit field first, so that one
//            table entry is the pair of values the MMA wants side by side and nothing is permuted afterwards.
// At the end of a group the warps meet in shared memory; a group that lies in one CTA is finished there (butterfly,
// signs, / dim / l), otherwise its partial state goes to the workspace and paged_merge_kernel joins it.
//
// Positions of a tile are dealt to MMA columns so that thread t of a quad owns 8 consecutive ones (norms come in two
// 16-byte loads); with 4-bit values the two positions of a pair change places in every other block of 8, which halves
// the bank conflicts of the 64-byte value rows.
#include <cuda_fp16.h>
#include <string.h>

#include <mutex>

#include "paged.cuh"
#include "paged_host.cuh"

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

// Shared memory of one CTA.
template <int KF, int VB, int W, int S>
struct Layout {
  static constexpr int entry = dense(KF) ? 128 : 256;                  // bytes between table entries (K and V side by side)
  static constexpr int v_entry = dense(KF) ? 0 : 128;
  static constexpr int entries = (KF == KF_P4 || VB == 4) ? 256 : 64;
  static constexpr int table = 0;
  static constexpr int q = table + entries * entry;                    // query fragments [k-step][lane][4]
  static constexpr int norms = q + 8 * 32 * 16;                        // per warp: key norms, log2 value norms, value norms of a tile
  static constexpr int xch_warps = (W + 1) / 2;
  static constexpr int xch_row = kDim + 4;                             // padded: conflict-free stores
  static constexpr int xch = norms + W * 3 * 32 * 4;                   // [xch_warps][8][xch_row] or [xch_warps][34][32]
  static constexpr int xch_bytes = xch_warps * 34 * 32 * 4;
  static constexpr int k_off = 0;
  static constexpr int kn_off = 32 * k_row_bytes(KF);
  static constexpr int v_off = kn_off + (dense(KF) ? 0 : 128);
  static constexpr int vn_off = v_off + 32 * v_row_bytes(VB);
  static constexpr int stage_bytes = vn_off + 128;
  static constexpr int ring = xch + xch_bytes;
  static constexpr int total = ring + W * S * stage_bytes;
  static_assert(xch_warps * 8 * xch_row * 4 <= xch_bytes, "row exchange fits");
  static_assert(ring % 16 == 0 && stage_bytes % 16 == 0 && q % 16 == 0 && norms % 16 == 0, "alignment");
  static_assert(total + 6 * 1024 <= 227 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t it = 0; it < kSpin; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
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

// What a warp fetches next: walks the warp's tiles of the CTA's run, one tile ahead of its page id.
struct Feed {
  Cursor c;
  int64_t t, t_end;      // run position of the current piece's first tile; end of the run
  int i, cnt, page;      // tile inside the piece (first: c.j); tiles of the piece; page of tile i, < 0: not in the pool
};

template <int KF, int VB, int W, int S>
__global__ void __launch_bounds__(W * 32, 1)
paged_mma_kernel(const __grid_constant__ PagedDecodeArgs a, const __grid_constant__ MmaTables tb) {
  using L = Layout<KF, VB, W, S>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int prefix[kPlanEntries + 1];
  __shared__ __align__(8) uint64_t bars[W * S];
  __shared__ float q_post_s[kPagedRows];
  __shared__ float m_s[W][kPagedRows], l_s[W][kPagedRows];
  __shared__ int gave_up_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = smem_u32(smem) + L::ring + warp * S * L::stage_bytes;
  const uint32_t bar0 = smem_u32(bars) + warp * S * 8;

  if (threadIdx.x == 0) gave_up_s = 0;
  if (lane == 0) {
    for (int s = 0; s < S; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8 * s) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // pair tables, one copy per lane: K entry = (code of the lower element | code of the upper << bits), V entry =
  // (code of the lower position | code of the upper << bits)
  for (int i = threadIdx.x; i < L::entries * 32; i += W * 32) {
    const int e = i >> 5;
    uint32_t* at = reinterpret_cast<uint32_t*>(smem + L::table + e * L::entry) + (i & 31);
    if (!dense(KF)) {
      constexpr int KB = KF == KF_P4 ? 4 : 3;
      if (e < (1 << (2 * KB))) at[0] = (uint32_t)tb.k_c16[e & ((1 << KB) - 1)] | ((uint32_t)tb.k_c16[e >> KB] << 16);
    }
    if (e < (1 << (2 * VB))) at[L::v_entry / 4] = (uint32_t)tb.v_c16[e & ((1 << VB) - 1)] | ((uint32_t)tb.v_c16[e >> VB] << 16);
  }
  plan_tiles(a, prefix);          // also the barrier behind the tables
  const Plan plan = make_paged_plan(a, prefix);
  const int cta = blockIdx.x;
  if (plan.total == 0 || cta >= plan.ctas) return;
  const int rg_per_head = a.groups / a.n_kv_heads;

  // ---------------- the warp's copies ----------------
  Feed f;
  f.t = plan.begin(cta);
  f.t_end = plan.begin(cta + 1);
  f.c.seek(a, prefix, f.t);
  f.cnt = (int)min((int64_t)(f.c.span.tiles - f.c.j), f.t_end - f.t);
  f.i = warp;
  Cursor cur = f.c;
  int64_t run = f.t;
  const int64_t run_end = f.t_end;
  uint32_t bad = 0;               // bit s: the tile of stage s has no page in the pool
  int issued = 0, used = 0;       // tiles fetched and consumed by this warp
  auto settle = [&]() {           // to the next tile this warp owns; starts loading its page id
    while (f.i >= f.cnt) {
      f.t += f.cnt;
      if (f.t >= f.t_end) {
        f.cnt = 0;
        return;
      }
      f.c.next_group(a);
      f.cnt = (int)min((int64_t)f.c.span.tiles, f.t_end - f.t);
      f.i = warp;
    }
    const int pos = f.c.span.tile_at(f.c.j + f.i) * kPagedTile;
    f.page = __ldg(a.view.table + f.c.b * a.view.table_stride + (pos >> a.view.page_shift));
  };
  auto fetch = [&]() {            // issues the copies of the current tile into the next stage
    if (f.cnt == 0) return;
    const int s = issued % S;
    const int pos = f.c.span.tile_at(f.c.j + f.i) * kPagedTile;
    const int row = pos & ((1 << a.view.page_shift) - 1);
    const int head = f.c.group / rg_per_head;
    const bool ok = f.page >= 0 && f.page < a.view.n_pages;
    bad = (bad & ~(1u << s)) | (ok ? 0u : 1u << s);
    if (lane == 0) {
      const uint32_t bar = bar0 + 8 * s, st = ring + s * L::stage_bytes;
      const uint32_t tx = ok ? L::stage_bytes : 0;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(tx) : "memory");
      if (ok) {
        const int64_t page = f.page;
        constexpr int kunit = dense(KF) ? 2 : 4;
        bulk_g2s(st + L::k_off,
                 reinterpret_cast<const uint8_t*>(a.k.data) + (page * a.k.page_stride + head * a.k.head_stride) * kunit +
                     (int64_t)row * k_row_bytes(KF),
                 32 * k_row_bytes(KF), bar);
        if (!dense(KF))
          bulk_g2s(st + L::kn_off, a.k.norms + page * a.k.norm_page_stride + head * a.k.norm_head_stride + row, 128, bar);
        bulk_g2s(st + L::v_off,
                 reinterpret_cast<const uint8_t*>(a.v.data) + (page * a.v.page_stride + head * a.v.head_stride) * 4 +
                     (int64_t)row * v_row_bytes(VB),
                 32 * v_row_bytes(VB), bar);
        bulk_g2s(st + L::vn_off, a.v.norms + page * a.v.norm_page_stride + head * a.v.norm_head_stride + row, 128, bar);
      } else {
        atomicExch(a.view.status, 1);
      }
    }
    ++issued;
    f.i += W;
    settle();
  };
  settle();
#pragma unroll
  for (int s = 0; s < S; ++s) fetch();

  // this thread's rows of a tile: key row of n-group ng: k_row0 + 2 ng; value rows of its ng-th pair: v_row0 + 2 ng, v_row1 + 2 ng
  constexpr bool kSwap = VB == 4;
  const int k_row0 = 8 * (g >> 1) + ((g & 1) ^ (kSwap ? (g >> 1) & 1 : 0));
  const int v_row0 = 8 * t4 + (kSwap ? t4 & 1 : 0), v_row1 = 8 * t4 + 1 - (kSwap ? t4 & 1 : 0);
  const uint32_t lane4 = lane * 4;
  float* nrm = reinterpret_cast<float*>(smem + L::norms) + warp * 96;
  const int nrm_at = kSwap ? lane ^ ((lane >> 3) & 1) : lane;      // the place of position `lane` in that order
  const uint8_t* table = smem + L::table;
  auto k_lut = [&](uint32_t off) { return *reinterpret_cast<const uint32_t*>(table + off); };
  auto v_lut = [&](uint32_t off) { return *reinterpret_cast<const uint32_t*>(table + L::v_entry + off); };
  // byte j of a word as a table offset: byte 1 = the code pair, byte 0 = the lane's copy
  auto byte_off = [&](uint32_t w, int j) {
    return L::entry == 256 ? __byte_perm(w, lane4, 0x5504 | (j << 4))
                           : ((j == 0 ? w << 7 : w >> (8 * j - 7)) & 0x7F80u) | lane4;
  };
  // 6-bit field i of a word as a table offset
  auto field_off = [&](uint32_t w, int i) {
    constexpr int sh = L::entry == 256 ? 8 : 7;
    return ((6 * i >= sh ? w >> (6 * i - sh) : w << (sh - 6 * i)) & (0x3Fu << sh)) | lane4;
  };

  while (run < run_end) {
    const int cnt = (int)min((int64_t)(cur.span.tiles - cur.j), run_end - run);
    const int b = cur.b, kvh = cur.group / rg_per_head, r0 = (cur.group % rg_per_head) * kPagedRows;
    const int nr = min(kPagedRows, a.n_rep - r0), h0 = kvh * a.n_rep + r0;
    // ---------------- query fragments ----------------
    for (int r = warp; r < kPagedRows; r += W) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = r < nr ? load_elem(a.q, a.q_dtype, b * a.q_batch_stride + (h0 + r) * a.q_head_stride + lane * 4 + j) : 0.f;
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
      if (lane == 0) q_post_s[r] = tb.k_post * __int_as_float((127 - up1) << 23) * __int_as_float((127 - up2) << 23);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        uint32_t hi, lo;
        split_pair<KF == KF_BF16>(x[j] * f1 * f2, x[j + 1] * f1 * f2, hi, lo);
        int ks, t, up;
        query_slot<KF>(lane * 4 + j, ks, t, up);
        uint32_t* at = reinterpret_cast<uint32_t*>(smem + L::q) + (ks * 32 + r * 4 + t) * 4 + 2 * up;
        at[0] = hi;
        at[1] = lo;
      }
    }
    __syncthreads();
    uint32_t aq[8][4];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      const uint4 w = *reinterpret_cast<const uint4*>(smem + L::q + (ks * 32 + lane) * 16);
      aq[ks][0] = w.x; aq[ks][1] = w.y; aq[ks][2] = w.z; aq[ks][3] = w.w;
    }
    const float post = q_post_s[g];

    float o[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    for (int i = warp; i < cnt; i += W) {
      const int s = used % S;
      if (!mbar_wait(bar0 + 8 * s, (used / S) & 1)) {      // gave up: everything this CTA produces from here on is NaN
        gave_up_s = 1;
        if (lane == 0) atomicExch(a.view.status, 3);
        break;
      }
      ++used;
      const uint8_t* st = smem + L::ring + (warp * S + s) * L::stage_bytes;
      const int p0 = cur.span.tile_at(cur.j + i) * kPagedTile;
      const bool full = p0 + kPagedTile <= cur.span.n && (p0 >= cur.span.lo || p0 + kPagedTile <= a.sinks);
      {   // norms: lane = position
        const bool seen = full || cur.span.sees(p0 + lane, a.sinks);
        const float vn = seen ? *reinterpret_cast<const float*>(st + L::vn_off + lane4) : 0.f;
        if (!dense(KF)) nrm[nrm_at] = *reinterpret_cast<const float*>(st + L::kn_off + lane4);
        nrm[32 + nrm_at] = lg2(fmaxf(vn, 1e-26f));
        nrm[64 + nrm_at] = vn;
        __syncwarp();
      }
      // ---------------- scores ----------------
      float sc[4][4];
#pragma unroll
      for (int ng = 0; ng < 4; ++ng) {
        sc[ng][0] = sc[ng][1] = sc[ng][2] = sc[ng][3] = 0.f;
        const uint8_t* row = st + L::k_off + (k_row0 + 2 * ng) * k_row_bytes(KF);
        if (dense(KF)) {
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const uint4 w = *reinterpret_cast<const uint4*>(row + t4 * 16 + it * 64);
            mma<KF == KF_BF16>(sc[ng], aq[2 * it], w.x, w.y);
            mma<KF == KF_BF16>(sc[ng], aq[2 * it + 1], w.z, w.w);
          }
        } else if (KF == KF_P4) {
          const uint4 w4 = *reinterpret_cast<const uint4*>(row + t4 * 16);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mma<false>(sc[ng], aq[2 * k], k_lut(byte_off(w[k], 0)), k_lut(byte_off(w[k], 1)));
            mma<false>(sc[ng], aq[2 * k + 1], k_lut(byte_off(w[k], 2)), k_lut(byte_off(w[k], 3)));
          }
        } else {
          const uint32_t* words = reinterpret_cast<const uint32_t*>(row);
          uint32_t w[3];
#pragma unroll
          for (int k = 0; k < 3; ++k) w[k] = words[3 * t4 + k];
          const uint32_t w12 = words[12] >> (6 * t4);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const int p = 2 * ks, p1 = 2 * ks + 1;
            mma<false>(sc[ng], aq[ks], k_lut(field_off(w[p / 5], p % 5)),
                       p1 < 15 ? k_lut(field_off(w[p1 < 15 ? p1 / 5 : 0], p1 % 5)) : k_lut(field_off(w12, 0)));
          }
        }
      }
      // ---------------- softmax: head g, positions 8 t4 + 2 ng + c in this tile's order ----------------
      const bool missing = (bad >> s) & 1u;
      float kn[8], lv[8], vn[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!dense(KF)) *reinterpret_cast<float4*>(kn + 4 * h) = *reinterpret_cast<const float4*>(nrm + 8 * t4 + 4 * h);
        *reinterpret_cast<float4*>(lv + 4 * h) = *reinterpret_cast<const float4*>(nrm + 32 + 8 * t4 + 4 * h);
        *reinterpret_cast<float4*>(vn + 4 * h) = *reinterpret_cast<const float4*>(nrm + 64 + 8 * t4 + 4 * h);
      }
      float s2[8], top = -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float raw = sc[k >> 1][k & 1] + sc[k >> 1][(k & 1) + 2];
        s2[k] = raw * (dense(KF) ? post : kn[k] * post);
      }
      if (!full || missing) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int pos = p0 + ((k & 1) ? v_row1 : v_row0) + (k & 6);
          if (missing) s2[k] = __int_as_float(0x7fc00000);
          else if (!cur.span.sees(pos, a.sinks)) s2[k] = -INFINITY;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, s2[k] + lv[k]);
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
      uint32_t pb[4];
#pragma unroll
      for (int ng = 0; ng < 4; ++ng) {
        const float e0 = paged_ex2(s2[2 * ng] - m_use), e1 = paged_ex2(s2[2 * ng + 1] - m_use);
        l_run += e0 + e1;
        const __half2 h = __floats2half2_rn(e0 * vn[2 * ng], e1 * vn[2 * ng + 1]);
        pb[ng] = *reinterpret_cast<const uint32_t*>(&h);
      }
      // ---------------- values ----------------
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t off[2][16];          // table offsets of the 16 slots, for the two position pairs of this k-step
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int ng = 2 * half + p;
          const uint8_t* r0p = st + L::v_off + (v_row0 + 2 * ng) * v_row_bytes(VB);
          const uint8_t* r1p = st + L::v_off + (v_row1 + 2 * ng) * v_row_bytes(VB);
          if (VB == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(r0p + 8 * g), y = *reinterpret_cast<const uint2*>(r1p + 8 * g);
            const uint32_t xs[2] = {x.x, x.y}, ys[2] = {y.x, y.y};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t ev = (xs[w] & 0x0F0F0F0Fu) | ((ys[w] << 4) & 0xF0F0F0F0u);     // even elements
              const uint32_t od = ((xs[w] >> 4) & 0x0F0F0F0Fu) | (ys[w] & 0xF0F0F0F0u);     // odd elements
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                off[p][8 * w + 2 * k] = byte_off(ev, k);
                off[p][8 * w + 2 * k + 1] = byte_off(od, k);
              }
            }
          } else {
            const uint32_t *xw = reinterpret_cast<const uint32_t*>(r0p), *yw = reinterpret_cast<const uint32_t*>(r1p);
            constexpr uint32_t kEven = 0707070707u;      // codes 0, 2, 4, 6, 8 of a word
            const int shb = 15 * (g & 1), shc = 3 * g;
            const uint32_t xa = xw[g], ya = yw[g], xb = xw[8 + (g >> 1)] >> shb, yb = yw[8 + (g >> 1)] >> shb,
                           xc = xw[12] >> shc, yc = yw[12] >> shc;
            const uint32_t ea = (xa & kEven) | ((ya << 3) & (kEven << 3)), oa = ((xa >> 3) & kEven) | (ya & (kEven << 3));
            const uint32_t eb = (xb & kEven) | ((yb << 3) & (kEven << 3)), ob = ((xb >> 3) & kEven) | (yb & (kEven << 3));
            const uint32_t ec = (xc & 7u) | ((yc & 7u) << 3);
#pragma unroll
            for (int k = 0; k < 5; ++k) {
              off[p][2 * k] = field_off(ea, k);
              off[p][2 * k + 1] = field_off(oa, k);
            }
            off[p][10] = field_off(eb, 0);
            off[p][11] = field_off(ob, 0);
            off[p][12] = field_off(eb, 1);
            off[p][13] = field_off(ob, 1);
            off[p][14] = field_off(eb, 2);
            off[p][15] = field_off(ec, 0);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t af[4] = {v_lut(off[0][2 * j]), v_lut(off[0][2 * j + 1]), v_lut(off[1][2 * j]), v_lut(off[1][2 * j + 1])};
          mma<false>(o[j], af, pb[2 * half], pb[2 * half + 1]);
        }
      }
      __syncwarp();            // every lane is done with the stage (and with the norms)
      fetch();
    }

    // ---------------- the warps meet ----------------
    // the upper half of the warps hands its state to the lower half, which hands rows to one warp per head
    constexpr int HW = L::xch_warps;
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (warp >= HW) {
      float* to = reinterpret_cast<float*>(smem + L::xch) + (warp - HW) * 34 * 32 + lane;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) to[(4 * j + c) * 32] = o[j][c];
      to[32 * 32] = m_run;
      to[33 * 32] = l_run;
    }
    __syncthreads();
    if (warp < HW && warp + HW < W) {
      const float* from = reinterpret_cast<const float*>(smem + L::xch) + warp * 34 * 32;
      const float m2 = from[32 * 32 + lane], l2 = from[33 * 32 + lane];
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
          o[j][c] = o[j][c] * ((c & 1) ? fa1 : fa0) + from[(4 * j + c) * 32 + lane] * ((c & 1) ? fb1 : fb0);
    }
    __syncthreads();
    if (warp < HW) {
      float* to = reinterpret_cast<float*>(smem + L::xch) + warp * kPagedRows * L::xch_row;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) to[(2 * t4 + (c & 1)) * L::xch_row + (2 * j + (c >> 1)) * 8 + g] = o[j][c];
      if (t4 == 0) {
        m_s[warp][g] = m_run;
        l_s[warp][g] = l_run;
      }
    }
    __syncthreads();
    for (int r = warp; r < nr; r += W) {
      float mx = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
      int at[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int gg, sl;
        value_slot<VB>(lane * 4 + j, gg, sl);
        at[j] = sl * 8 + gg;
      }
      for (int w = 0; w < HW; ++w) mx = fmaxf(mx, m_s[w][r]);
      for (int w = 0; w < HW; ++w) {
        const float fw = m_s[w][r] == -INFINITY ? 1.f : paged_ex2(m_s[w][r] - mx);
        l += l_s[w][r] * fw;
        const float* from = reinterpret_cast<const float*>(smem + L::xch) + (w * kPagedRows + r) * L::xch_row;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += from[at[j]] * fw;
      }
      if (gave_up_s) l = __int_as_float(0x7fc00000);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= tb.v_post;
      if (cnt == cur.span.tiles) {
        finish_row<4>(a, b, h0 + r, v, l, lane);
      } else {
        float* part = a.part + ((int64_t)(2 * cta + (cur.j == 0)) * kPagedRows + r) * (kDim + 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) part[lane * 4 + j] = v[j];
        if (lane == 0) {
          part[kDim] = mx;
          part[kDim + 1] = l;
        }
      }
    }
    __syncthreads();
    if (gave_up_s) {           // every warp leaves together; its copies still in flight land first (bounded)
      for (; used < issued; ++used) mbar_wait(bar0 + 8 * (used % S), (used / S) & 1);
      return;
    }
    run += cnt;
    if (cur.j + cnt == cur.span.tiles) cur.next_group(a);
  }
}

// ---- host side ---------------------------------------------------------------------------------------------
// 16-bit floats hold 11 bits; rounding the centroids directly would leave a fixed relative error of up to 2^-12 on each.
// A common factor beta in [1, 2) is searched so that every beta * c lands (almost) on a 16-bit value; 1 / beta is
// applied in 32 bits.  Kept by value (the codebook), not by address.
struct ScaledBook {
  int n;
  float key[16];
  uint16_t c16[16];
  float beta;
};
void scale_book(const float* c, int n, ScaledBook* out) {
  static std::mutex mu;
  static ScaledBook kept[8];
  static int n_kept = 0;
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < n_kept; ++i)
    if (kept[i].n == n && memcmp(kept[i].key, c, n * sizeof(float)) == 0) {
      *out = kept[i];
      return;
    }
  ScaledBook sb;
  memset(&sb, 0, sizeof(sb));
  sb.n = n;
  memcpy(sb.key, c, n * sizeof(float));
  double best = 1e30;
  sb.beta = 1.f;
  for (int step = 0; step < (1 << 16); ++step) {
    const float beta = 1.0f + step * (1.0f / 65536.0f);
    double worst = 0.0;
    for (int i = 0; i < n && worst < best; ++i) {
      if (c[i] == 0.f) continue;
      const double exact = (double)beta * (double)c[i];
      const double rel = fabs((double)__half2float(__float2half_rn((float)exact)) - exact) / fabs(exact);
      if (rel > worst) worst = rel;
    }
    if (worst < best) {
      best = worst;
      sb.beta = beta;
    }
  }
  for (int i = 0; i < n; ++i) sb.c16[i] = __half_as_ushort(__float2half_rn(sb.beta * c[i]));
  if (n_kept < 8) kept[n_kept++] = sb;
  *out = sb;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int KF, int VB, int W, int S>
int launch(PagedDecodeArgs& a, const MmaTables& tb, cudaStream_t st) {
  using L = Layout<KF, VB, W, S>;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_mma_kernel<KF, VB, W, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::total);
    if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  a.min_tiles = W;
  paged_mma_kernel<KF, VB, W, S><<<a.ctas, W * 32, L::total, st>>>(a, tb);
  const int rc = check_launch("tq_paged_decode");
  return rc ? rc : launch_paged_merge(a, kDim, st);
}

}  // namespace

// Queries in 32 bits ask for 32-bit weights and take the general kernel.
bool paged_mma_supported(const PagedDecodeArgs& a, int dim) {
  if (dim != kDim || a.q_dtype == TQ_F32 || a.v.format != TQ_KV_POLAR || (a.v.bits != 3 && a.v.bits != 4)) return false;
  if (!aligned16(a.v.data) || a.v.page_stride % 4 || a.v.head_stride % 4) return false;
  if (!aligned16(a.v.norms) || a.v.norm_page_stride % 4 || a.v.norm_head_stride % 4) return false;
  if (!aligned16(a.k.data)) return false;
  if (a.k.format == TQ_KV_DENSE) return a.k.dtype != TQ_F32 && a.k.page_stride % 8 == 0 && a.k.head_stride % 8 == 0;
  return (a.k.bits == 3 || a.k.bits == 4) && a.k.page_stride % 4 == 0 && a.k.head_stride % 4 == 0 && aligned16(a.k.norms) &&
         a.k.norm_page_stride % 4 == 0 && a.k.norm_head_stride % 4 == 0;
}

int launch_paged_mma(PagedDecodeArgs a, cudaStream_t st) {
  MmaTables tb;
  memset(&tb, 0, sizeof(tb));
  ScaledBook vb;
  scale_book(a.v.cent.v, 1 << a.v.bits, &vb);
  memcpy(tb.v_c16, vb.c16, sizeof(tb.v_c16));
  tb.v_post = 1.0f / vb.beta;
  tb.k_post = a.scale_log2;
  if (a.k.format == TQ_KV_POLAR) {
    ScaledBook kb;
    scale_book(a.k.cent.v, 1 << a.k.bits, &kb);
    memcpy(tb.k_c16, kb.c16, sizeof(tb.k_c16));
    tb.k_post = a.scale_log2 / ((float)kDim * kb.beta);
  }
  const bool v3 = a.v.bits == 3;
  if (a.k.format == TQ_KV_DENSE) {
    if (a.k.dtype == TQ_BF16) return v3 ? launch<KF_BF16, 3, 8, 2>(a, tb, st) : launch<KF_BF16, 4, 8, 2>(a, tb, st);
    return v3 ? launch<KF_F16, 3, 8, 2>(a, tb, st) : launch<KF_F16, 4, 8, 2>(a, tb, st);
  }
  if (a.k.bits == 3) return v3 ? launch<KF_P3, 3, 12, 4>(a, tb, st) : launch<KF_P3, 4, 12, 2>(a, tb, st);
  return v3 ? launch<KF_P4, 3, 12, 2>(a, tb, st) : launch<KF_P4, 4, 12, 2>(a, tb, st);
}

}  // namespace tq
