// tq_prefill_sdpa: causal (or full) scaled-dot-product attention over dense
// f16 / bf16 Q, K, V with head_dim 128 -- the prefill step that precedes the
// quantized decode path (the reference hands this to its array library's SDPA,
// turboquant_mlx/patch.py:37, on keys / values that update_and_fetch returned
// in the input dtype, cache.py:100-150).
//
// Blackwell-native formulation, one persistent CTA per SM over the items (128-query tile, query head, batch):
//   * Q, K and V tiles arrive by TMA (cp.async.bulk.tensor, 128-byte swizzle)
//     into shared memory; K tiles of 128 keys run through a ring of three, V tiles through another,
//     from item to item without a break.
//   * S = Q K^T and O += P V are tcgen05.mma (cta_group::1, kind::f16, M = N =
//     128, K = 16 per instruction) issued by one thread.  Three score buffers
//     and O live in tensor memory (128 lanes x 128 fp32 columns each); P goes
//     over the upper half of its scores as packed 16-bit pairs and is the A
//     operand of the second product straight from tensor memory.  V is consumed
//     as stored (keys x head_dim, head_dim contiguous) through an MN-major
//     descriptor.
//   * Two groups of four warps (one thread per query row each) take the K/V tiles
//     in turn, group 0 the even ones and group 1 the odd ones: tcgen05.ld the
//     scores, online softmax in the log2 domain, tcgen05.st of P.  The running
//     row maximum travels from tile to tile through a shared-memory mailbox; a
//     group's exponentials (special-function unit) run while the other group
//     loads, masks and reduces its scores, and the tensor core works meanwhile
//     on the products of the surrounding tiles.  O is rescaled lazily (only when
//     a row maximum grows by more than 2^8) by the group that sees the growth.
//   * A sliding window with sinks (tq_prefill_sdpa_window) is the same kernel over a shorter list of key tiles: those
//     of the sinks, then those from the window of the tile's first row to its diagonal.  Tiles that the window's
//     edge, the sinks' end or the diagonal crosses are masked per row; a row whose first tiles are masked whole keeps
//     m = -inf and its P at zero until it sees a key.  The full form is compiled without any of it.
// Measured: 32768 tokens causal, 28 / 4 heads, bf16: 1.33 PFLOP/s; 7000 tokens behind 1192 under a window of 2048 with 64
// sinks: 208 to 217 us = 0.95 to 0.99 PFLOP/s in short runs of replays, 248 us = 0.83 under sustained load (one CTA per
// item, without the overlap from item to item, the scores read twice and scalar arithmetic: 285 us against 208).  Of its
// products 15 % are on pairs that the window, the sinks' end or the diagonal hides.  Without the softmax's arithmetic it
// takes 187 us, without most of the products 113: what bounds it is the rate of 128 x 128 x 16 products, whose operands
// and the arriving tiles share the bandwidth of shared memory.
//   * Every wait is bounded; a wait that gives up sets the status word, the CTA
//     drains its copies, frees its tensor memory and returns.
#include <cuda.h>

#include <mutex>

#include "common.cuh"

namespace tq {
namespace {

constexpr int kD = 128;          // head_dim
constexpr int kBM = 128;         // queries per CTA
constexpr int kBN = 128;         // keys per tile
constexpr int kKStages = 3;      // K tiles run three ahead of the softmax
constexpr int kVStages = 3;
constexpr int kSBufs = 3;        // score buffers in tensor memory: tile j uses buffer j % 3
constexpr int kGroupThreads = 128;               // one softmax group: one thread per query row
constexpr int kSoftmaxThreads = 2 * kGroupThreads;
constexpr int kThreads = kSoftmaxThreads + 96;   // + TMA warps (Q and K; V) + MMA warp
constexpr int kKWarp = kSoftmaxThreads / 32, kVWarp = kKWarp + 1, kMmaWarp = kKWarp + 2;
constexpr uint32_t kTileBytes = kBM * kD * 2;    // 32 KiB: one 128 x 128 16-bit tile
constexpr uint32_t kHalfBytes = kTileBytes / 2;  // one 128-row x 64-element swizzle block
constexpr uint32_t kSpin = 1u << 20;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.0f;                 // log2 units: P stays <= 2^8
// Tensor memory (512 columns x 128 lanes): scores of tile j at columns 128 (j % 3); its P (16-bit
// pairs, 64 columns for 128 keys) goes over columns 64..127 of the same buffer; O at 384.
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColO = 384, kColPinS = 64;

struct Smem {                    // offsets from the 1024-byte aligned base
  static constexpr uint32_t q = 0;
  static constexpr uint32_t k0 = q + kTileBytes;                   // K stage s: k0 + s * kTileBytes
  static constexpr uint32_t v0 = k0 + kKStages * kTileBytes;       // V stage s: v0 + s * kTileBytes
  static constexpr uint32_t mbox = v0 + kVStages * kTileBytes;     // running row maxima [2][128], row sums handed over [2][128]
  static constexpr uint32_t bars = mbox + 4 * kBM * 4;
  static constexpr uint32_t tmem_slot = bars + 42 * 8;           // B_COUNT barriers
  static constexpr uint32_t total = tmem_slot + 16;
};
constexpr uint32_t kSmemBytes = Smem::total;          // dynamic memory begins at a multiple of 1024 (checked)
static_assert(kSmemBytes <= 227 * 1024, "shared memory of a CTA");

struct PrefillArgs {
  void* out;
  int64_t o_batch_stride, o_head_stride, o_row_stride;   // elements
  int seq_q, seq_k, n_rep, causal;
  int n_heads, heads_batches, items;     // query heads; heads * batch; work items = query tiles * heads * batch
  int window, sinks;             // windowed kernel: row i sees keys > i + off - window and keys < sinks
  float scale_log2;
  int* status;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait; gives up early once any wait of this launch has already failed.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const int* status) {
  for (uint32_t it = 0; it < kSpin; ++it) {
    if (status && (it & 1023u) == 1023u && *reinterpret_cast<const volatile int*>(status) != 0) return false;
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
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart.
// K-major operands ignore the leading offset; MN-major ones use it as the distance
// between 64-element blocks along M / N.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((leading_bytes >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The whole warp executes these with the same operands and one elected lane issues: operands that the compiler knows to
// be uniform go straight to the uniform registers the instruction reads.
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A operand from tensor memory (row i in lane i, 16-bit elements packed two per column)
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// two 32-bit floats at once, each rounded like the scalar operation
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return r;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Barrier slots (8 bytes each) inside Smem::bars.
enum : int { B_Q_FULL = 0, B_Q_EMPTY = 1, B_K_FULL = 2, B_K_EMPTY = 5, B_V_FULL = 8, B_V_EMPTY = 11, B_S_FULL = 14,
             B_P_FULL = 17, B_PV_DONE = 20 /* 2: by tile parity */, B_ALL_DONE = 22, B_O_FREE = 23,
             B_MBOX = 24 /* 8: [row group][tile parity] */, B_SUM = 32 /* 8: [row group][exchange parity] */,
             B_ITEM_DONE = 40 /* 2: by item parity */, B_COUNT = 42 };

// One work item: the 128-query tile of one head, and the key tiles it sees.
struct Item {
  int q0, head, batch;
  int first, sink_tiles, n;      // windowed: tiles 0 .. sink_tiles - 1, then from tile `first` on; n in all
  __device__ __forceinline__ int key0(int j) const { return (j < sink_tiles ? j : j - sink_tiles + first) * kBN; }
};
// The i-th item of this CTA; false behind the last.  Items are numbered by falling cost (latest queries first, then head by
// head) and dealt out round by round, every other round backwards, so that no CTA gets the longest of every round.
template <bool WINDOW>
__device__ __forceinline__ bool item_at(const PrefillArgs& a, int i, Item& it) {
  const int64_t at = (int64_t)i * gridDim.x + ((i & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  if (at >= a.items) return false;
  const int rank = (int)at / a.heads_batches, rest = (int)at - rank * a.heads_batches;
  const int off = a.seq_k - a.seq_q;                     // key index of query row 0's diagonal
  it.q0 = ((a.seq_q + kBM - 1) / kBM - 1 - rank) * kBM;
  it.batch = rest / a.n_heads;
  it.head = rest - it.batch * a.n_heads;
  // keys the item can see: [0, k_end), windowed without those between the sinks and the window of its first row
  const int k_end = a.causal ? min(a.seq_k, it.q0 + kBM + off) : a.seq_k;
  it.first = WINDOW ? (int)(max((int64_t)0, (int64_t)it.q0 + off - a.window + 1) / kBN) : 0;
  it.sink_tiles = WINDOW ? min((min(a.sinks, a.seq_k) + kBN - 1) / kBN, it.first) : 0;
  it.n = (k_end + kBN - 1) / kBN - it.first + it.sink_tiles;
  return true;
}

// Persistent: a CTA takes item after item, and the tiles of all its items form one sequence t = 0, 1, ... through the
// rings of K, V and score buffers.  The loads and score products of the next item run while this one ends.
template <bool WINDOW, bool BF>
__global__ void __launch_bounds__(kThreads, 1)
prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const PrefillArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023u) {           // the launcher has checked that this cannot be
    if (threadIdx.x == 0) atomicExch(a.status, 20);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);          // uniform, and known to be
  auto bar = [&](int i) { return sbase + Smem::bars + 8u * i; };
  auto wait = [&](uint32_t b, uint32_t parity) { return mbar_wait(b, parity, a.status); };

  if (tid == 0) {
    mbar_init(bar(B_Q_FULL), 1);
    mbar_init(bar(B_Q_EMPTY), 1);
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(bar(B_K_FULL + s), 1);
      mbar_init(bar(B_K_EMPTY + s), 1);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(bar(B_V_FULL + s), 1);
      mbar_init(bar(B_V_EMPTY + s), 1);
    }
    for (int i = 0; i < kSBufs; ++i) {
      mbar_init(bar(B_S_FULL + i), 1);
      mbar_init(bar(B_P_FULL + i), kGroupThreads);
    }
    mbar_init(bar(B_PV_DONE), 1);
    mbar_init(bar(B_PV_DONE + 1), 1);
    mbar_init(bar(B_ALL_DONE), 1);
    mbar_init(bar(B_ITEM_DONE), 1);
    mbar_init(bar(B_ITEM_DONE + 1), 1);
    mbar_init(bar(B_O_FREE), kGroupThreads);
    for (int i = 0; i < 8; ++i) mbar_init(bar(B_MBOX + i), 32);
    for (int i = 0; i < 8; ++i) mbar_init(bar(B_SUM + i), 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {   // this warp owns the tensor-memory allocation
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + Smem::tmem_slot),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + Smem::tmem_slot);
  const uint32_t tmem_o = tmem + kColO;

  if (warp == kKWarp) {
    // ------------------------------ TMA producer of Q and K ------------------------------
    if (lane == 0) {
      int items = 0, t = 0;            // loads issued: items' Q, tiles
      bool ok = true;
      Item it;
      for (; ok && item_at<WINDOW>(a, items, it); ) {
        if (items > 0 && !wait(bar(B_Q_EMPTY), (items - 1) & 1)) break;
        mbar_expect_tx(bar(B_Q_FULL), kTileBytes);
        tma_load_4d(sbase + Smem::q, &map_q, 0, it.q0, it.head, it.batch, bar(B_Q_FULL));
        tma_load_4d(sbase + Smem::q + kHalfBytes, &map_q, 64, it.q0, it.head, it.batch, bar(B_Q_FULL));
        ++items;
        const int kv_head = it.head / a.n_rep;
        for (int j = 0; j < it.n; ++j, ++t) {
          const int s = t % kKStages;
          if (t >= kKStages && !wait(bar(B_K_EMPTY + s), ((t / kKStages) - 1) & 1)) {
            ok = false;
            break;
          }
          const uint32_t dst = sbase + Smem::k0 + s * kTileBytes;
          mbar_expect_tx(bar(B_K_FULL + s), kTileBytes);
          tma_load_4d(dst, &map_k, 0, it.key0(j), kv_head, it.batch, bar(B_K_FULL + s));
          tma_load_4d(dst + kHalfBytes, &map_k, 64, it.key0(j), kv_head, it.batch, bar(B_K_FULL + s));
        }
      }
      if (!ok || item_at<WINDOW>(a, items, it)) atomicExch(a.status, 11);
      // drain: every copy this thread issued has landed before the CTA may exit
      if (items > 0) mbar_wait(bar(B_Q_FULL), (items - 1) & 1, nullptr);
      for (int j = max(0, t - kKStages); j < t; ++j) mbar_wait(bar(B_K_FULL + j % kKStages), (j / kKStages) & 1, nullptr);
    }
  } else if (warp == kVWarp) {
    // ------------------------------ TMA producer of V ------------------------------
    if (lane == 0) {
      int t = 0;
      bool ok = true;
      Item it;
      for (int i = 0; ok && item_at<WINDOW>(a, i, it); ++i) {
        const int kv_head = it.head / a.n_rep;
        for (int j = 0; j < it.n; ++j, ++t) {
          const int s = t % kVStages;
          if (t >= kVStages && !wait(bar(B_V_EMPTY + s), ((t / kVStages) - 1) & 1)) {
            ok = false;
            break;
          }
          const uint32_t dst = sbase + Smem::v0 + s * kTileBytes;
          mbar_expect_tx(bar(B_V_FULL + s), kTileBytes);
          tma_load_4d(dst, &map_v, 0, it.key0(j), kv_head, it.batch, bar(B_V_FULL + s));
          tma_load_4d(dst + kHalfBytes, &map_v, 64, it.key0(j), kv_head, it.batch, bar(B_V_FULL + s));
        }
      }
      if (!ok) atomicExch(a.status, 11);
      for (int j = max(0, t - kVStages); j < t; ++j) mbar_wait(bar(B_V_FULL + j % kVStages), (j / kVStages) & 1, nullptr);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------ MMA issuer ------------------------------
    {
      auto all_wait = [&](uint32_t b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(b, parity, a.status)) != 0; };
      const uint32_t fmt = BF ? 1u : 0u;
      // D f32, A / B f16 or bf16, M = 128, N = 128; B of the second product is MN-major
      const uint32_t idesc_qk = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kBN >> 3) << 17) |
                                ((uint32_t)(kBM >> 4) << 24);
      const uint32_t idesc_pv = idesc_qk | (1u << 16);
      bool ok = true;
      int fail = 0;
      // descriptors are built once; inside the loops only the 16-byte-unit address field moves
      uint64_t q_desc[kD / 16];
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)
        q_desc[kk] = smem_desc(sbase + Smem::q + (kk >> 2) * kHalfBytes + (kk & 3) * 32, 16);
      const uint64_t k_desc0 = smem_desc(sbase + Smem::k0, 16), v_desc0 = smem_desc(sbase + Smem::v0, kHalfBytes);
      Item qi, pi;                     // of the next score product and of the next value product
      int q_item = 0, qj = 0, qt = 0;
      bool q_more = item_at<WINDOW>(a, 0, qi);
      auto issue_qk = [&]() {          // S[t % 3] = Q K_t^T for the next tile t of the sequence
        const int s = qt % kKStages;
        if (qj == 0 && !all_wait(bar(B_Q_FULL), q_item & 1)) {
          fail = 12;
          return false;
        }
        if (!all_wait(bar(B_K_FULL + s), (qt / kKStages) & 1)) {
          fail = 13;
          return false;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t kd = k_desc0 + (uint64_t)(s * (kTileBytes >> 4));
        const uint32_t d_tmem = tmem + kColS + (qt % kSBufs) * kBN;
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)
          umma_f16(d_tmem, q_desc[kk], kd + (uint64_t)(((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4), idesc_qk, kk > 0);
        umma_commit(bar(B_K_EMPTY + s));
        umma_commit(bar(B_S_FULL + qt % kSBufs));
        ++qt;
        if (++qj == qi.n) {
          umma_commit(bar(B_Q_EMPTY));
          qj = 0;
          q_more = item_at<WINDOW>(a, ++q_item, qi);
        }
        return true;
      };
      for (int k = 0; k < kSBufs && q_more && ok; ++k) ok = issue_qk();
      int t = 0;
      for (int i = 0; ok && item_at<WINDOW>(a, i, pi); ++i)
        for (int j = 0; j < pi.n && ok; ++j, ++t) {
          const int s = t % kVStages;
          // O is free for the next item once the last one's has been read
          if (!all_wait(bar(B_V_FULL + s), (t / kVStages) & 1) || !all_wait(bar(B_P_FULL + t % kSBufs), (t / kSBufs) & 1) ||
              (j == 0 && i > 0 && !all_wait(bar(B_O_FREE), (i - 1) & 1))) {
            ok = false;
            fail = 14;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t vd = v_desc0 + (uint64_t)(s * (kTileBytes >> 4));
          const uint32_t p_tmem = tmem + kColS + (t % kSBufs) * kBN + kColPinS;
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk)    // 16 keys = 8 packed columns of P, 2 x 1024 bytes of V
            umma_f16_ts(tmem_o, p_tmem + kk * 8, vd + (uint64_t)(kk * (2048 >> 4)), idesc_pv,
                        (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(bar(B_V_EMPTY + s));
          umma_commit(bar(B_PV_DONE + (t & 1)));
          if (j == pi.n - 1) umma_commit(bar(B_ITEM_DONE + (i & 1)));
          // the scores three tiles on go over this tile's buffer: the tensor core runs its work in
          // issue order, so they follow the product that has just read P from it
          if (q_more) ok = issue_qk();
        }
      umma_commit(bar(B_ALL_DONE));
      if (fail && lane == 0) atomicExch(a.status, fail);
    }
  } else {
    // ---------------- softmax: group `who` takes the tiles t = who, who + 2, ...; one row per thread ----------------
    // An item's output is written by the group that has its last tile; the other has handed over its row sums and is at
    // the next item by then.  At an item's first tile a group still waits for the maximum of the tile in front (and
    // ignores it), so neither gets more than one tile ahead of what the other has still to read.  Whoever waits for a
    // phase of a barrier knows the phase in front of it to be over: a parity says no more than that.
    const int who = warp >> 2, rg = warp & 3;
    const int row = rg * 32 + lane;                        // = tensor-memory lane
    const uint32_t lane_base = (uint32_t)(rg * 32) << 16;
    float* mbox = reinterpret_cast<float*>(smem + Smem::mbox);    // [tile parity][row]
    float* sums = mbox + 2 * kBM;                                 // [exchange parity][row]
    const int off = a.seq_k - a.seq_q;
    Item it = {};
    int kmax = 0;                                                 // last key this row may see
    float m_mine = -INFINITY, l_mine = 0.f;                       // l_mine is relative to m_mine
    bool ok = true;
    // the 128 scores of a row: load, mask what the row may not see
    auto load_row = [&](int t, int k0, uint32_t (&v)[4][32]) {
      const uint32_t src = tmem + kColS + (t % kSBufs) * kBN + lane_base;
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(src + 32 * c, v[c]);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      const bool need_mask = (k0 + kBN - 1 > (a.causal ? it.q0 + off : a.seq_k - 1)) || (k0 + kBN > a.seq_k);
      if (WINDOW && k0 <= it.q0 + off + kBM - 1 - a.window && k0 + kBN > a.sinks) {
        // the window of the item's last row starts inside or behind this key tile, and not all of it are sinks:
        // columns in [slim, wlo) are hidden
        const int slim = a.sinks - k0, wlo = kmax - a.window + 1 - k0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= slim && c * 32 + i < wlo) v[c][i] = 0xff800000u;
      }
      if (need_mask) {
        const int klim = min(kmax, a.seq_k - 1) - k0;     // columns <= klim are visible
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i > klim) v[c][i] = 0xff800000u;   // -inf
      }
    };
    auto row_max = [&](const uint32_t (&v)[4][32]) {
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // four independent chains
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
      return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    };
    // exponentials of a half row -> 32 packed columns of P at `dst`; returns their sum
    auto half_exp = [&](const uint32_t (&v0)[32], const uint32_t (&v1)[32], float neg_m, uint32_t dst) {
      uint32_t pk[32];
      const float2 scale = make_float2(a.scale_log2, a.scale_log2), shift = make_float2(neg_m, neg_m);
      float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const uint32_t (&v)[32] = c ? v1 : v0;
          const float2 x = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scale, shift);
          const float2 y = fma2(make_float2(__uint_as_float(v[2 * i + 2]), __uint_as_float(v[2 * i + 3])), scale, shift);
          const float p0 = ex2(x.x), p1 = ex2(x.y), p2 = ex2(y.x), p3 = ex2(y.y);
          ls[(i >> 1) & 1] = add2(ls[(i >> 1) & 1], add2(make_float2(p0, p2), make_float2(p1, p3)));
          pk[c * 16 + i] = pack16<BF>(p0, p1);
          pk[c * 16 + i + 1] = pack16<BF>(p2, p3);
        }
      tmem_st32(dst, pk);
      return (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
    };
    int t0 = 0, xi = 0;              // first tile of the item in the sequence; items with an exchange so far
    for (int i = 0; ok && item_at<WINDOW>(a, i, it); ++i) {
      kmax = a.causal ? it.q0 + row + off : a.seq_k - 1;
      m_mine = -INFINITY;
      l_mine = 0.f;
      float m_oth = -INFINITY;       // reference of the other group's sum, at the item's last tile
      for (int j = (who ^ t0) & 1; j < it.n; j += 2) {
        const int t = t0 + j, k0 = it.key0(j);
        if (!__all_sync(0xffffffffu, wait(bar(B_S_FULL + t % kSBufs), (t / kSBufs) & 1))) {   // warp-uniform: aligned tcgen05 ops follow
          if (lane == 0) atomicExch(a.status, 15);
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t sv[4][32];
        load_row(t, k0, sv);
        const float mraw = row_max(sv);
        const float mt = mraw * a.scale_log2;              // scale > 0: order preserved
        // the running maximum after the previous tile comes from the other group
        if (t > 0) {
          if (!__all_sync(0xffffffffu, wait(bar(B_MBOX + rg * 2 + ((t - 1) & 1)), ((t - 1) >> 1) & 1))) {
            if (lane == 0) atomicExch(a.status, 18);
            ok = false;
            break;
          }
          if (j > 0) {
            m_oth = mbox[((t - 1) & 1) * kBM + row];
            if (m_oth != m_mine) {
              l_mine *= m_mine == -INFINITY ? 0.f : ex2(m_mine - m_oth);
              m_mine = m_oth;
            }
          }
        }
        // lazy rescale: the reference maximum only moves when a row maximum outgrows it by 2^8
        const bool grow = mt > m_mine + kRescale;
        float alpha = 1.f;
        if (grow) {
          alpha = m_mine == -INFINITY ? 0.f : ex2(m_mine - mt);
          m_mine = mt;
          l_mine *= alpha;
        }
        // publish before touching O: the other group only scales its P with it, and its product is
        // issued after this tile's, which waits for the arrival at the end of this iteration
        mbox[(t & 1) * kBM + row] = m_mine;
        mbar_arrive(bar(B_MBOX + rg * 2 + (t & 1)));
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
          // O must be complete up to the previous tile before it is rescaled
          if (!__all_sync(0xffffffffu, wait(bar(B_PV_DONE + ((t - 1) & 1)), ((t - 1) >> 1) & 1))) {
            if (lane == 0) atomicExch(a.status, 16);
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {      // rare path: kept small in registers
            uint32_t ov[16];
            tmem_ld16(tmem_o + lane_base + c * 16, ov);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 16; ++k) ov[k] = __float_as_uint(__uint_as_float(ov[k]) * alpha);
            tmem_st16(tmem_o + lane_base + c * 16, ov);
          }
        }
        // P over columns 64..127 of the scores, which are in registers by now
        const float neg_m = m_mine == -INFINITY ? 0.f : -m_mine;
        const uint32_t p_dst = tmem + kColS + (t % kSBufs) * kBN + lane_base + kColPinS;
        l_mine += half_exp(sv[2], sv[3], neg_m, p_dst + 32);          // keys 64..127 -> packed columns 32..63
        l_mine += half_exp(sv[0], sv[1], neg_m, p_dst);               // keys 0..63 -> packed columns 0..31
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(bar(B_P_FULL + t % kSBufs));
      }
      const int tl = t0 + it.n - 1, slot = xi & 1, turn = (xi >> 1) & 1;      // the item's last tile
      t0 += it.n;
      xi += it.n > 1;
      if (!ok) break;
      if ((tl & 1) != who) {
        if (it.n > 1) {
          sums[slot * kBM + row] = l_mine;
          mbar_arrive(bar(B_SUM + rg * 2 + slot));
        }
        continue;
      }
      if (!__all_sync(0xffffffffu, wait(bar(B_ITEM_DONE + (i & 1)), (i >> 1) & 1) &&
                                       (it.n == 1 || wait(bar(B_SUM + rg * 2 + slot), turn)))) {
        if (lane == 0) atomicExch(a.status, 17);
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float l_oth = m_oth == -INFINITY ? 0.f : sums[slot * kBM + row] * ex2(m_oth - m_mine);
      const float l_row = (m_mine == -INFINITY ? 0.f : l_mine) + l_oth;
      const float inv = l_row > 0.f ? 1.f / l_row : 0.f;
      uint32_t pk[kD / 2];
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t ov[32];
        tmem_ld32(tmem_o + lane_base + c * 32, ov);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int k = 0; k < 16; ++k)
          pk[c * 16 + k] = pack16<BF>(__uint_as_float(ov[2 * k]) * inv, __uint_as_float(ov[2 * k + 1]) * inv);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      mbar_arrive(bar(B_O_FREE));
      if (it.q0 + row < a.seq_q) {
        uint8_t* orow = reinterpret_cast<uint8_t*>(a.out) +
                        2 * (it.batch * a.o_batch_stride + it.head * a.o_head_stride + (int64_t)(it.q0 + row) * a.o_row_stride);
#pragma unroll
        for (int k = 0; k < kD / 8; ++k)
          *reinterpret_cast<uint4*>(orow + k * 16) = make_uint4(pk[4 * k], pk[4 * k + 1], pk[4 * k + 2], pk[4 * k + 3]);
      }
    }
    // nothing of the tensor core's is left when the CTA ends
    if (!__all_sync(0xffffffffu, wait(bar(B_ALL_DONE), 0)) && lane == 0) atomicExch(a.status, 17);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---- host side: tensor maps ------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// (batch, heads, rows, 128) tensor with arbitrary (16-byte multiple) strides; box = 64 elements x 128 rows
int make_map(CUtensorMap* map, const void* base, int bf16, int64_t batch, int64_t heads, int64_t rows,
             int64_t batch_stride, int64_t head_stride, int64_t row_stride) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return set_error(TQ_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[4] = {(cuuint64_t)kD, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
  // a stride of a size-1 dimension is never used for addressing: give the encoder the packed value
  if (heads == 1) head_stride = rows * row_stride;
  if (batch == 1) batch_stride = heads * head_stride;
  const cuuint64_t strides[3] = {(cuuint64_t)row_stride * 2, (cuuint64_t)head_stride * 2, (cuuint64_t)batch_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)kBM, 1, 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                        const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(TQ_ERR_LAUNCH, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return TQ_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace tq

static int prefill_sdpa(const void* q, const void* k, const void* v, void* out, int dtype, int batch, int n_q_heads,
                        int n_kv_heads, int64_t seq_q, int64_t seq_k, int dim, int64_t q_batch_stride, int64_t q_head_stride,
                        int64_t q_row_stride, int64_t k_batch_stride, int64_t k_head_stride, int64_t k_row_stride,
                        int64_t v_batch_stride, int64_t v_head_stride, int64_t v_row_stride, int64_t o_batch_stride,
                        int64_t o_head_stride, int64_t o_row_stride, float attn_scale, int causal, int64_t window,
                        int64_t sinks, int* status, void* stream) {
  using namespace tq;
  TQ_REQUIRE(window >= 0 && sinks >= 0, TQ_ERR_BAD_ARG, "window and sinks must not be negative");
  TQ_REQUIRE(window == 0 || causal, TQ_ERR_UNSUPPORTED, "a window needs causal attention");
  TQ_REQUIRE(window > 0 || sinks == 0, TQ_ERR_BAD_ARG, "sinks need a window");
  TQ_REQUIRE(q && k && v && out && status, TQ_ERR_BAD_ARG, "tq_prefill_sdpa: NULL pointer");
  TQ_REQUIRE(dim == kD, TQ_ERR_BAD_DIM, "tq_prefill_sdpa supports head_dim 128, got %d", dim);
  TQ_REQUIRE(dtype == TQ_F16 || dtype == TQ_BF16, TQ_ERR_UNSUPPORTED, "tq_prefill_sdpa takes f16 or bf16 tensors");
  TQ_REQUIRE(batch > 0 && n_q_heads > 0 && n_kv_heads > 0 && seq_q > 0 && seq_k > 0, TQ_ERR_BAD_ARG,
             "batch, head counts and sequence lengths must be positive");
  TQ_REQUIRE(n_q_heads % n_kv_heads == 0, TQ_ERR_HEAD_MISMATCH, "n_q_heads (%d) must equal n_kv_heads (%d) * n_rep",
             n_q_heads, n_kv_heads);
  TQ_REQUIRE(!causal || seq_k >= seq_q, TQ_ERR_BAD_ARG, "causal attention needs seq_k >= seq_q");
  TQ_REQUIRE(attn_scale > 0.f, TQ_ERR_BAD_ARG, "attn_scale must be positive, got %g", (double)attn_scale);
  TQ_REQUIRE(seq_k < (1ll << 31) - 256 && seq_q < (1ll << 31) - 256 && batch <= 65535 && n_q_heads <= 65535,
             TQ_ERR_BAD_ARG, "shape out of range");
  const int64_t strides[] = {q_batch_stride, q_head_stride, q_row_stride, k_batch_stride, k_head_stride, k_row_stride,
                             v_batch_stride, v_head_stride, v_row_stride, o_batch_stride, o_head_stride, o_row_stride};
  for (int64_t s : strides)
    TQ_REQUIRE(s >= 0 && s % 8 == 0, TQ_ERR_MISALIGNED, "tq_prefill_sdpa: strides must be multiples of 8 elements");
  TQ_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), TQ_ERR_MISALIGNED,
             "tq_prefill_sdpa: tensors must be 16-byte aligned");
  const int bf16 = dtype == TQ_BF16;
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = make_map(&mq, q, bf16, batch, n_q_heads, seq_q, q_batch_stride, q_head_stride, q_row_stride))) return rc;
  if ((rc = make_map(&mk, k, bf16, batch, n_kv_heads, seq_k, k_batch_stride, k_head_stride, k_row_stride))) return rc;
  if ((rc = make_map(&mv, v, bf16, batch, n_kv_heads, seq_k, v_batch_stride, v_head_stride, v_row_stride))) return rc;
  PrefillArgs a;
  a.out = out;
  a.o_batch_stride = o_batch_stride;
  a.o_head_stride = o_head_stride;
  a.o_row_stride = o_row_stride;
  a.seq_q = (int)seq_q;
  a.seq_k = (int)seq_k;
  a.n_rep = n_q_heads / n_kv_heads;
  a.causal = causal ? 1 : 0;
  a.scale_log2 = attn_scale * kLog2e;
  a.status = status;
  // a window that reaches the first key from every row hides nothing: the full form
  const bool windowed = window > 0 && window < seq_k;
  a.window = windowed ? (int)window : 0;
  a.sinks = windowed ? (int)(sinks < seq_k ? sinks : seq_k) : 0;
  auto kernel = windowed ? (bf16 ? prefill_kernel<true, true> : prefill_kernel<true, false>)
                         : (bf16 ? prefill_kernel<false, true> : prefill_kernel<false, false>);
  static bool ready_of[2][2][64] = {};         // per device: the attribute belongs to the device's context
  bool (&ready)[64] = ready_of[windowed][bf16];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && (dev < 0 || dev >= 64 || !ready[dev])) {
    int reserved = 0;
    err = cudaDeviceGetAttribute(&reserved, cudaDevAttrReservedSharedMemoryPerBlock, dev);
    TQ_REQUIRE(err != cudaSuccess || reserved % 1024 == 0, TQ_ERR_LAUNCH, "tq_prefill_sdpa: shared memory begins at %d", reserved);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (err == cudaSuccess && dev >= 0 && dev < 64) ready[dev] = true;
  }
  if (err != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "tq_prefill_sdpa: %s", cudaGetErrorString(err));
  const int64_t items = (seq_q + kBM - 1) / kBM * n_q_heads * batch;
  TQ_REQUIRE(items < (1ll << 31), TQ_ERR_BAD_ARG, "tq_prefill_sdpa: too many query tiles");
  a.n_heads = n_q_heads;
  a.heads_batches = n_q_heads * batch;
  a.items = (int)items;
  const unsigned grid = (unsigned)(items < num_sms() ? items : num_sms());
  kernel<<<grid, kThreads, kSmemBytes, static_cast<cudaStream_t>(stream)>>>(mq, mk, mv, a);
  return check_launch("tq_prefill_sdpa");
}

extern "C" int tq_prefill_sdpa(const void* q, const void* k, const void* v, void* out, int dtype, int batch,
                               int n_q_heads, int n_kv_heads, int64_t seq_q, int64_t seq_k, int dim,
                               int64_t q_batch_stride, int64_t q_head_stride, int64_t q_row_stride,
                               int64_t k_batch_stride, int64_t k_head_stride, int64_t k_row_stride,
                               int64_t v_batch_stride, int64_t v_head_stride, int64_t v_row_stride,
                               int64_t o_batch_stride, int64_t o_head_stride, int64_t o_row_stride,
                               float attn_scale, int causal, int* status, void* stream) {
  return prefill_sdpa(q, k, v, out, dtype, batch, n_q_heads, n_kv_heads, seq_q, seq_k, dim, q_batch_stride, q_head_stride,
                      q_row_stride, k_batch_stride, k_head_stride, k_row_stride, v_batch_stride, v_head_stride,
                      v_row_stride, o_batch_stride, o_head_stride, o_row_stride, attn_scale, causal, 0, 0, status, stream);
}

extern "C" int tq_prefill_sdpa_window(const tq_prefill_params* p) {
  using namespace tq;
  TQ_REQUIRE(p != nullptr, TQ_ERR_BAD_ARG, "params pointer is NULL");
  TQ_REQUIRE(p->struct_bytes == (int32_t)sizeof(tq_prefill_params), TQ_ERR_BAD_ARG,
             "struct_bytes %d does not match this library (%zu)", p->struct_bytes, sizeof(tq_prefill_params));
  return prefill_sdpa(p->q, p->k, p->v, p->out, p->dtype, p->batch, p->n_q_heads, p->n_kv_heads, p->seq_q, p->seq_k, p->dim,
                      p->q_strides[0], p->q_strides[1], p->q_strides[2], p->k_strides[0], p->k_strides[1], p->k_strides[2],
                      p->v_strides[0], p->v_strides[1], p->v_strides[2], p->o_strides[0], p->o_strides[1], p->o_strides[2],
                      p->attn_scale, p->causal, p->window, p->sinks, p->status, p->stream);
}
