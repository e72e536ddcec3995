// Paged caches: argument checks, the general decode kernel, page copies.
// (The tensor-core decode kernel is paged_mma.cu; insert and read-back are paged_rows.cu.)
#include <math.h>
#include <string.h>

#include "paged.cuh"
#include "paged_host.cuh"

namespace tq {

// One word per device: what a kernel of this file's family found wrong with its inputs since the last
// tq_paged_status (1: a page id outside the pool, 2: a position behind the page table, 3: a bounded wait gave up,
// 4: shared memory does not begin where the tensor-core decode kernel counts on it).
__device__ int g_paged_status = 0;

int paged_status_ptr(int** out) {
  static int* cached[64] = {nullptr};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error(TQ_ERR_LAUNCH, "no current CUDA device");
  if (!cached[dev]) {
    void* p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, g_paged_status);
    if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "cudaGetSymbolAddress: %s", cudaGetErrorString(e));
    cached[dev] = (int*)p;
  }
  *out = cached[dev];
  return TQ_OK;
}

namespace {

constexpr int kWarps = 16;
constexpr int kTile = 32;            // positions per tile of the general kernel: one per lane

// two 32-bit floats at once, each rounded like the scalar operation
__device__ __forceinline__ float2 fma2(float2 x, float y, float2 z) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %6};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(y), "f"(z.x), "f"(z.y));
  return r;
}

// ---- general decode -----------------------------------------------------------------------------------
// out = sum_p softmax(scale * q . k_p) v_p in 32 bits on the CUDA cores, for every head dimension, code width
// and key format; calls that qualify take the tensor-core kernel instead.  One pass over the rows with a
// running maximum m and sum l per (warp, query head):
//   scores : lane = position; a lane walks its key row (packed: centroid of every code) against the query
//            rows, which lie in shared memory element by element, eight heads side by side
//   values : lane = EPL consecutive elements; the 32 weights come back from shared memory
// The warps of a CTA take the tiles of its run in turn and meet in shared memory at the end of a group.
// (128 registers; at head_dim 256 it spills 296 bytes per thread.)
// Bound by its shared-memory reads (two vectors of queries or weights and a centroid per element), hidden by 16 warps:
// 32 sequences of 8192 tokens, 32 / 8 heads: 4-bit keys + 3-bit values 490 us (with 8 warps 1.7 times that), 16-bit keys
// 475 us.
template <int EPL>
__global__ void __launch_bounds__(kWarps * 32)
paged_decode_general_kernel(const PagedDecodeArgs a) {
  constexpr int DIM = EPL * 32;
  extern __shared__ float dyn_s[];
  float* q_s = dyn_s;                                   // [DIM][8]
  float* o_s = q_s + DIM * kPagedRows;                  // [kWarps][8][DIM]
  float* p_s = o_s + kWarps * kPagedRows * DIM;         // [kWarps][32][8]
  __shared__ int prefix[kPlanInts];
  __shared__ float kc_s[16], vc_s[16];
  __shared__ float m_s[kWarps][kPagedRows], l_s[kWarps][kPagedRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < 16) {
    kc_s[threadIdx.x] = a.k.cent.v[threadIdx.x];
    vc_s[threadIdx.x] = a.v.cent.v[threadIdx.x];
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  plan_costs(a, prefix, cost_early(a));
  zero_empty(a, DIM);
  const Plan plan = make_paged_plan(a, prefix);
  const int cta = blockIdx.x;
  if (plan.total == 0 || cta >= plan.ctas) return;
  Cursor cur, end;
  cur.seek_run(a, prefix, plan, cta, false, lane);
  end.seek_run(a, prefix, plan, cta, true, lane);
  const int kvpw = vals_per_word(a.k.bits), kpd = packed_words(DIM, a.k.bits);
  const int vvpw = vals_per_word(a.v.bits), vpd = packed_words(DIM, a.v.bits);
  const uint32_t kmask = (1u << a.k.bits) - 1u, vmask = (1u << a.v.bits) - 1u;
  // a lane's elements lie in one word or two neighbours
  const int v_word0 = lane * EPL / vvpw, v_word1 = (lane * EPL + EPL - 1) / vvpw;
  const bool polar = a.k.format == TQ_KV_POLAR;
  const int rg_per_head = a.groups / a.n_kv_heads;

  while (!cur.at(end)) {
    const int cnt = cur.count_to(end);
    const int b = cur.b, kvh = cur.group / rg_per_head, r0 = (cur.group % rg_per_head) * kPagedRows;
    const int nr = min(kPagedRows, a.n_rep - r0), h0 = kvh * a.n_rep + r0;
    if (warp < kPagedRows) {   // query rows of the group: warp r prepares row r (rotated for packed keys), stored [element][row]
      float x[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        x[j] = warp < nr ? load_elem(a.q, a.q_dtype, b * a.q_batch_stride + (h0 + warp) * a.q_head_stride + lane * EPL + j) : 0.f;
      if (polar) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] *= sign_at(a.k.signs, lane * EPL + j);
        warp_butterfly<EPL>(x, lane);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) q_s[(lane * EPL + j) * kPagedRows + warp] = x[j];
    }
    __syncthreads();
    float m[kPagedRows], l[kPagedRows];
    float2 o[kPagedRows / 2][EPL];                     // two heads side by side
#pragma unroll
    for (int r = 0; r < kPagedRows; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) o[r / 2][j] = make_float2(0.f, 0.f);
    }
    for (int i = warp; i < cnt; i += kWarps) {
      const int p0 = cur.span.tile_at(cur.j + i) * kTile, pos = p0 + lane;
      const int page = a.view.page_of(b, p0);
      const int row = p0 & ((1 << a.view.page_shift) - 1);
      if (page < 0 && lane == 0) atomicExch(a.view.status, 1);
      const bool seen = cur.span.sees(pos, a.sinks);
      float2 s2[kPagedRows / 2];
#pragma unroll
      for (int r = 0; r < kPagedRows / 2; ++r) s2[r] = make_float2(0.f, 0.f);
      if (page >= 0 && seen) {
        auto add = [&](int e, float c) {
          const float4 qa = *reinterpret_cast<const float4*>(q_s + e * kPagedRows);
          const float4 qb = *reinterpret_cast<const float4*>(q_s + e * kPagedRows + 4);
          s2[0] = fma2(make_float2(qa.x, qa.y), c, s2[0]);
          s2[1] = fma2(make_float2(qa.z, qa.w), c, s2[1]);
          s2[2] = fma2(make_float2(qb.x, qb.y), c, s2[2]);
          s2[3] = fma2(make_float2(qb.z, qb.w), c, s2[3]);
        };
        float post = a.scale_log2;
        if (polar) {
          const uint32_t* kr = reinterpret_cast<const uint32_t*>(a.k.data) + page * a.k.page_stride + kvh * a.k.head_stride +
                               (int64_t)(row + lane) * kpd;
          uint32_t next = __ldg(kr);
          for (int w = 0; w < kpd; ++w) {
            const uint32_t word = next;
            if (w + 1 < kpd) next = __ldg(kr + w + 1);
            for (int k = 0; k < kvpw && w * kvpw + k < DIM; ++k) add(w * kvpw + k, kc_s[(word >> (k * a.k.bits)) & kmask]);
          }
          post *= a.k.norms[page * a.k.norm_page_stride + kvh * a.k.norm_head_stride + row + lane] * (1.0f / DIM);
        } else {
          const int64_t off = page * a.k.page_stride + kvh * a.k.head_stride + (int64_t)(row + lane) * DIM;
          const uint16_t* kr = reinterpret_cast<const uint16_t*>(a.k.data) + off;
          if (a.k.dtype != TQ_F32 && ((uintptr_t)kr & 15) == 0) {
            for (int e = 0; e < DIM; e += 8) {
              const uint4 w4 = __ldg(reinterpret_cast<const uint4*>(kr + e));
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 f = a.k.dtype == TQ_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[k]))
                                                     : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
                add(e + 2 * k, f.x);
                add(e + 2 * k + 1, f.y);
              }
            }
          } else {
            for (int e = 0; e < DIM; ++e) add(e, load_elem(a.k.data, a.k.dtype, off + e));
          }
        }
#pragma unroll
        for (int r = 0; r < kPagedRows / 2; ++r) s2[r] = make_float2(s2[r].x * post, s2[r].y * post);
      }
      const float vn = page >= 0 && seen
                           ? a.v.norms[page * a.v.norm_page_stride + kvh * a.v.norm_head_stride + row + lane] : 0.f;
      float* pw = p_s + warp * 32 * kPagedRows;
      __syncwarp();
#pragma unroll
      for (int r = 0; r < kPagedRows; ++r) {
        // a page outside the pool: the sequence's output becomes NaN instead of a plausible number
        const float sr = page < 0 ? __int_as_float(0x7fc00000) : seen ? (r & 1 ? s2[r / 2].y : s2[r / 2].x) : -INFINITY;
        const float mn = fmaxf(m[r], warp_max(sr));       // fmaxf passes over NaN: the sum below carries it
        const float alpha = mn == -INFINITY ? 1.f : paged_ex2(m[r] - mn);
        const float p = mn == -INFINITY ? (page < 0 ? sr : 0.f) : paged_ex2(sr - mn);
        m[r] = mn;
        l[r] = l[r] * alpha + warp_sum(p);
        pw[lane * kPagedRows + r] = p * vn;
#pragma unroll
        for (int j = 0; j < EPL; ++j) (r & 1 ? o[r / 2][j].y : o[r / 2][j].x) *= alpha;
      }
      __syncwarp();
      if (page >= 0) {
        const uint32_t* vr = reinterpret_cast<const uint32_t*>(a.v.data) + page * a.v.page_stride + kvh * a.v.head_stride +
                             (int64_t)row * vpd;
        // hidden positions have weight 0; four rows' words are on their way at a time
#pragma unroll 1
        for (int k0 = 0; k0 < kTile; k0 += 4) {
          uint32_t w0[4], w1[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            w0[k] = __ldg(vr + (k0 + k) * vpd + v_word0);
            w1[k] = __ldg(vr + (k0 + k) * vpd + v_word1);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 wa = *reinterpret_cast<const float4*>(pw + (k0 + k) * kPagedRows);
            const float4 wb = *reinterpret_cast<const float4*>(pw + (k0 + k) * kPagedRows + 4);
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
              const int e = lane * EPL + j, at = e / vvpw;
              const float c = vc_s[((at == v_word0 ? w0[k] : w1[k]) >> ((e - at * vvpw) * a.v.bits)) & vmask];
              o[0][j] = fma2(make_float2(wa.x, wa.y), c, o[0][j]);
              o[1][j] = fma2(make_float2(wa.z, wa.w), c, o[1][j]);
              o[2][j] = fma2(make_float2(wb.x, wb.y), c, o[2][j]);
              o[3][j] = fma2(make_float2(wb.z, wb.w), c, o[3][j]);
            }
          }
        }
      }
    }
    // the warps meet: warp r joins row r
#pragma unroll
    for (int r = 0; r < kPagedRows; ++r) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) o_s[(warp * kPagedRows + r) * DIM + lane * EPL + j] = r & 1 ? o[r / 2][j].y : o[r / 2][j].x;
      if (lane == 0) {
        m_s[warp][r] = m[r];
        l_s[warp][r] = l[r];
      }
    }
    __syncthreads();
    if (warp < nr) {
      float mx = -INFINITY, ls = 0.f, v[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) v[j] = 0.f;
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, m_s[w][warp]);
      for (int w = 0; w < kWarps; ++w) {
        const float f = m_s[w][warp] == -INFINITY ? (l_s[w][warp] == 0.f ? 0.f : 1.f) : paged_ex2(m_s[w][warp] - mx);
        ls += l_s[w][warp] * f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) v[j] += o_s[(w * kPagedRows + warp) * DIM + lane * EPL + j] * f;
      }
      if (cnt == cur.span.tiles) {
        finish_row<EPL>(a, b, h0 + warp, v, ls, lane);
      } else {
        float* part = part_of(a, cta, cur.j == 0 ? cta : -1, warp, DIM);
#pragma unroll
        for (int j = 0; j < EPL; ++j) part[lane * EPL + j] = v[j];
        if (lane == 0) {
          part[DIM] = mx;
          part[DIM + 1] = ls;
        }
      }
    }
    __syncthreads();
    if (cnt != cur.span.tiles) {
      // where the group begins in the plan's numbering: from the end of this run, or from its beginning
      const int64_t first = cur.j == 0 ? plan.begin(cta + 1) - end.j : plan.begin(cta) - cur.j;
      const int c0 = plan.owner(first), c1 = plan.owner(first + cur.span.tiles - 1);
      __shared__ int last_s;
      if (threadIdx.x == 0) last_s = last_part(a, c0, c1);
      __syncthreads();
      if (last_s && warp < nr) join_row<EPL>(a, c0, c1, warp, b, h0 + warp, lane);
      __syncthreads();
    }
    if (cur.j + cnt < cur.span.tiles) break;
    cur.next_group(a);
  }
}

template <int EPL>
int launch_general(const PagedDecodeArgs& a, cudaStream_t st) {
  constexpr int DIM = EPL * 32;
  constexpr int smem = (DIM * kPagedRows + kWarps * kPagedRows * DIM + kWarps * 32 * kPagedRows) * (int)sizeof(float);
  int dev = 0;
  cudaGetDevice(&dev);
  static bool done[64] = {false};
  if (dev >= 0 && dev < 64 && !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_decode_general_kernel<EPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
  }
  return launch_dependent("tq_paged_decode (general)", paged_decode_general_kernel<EPL>, dim3(a.ctas), kWarps * 32, smem, st, a);
}

// ---- page copies -------------------------------------------------------------------------------------------
// HBM-bound, four 16-byte words per thread in flight: 1500 pages of 8 tensors, 381 MB read and written, 63 us = 6.05 TB/s
// (0.93 of the copy peak).
constexpr int kCopyPools = 128;          // pools per launch: their pointers travel as kernel parameters
constexpr int kCopyUnit = 1024;          // 16-byte words a block moves per step: 4 per thread, all in flight
struct CopyArgs {
  uint4* pool[kCopyPools];
  uint32_t page16[kCopyPools];           // 16-byte words of a page
  const int* src;
  const int* dst;
  int n_pairs;
  int n_pages;
  int* status;
};

__global__ void __launch_bounds__(256)
copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  uint4* pool = a.pool[blockIdx.y];
  const uint32_t words = a.page16[blockIdx.y], per = (words + kCopyUnit - 1) / kCopyUnit;
  const int64_t units = (int64_t)a.n_pairs * per;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int pair = (int)(u / per);
    const uint32_t w0 = (uint32_t)(u - (int64_t)pair * per) * kCopyUnit + threadIdx.x;
    const int s = __ldg(a.src + pair), d = __ldg(a.dst + pair);
    if (s < 0 || s >= a.n_pages || d < 0 || d >= a.n_pages) {
      if (threadIdx.x == 0) atomicExch(a.status, 1);
      continue;
    }
    const uint4* from = pool + (int64_t)s * words;
    uint4* to = pool + (int64_t)d * words;
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w0 + k * 256 < words) v[k] = from[w0 + k * 256];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w0 + k * 256 < words) to[w0 + k * 256] = v[k];
  }
}

}  // namespace

// ---- host-side checks shared by the entry points ------------------------------------------------------------
int check_paged_params(const tq_paged_params* p) {
  TQ_REQUIRE(p != nullptr, TQ_ERR_BAD_ARG, "params pointer is NULL");
  TQ_REQUIRE(p->struct_bytes == (int32_t)sizeof(tq_paged_params), TQ_ERR_BAD_ARG,
             "struct_bytes %d does not match this library (%zu)", p->struct_bytes, sizeof(tq_paged_params));
  TQ_REQUIRE(p->dim >= 32 && p->dim <= 256 && !(p->dim & (p->dim - 1)), TQ_ERR_BAD_DIM,
             "dim must be a power of 2 in [32, 256], got %d", p->dim);
  TQ_REQUIRE(p->page_size >= kMinPage && p->page_size <= (1 << 20) && !(p->page_size & (p->page_size - 1)), TQ_ERR_BAD_ARG,
             "page_size must be a power of 2, at least %d, got %d", kMinPage, p->page_size);
  TQ_REQUIRE(p->batch > 0 && p->batch <= (1 << 20) && p->n_kv_heads > 0 && p->n_kv_heads <= (1 << 16), TQ_ERR_BAD_ARG,
             "batch and n_kv_heads must be positive (at most 2^20 and 2^16)");
  TQ_REQUIRE(p->n_pages > 0 && p->n_pages < (1ll << 31), TQ_ERR_BAD_ARG, "n_pages must be in [1, 2^31), got %lld",
             (long long)p->n_pages);
  TQ_REQUIRE(p->page_table && p->seq_lens && p->table_width > 0, TQ_ERR_BAD_ARG, "page_table and seq_lens are required");
  // plans number the tiles of a batch in 32 bits
  TQ_REQUIRE((int64_t)p->batch * ((int64_t)p->table_width * p->page_size / kMinPage + 64) < (1ll << 31), TQ_ERR_BAD_ARG,
             "batch * table_width * page_size is too large");
  return TQ_OK;
}

int fill_paged_half(const tq_paged_half* h, int dim, const char* what, bool encode, bool need_signs, PagedHalf* out,
                    Table16* thresholds) {
  memset(out, 0, sizeof(*out));
  TQ_REQUIRE(h->data, TQ_ERR_BAD_ARG, "%s: NULL data pointer", what);
  TQ_REQUIRE(h->format == TQ_KV_POLAR || h->format == TQ_KV_DENSE, TQ_ERR_UNSUPPORTED, "%s: pages hold polar or dense rows",
             what);
  out->format = h->format;
  out->bits = 4;
  out->dtype = h->dtype;
  out->data = h->data;
  out->norms = h->norms;
  out->page_stride = h->page_stride;
  out->head_stride = h->head_stride;
  out->norm_page_stride = h->norm_page_stride;
  out->norm_head_stride = h->norm_head_stride;
  TQ_REQUIRE(h->page_stride >= 0 && h->head_stride >= 0 && h->norm_page_stride >= 0 && h->norm_head_stride >= 0,
             TQ_ERR_BAD_ARG, "%s: negative stride", what);
  if (h->format == TQ_KV_DENSE) {
    TQ_REQUIRE(h->dtype >= TQ_F32 && h->dtype <= TQ_BF16, TQ_ERR_BAD_ARG, "%s: bad dtype", what);
    return TQ_OK;
  }
  TQ_REQUIRE(h->bits >= 1 && h->bits <= 4, TQ_ERR_BAD_BITS, "Unsupported bit width: %d. Use 1-4.", h->bits);
  TQ_REQUIRE(h->norms, TQ_ERR_BAD_ARG, "%s: packed pages need norms", what);
  out->bits = h->bits;
  if (h->centroids_host)
    for (int i = 0; i < (1 << h->bits); ++i) out->cent.v[i] = h->centroids_host[i];
  else
    TQ_REQUIRE(encode, TQ_ERR_BAD_ARG, "%s: packed pages need centroids", what);
  if (need_signs) {
    const int rc = make_sign_mask(h->signs_host, dim, &out->signs);
    if (rc) return rc;
  }
  if (encode) {
    TQ_REQUIRE(h->boundaries_host, TQ_ERR_BAD_ARG, "%s: inserting packed rows needs boundaries", what);
    make_raw_thresholds(h->boundaries_host, (1 << h->bits) - 1, dim, thresholds);
  }
  return TQ_OK;
}

int fill_page_view(const tq_paged_params* p, PageView* v) {
  v->table = p->page_table;
  v->table_stride = p->table_stride;
  v->table_width = p->table_width;
  v->page_shift = 0;
  while ((1 << v->page_shift) < p->page_size) ++v->page_shift;
  v->n_pages = p->n_pages;
  return paged_status_ptr(&v->status);
}

}  // namespace tq

using namespace tq;

extern "C" int64_t tq_paged_decode_workspace_bytes(int dim) {
  return kMaxCtas * (int64_t)sizeof(int) + (int64_t)2 * num_sms() * kPagedRows * (dim + 4) * (int64_t)sizeof(float);
}

extern "C" int tq_paged_decode(const tq_paged_params* p) {
  int rc = check_paged_params(p);
  if (rc) return rc;
  TQ_REQUIRE(p->n_q_heads > 0 && p->n_q_heads % p->n_kv_heads == 0, TQ_ERR_HEAD_MISMATCH,
             "n_q_heads (%d) must equal n_kv_heads (%d) * n_rep", p->n_q_heads, p->n_kv_heads);
  TQ_REQUIRE(p->q && p->out && p->q_dtype >= TQ_F32 && p->q_dtype <= TQ_BF16 && p->out_dtype >= TQ_F32 &&
                 p->out_dtype <= TQ_BF16,
             TQ_ERR_BAD_ARG, "q and out must be given, as float32, float16 or bfloat16");
  TQ_REQUIRE(p->window >= 0 && p->sinks >= 0, TQ_ERR_BAD_ARG, "window and sinks must not be negative");
  TQ_REQUIRE(p->window > 0 || p->sinks == 0, TQ_ERR_BAD_ARG, "sinks need a window");
  TQ_REQUIRE(p->attn_scale == p->attn_scale && fabsf(p->attn_scale) < INFINITY, TQ_ERR_BAD_ARG, "attn_scale must be finite");
  TQ_REQUIRE(p->v.format == TQ_KV_POLAR, TQ_ERR_UNSUPPORTED, "decode reads packed values");
  const int64_t need = tq_paged_decode_workspace_bytes(p->dim);
  TQ_REQUIRE(p->workspace && p->workspace_bytes >= need, TQ_ERR_WORKSPACE, "workspace of %lld bytes required, got %lld",
             (long long)need, (long long)p->workspace_bytes);
  TQ_REQUIRE(((uintptr_t)p->workspace & 15) == 0, TQ_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  PagedDecodeArgs a;
  memset(&a, 0, sizeof(a));
  if ((rc = fill_paged_half(&p->k, p->dim, "keys", false, p->k.format == TQ_KV_POLAR, &a.k, nullptr))) return rc;
  if ((rc = fill_paged_half(&p->v, p->dim, "values", false, true, &a.v, nullptr))) return rc;
  if ((rc = fill_page_view(p, &a.view))) return rc;
  a.batch = p->batch;
  a.n_q_heads = p->n_q_heads;
  a.n_kv_heads = p->n_kv_heads;
  a.n_rep = p->n_q_heads / p->n_kv_heads;
  const int64_t groups = (int64_t)p->n_kv_heads * ((a.n_rep + kPagedRows - 1) / kPagedRows);
  TQ_REQUIRE(groups <= (1 << 20), TQ_ERR_BAD_ARG, "too many query heads");
  a.groups = (int)groups;
  a.lens = p->seq_lens;
  a.window = p->window;
  a.sinks = p->sinks;
  a.q = p->q;
  a.q_dtype = p->q_dtype;
  a.q_batch_stride = p->q_batch_stride;
  a.q_head_stride = p->q_head_stride;
  a.out = p->out;
  a.out_dtype = p->out_dtype;
  a.out_batch_stride = p->out_batch_stride;
  a.out_head_stride = p->out_head_stride;
  a.scale_log2 = p->attn_scale * kPagedLog2e;
  a.counters = (int*)p->workspace;
  a.part = (float*)(a.counters + kMaxCtas);
  a.ctas = num_sms() < kMaxCtas ? num_sms() : kMaxCtas;
  cudaStream_t st = (cudaStream_t)p->stream;
  // 32 sequences of 8192 tokens, 4 + 3 bits: 93 us on tensor cores, 490 us in 32 bits
  if (paged_mma_supported(a, p->dim)) {
    bool taken = false;
    rc = launch_paged_mma(a, st, &taken);
    if (taken) return rc;
  }
  a.tile_shift = 5;
  a.min_tiles = kWarps;
  a.group_cost = 2;
  switch (p->dim) {
    case 32: return launch_general<1>(a, st);
    case 64: return launch_general<2>(a, st);
    case 128: return launch_general<4>(a, st);
    default: return launch_general<8>(a, st);
  }
}

extern "C" int tq_copy_pages(void* const* pools, const int64_t* page_bytes, int n_pools, int64_t n_pages, const int32_t* src,
                             const int32_t* dst, int64_t n_pairs, void* stream) {
  TQ_REQUIRE(n_pools >= 0 && n_pairs >= 0 && n_pairs < (1ll << 31), TQ_ERR_BAD_ARG, "bad pool or pair count");
  if (n_pools == 0 || n_pairs == 0) return TQ_OK;
  TQ_REQUIRE(pools && page_bytes && src && dst, TQ_ERR_BAD_ARG, "NULL pointer");
  TQ_REQUIRE(n_pages > 0 && n_pages < (1ll << 31), TQ_ERR_BAD_ARG, "n_pages must be in [1, 2^31), got %lld", (long long)n_pages);
  CopyArgs a;
  a.src = src;
  a.dst = dst;
  a.n_pairs = (int)n_pairs;
  a.n_pages = (int)n_pages;
  for (int i = 0; i < n_pools; ++i)
    TQ_REQUIRE(pools[i] && ((uintptr_t)pools[i] & 15) == 0 && page_bytes[i] > 0 && page_bytes[i] % 16 == 0 &&
                   page_bytes[i] < (1ll << 34),
               TQ_ERR_MISALIGNED, "pool %d: pages must be 16-byte aligned and a multiple of 16 bytes", i);
  int rc = paged_status_ptr(&a.status);
  if (rc) return rc;
  for (int i0 = 0; i0 < n_pools; i0 += kCopyPools) {
    const int n = n_pools - i0 < kCopyPools ? n_pools - i0 : kCopyPools;
    int64_t units = 0;
    for (int i = 0; i < n; ++i) {
      a.pool[i] = (uint4*)pools[i0 + i];
      a.page16[i] = (uint32_t)(page_bytes[i0 + i] / 16);
      const int64_t u = n_pairs * ((a.page16[i] + kCopyUnit - 1) / kCopyUnit);
      units = u > units ? u : units;
    }
    const int64_t cap = (int64_t)num_sms() * 8;
    copy_pages_kernel<<<dim3((unsigned)(units < cap ? units : cap), n), 256, 0, (cudaStream_t)stream>>>(a);
    if ((rc = check_launch("tq_copy_pages"))) return rc;
  }
  return TQ_OK;
}

extern "C" int tq_paged_status(int* status, void* stream) {
  TQ_REQUIRE(status, TQ_ERR_BAD_ARG, "NULL pointer");
  int* word = nullptr;
  int rc = paged_status_ptr(&word);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cudaMemcpyAsync(status, word, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *status) e = cudaMemsetAsync(word, 0, sizeof(int), st);
  if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "tq_paged_status: %s", cudaGetErrorString(e));
  return TQ_OK;
}
