// Paged caches: quantize-on-insert of new rows into pages, and pages read back as dense rows.
#include <math.h>
#include <string.h>

#include "paged.cuh"
#include "paged_host.cuh"
#include "quantize_row.cuh"

namespace tq {
namespace {

constexpr int kWarps = 8;

struct AppendHalf {
  PagedHalf h;
  Table16 thr;                       // thresholds on the raw butterfly output
  const void* x;                     // new rows (batch, heads, tokens, dim), rows contiguous
  int x_dtype;
  int64_t batch_stride, head_stride, token_stride;
};
struct AppendArgs {
  AppendHalf half[2];                // keys, values
  PageView view;
  int batch, heads, tokens;
  const int* starts;                 // position of a sequence's first new token
  const int* counts;                 // new tokens per sequence (at most `tokens`), NULL: all
};

// Where new token t of sequence b goes: its page, or -1 when there is nothing to store.
__device__ __forceinline__ int append_place(const AppendArgs& a, int b, int t, int* row) {
  const int count = a.counts ? __ldg(a.counts + b) : a.tokens;
  if (t >= count) return -1;
  const int64_t pos = (int64_t)__ldg(a.starts + b) + t;
  if (pos < 0 || pos >= a.view.capacity()) {
    atomicExch(a.view.status, 2);
    return -1;
  }
  const int page = a.view.page_of(b, (int)pos);
  if (page < 0) atomicExch(a.view.status, 1);
  *row = (int)pos & ((1 << a.view.page_shift) - 1);
  return page;
}

// ---- insert, one warp per row: every head dimension, code width and input type --------------------------------
template <int EPL, int BITS>
__device__ __forceinline__ void encode_row(const AppendHalf& s, const float (&x)[EPL], uint8_t* idx_s, int page, int head,
                                           int row, int lane) {
  uint32_t* words = reinterpret_cast<uint32_t*>(s.h.data) + page * s.h.page_stride + head * s.h.head_stride +
                    (int64_t)row * packed_words(EPL * 32, BITS);
  quantize_row_warp<EPL, BITS>(x, s.h.signs, s.thr, idx_s, words,
                               s.h.norms + page * s.h.norm_page_stride + head * s.h.norm_head_stride + row, lane);
}

template <int EPL>
__global__ void __launch_bounds__(kWarps * 32)
paged_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int DIM = EPL * 32;
  __shared__ uint8_t idx_s[kWarps][DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const AppendHalf& s = a.half[blockIdx.y];
  const int64_t rows = (int64_t)a.batch * a.heads * a.tokens;
  for (int64_t v = (int64_t)blockIdx.x * kWarps + warp; v < rows; v += (int64_t)gridDim.x * kWarps) {
    const int64_t bh = v / a.tokens;
    const int t = (int)(v - bh * a.tokens), b = (int)(bh / a.heads), head = (int)(bh - (int64_t)b * a.heads);
    int row = 0;
    const int page = append_place(a, b, t, &row);
    if (page < 0) continue;
    const int64_t off = b * s.batch_stride + head * s.head_stride + t * s.token_stride + lane * EPL;
    if (s.h.format == TQ_KV_DENSE) {           // keys kept as they are, in their own type
      const int64_t to = page * s.h.page_stride + head * s.h.head_stride + (int64_t)row * DIM + lane * EPL;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        if (s.x_dtype == TQ_F32) reinterpret_cast<float*>(s.h.data)[to + j] = reinterpret_cast<const float*>(s.x)[off + j];
        else reinterpret_cast<uint16_t*>(s.h.data)[to + j] = reinterpret_cast<const uint16_t*>(s.x)[off + j];
      }
      continue;
    }
    float x[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) x[j] = load_elem(s.x, s.x_dtype, off + j);
    switch (s.h.bits) {
      case 1: encode_row<EPL, 1>(s, x, idx_s[warp], page, head, row, lane); break;
      case 2: encode_row<EPL, 2>(s, x, idx_s[warp], page, head, row, lane); break;
      case 3: encode_row<EPL, 3>(s, x, idx_s[warp], page, head, row, lane); break;
      default: encode_row<EPL, 4>(s, x, idx_s[warp], page, head, row, lane); break;
    }
  }
}

template <int EPL>
int launch_append(const AppendArgs& a, cudaStream_t st) {
  const int64_t blocks = ((int64_t)a.batch * a.heads * a.tokens + kWarps - 1) / kWarps;
  const int64_t cap = (int64_t)num_sms() * 8;
  paged_append_kernel<EPL><<<dim3((unsigned)(blocks < cap ? blocks : cap), 2), kWarps * 32, 0, st>>>(a);
  return check_launch("tq_paged_append");
}

// ---- read back -------------------------------------------------------------------------------------------------
struct ReadArgs {
  PagedHalf h;
  PageView view;
  int batch, heads;
  int64_t length;
  const int* lens;
  void* out;                         // (batch, heads, length, dim), contiguous
  int out_dtype;
  float s;                           // float32(1 / sqrt(dim)); h.cent holds centroid * s
};

// One warp per row, lane = EPL consecutive elements: ((butterfly(c * s) * s) * sign) * norm in the order of the
// contiguous decoder, so both give the same bits.  Rows behind a sequence are zero.
template <int EPL>
__global__ void __launch_bounds__(kWarps * 32)
paged_read_kernel(const ReadArgs a) {
  constexpr int DIM = EPL * 32;
  __shared__ float cs_s[16];
  if (threadIdx.x < 16) cs_s[threadIdx.x] = a.h.cent.v[threadIdx.x];
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int vpw = vals_per_word(a.h.bits), pd = packed_words(DIM, a.h.bits);
  const uint32_t mask = (1u << a.h.bits) - 1u;
  const int64_t rows = (int64_t)a.batch * a.heads * a.length;
  for (int64_t v = (int64_t)blockIdx.x * kWarps + warp; v < rows; v += (int64_t)gridDim.x * kWarps) {
    const int64_t bh = v / a.length;
    const int pos = (int)(v - bh * a.length), b = (int)(bh / a.heads), head = (int)(bh - (int64_t)b * a.heads);
    const int64_t to = v * DIM + lane * EPL;
    const int n = min(__ldg(a.lens + b), a.view.capacity());
    const int page = pos < n ? a.view.page_of(b, pos) : -1;
    if (pos < n && page < 0 && lane == 0) atomicExch(a.view.status, 1);
    if (page < 0) {                  // behind the sequence: zero; a page outside the pool: NaN
      const float x = pos < n ? __int_as_float(0x7fc00000) : 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) store_elem(a.out, a.out_dtype, to + j, x);
      continue;
    }
    const int row = pos & ((1 << a.view.page_shift) - 1);
    float y[EPL];
    if (a.h.format == TQ_KV_DENSE) {
      const int64_t from = page * a.h.page_stride + head * a.h.head_stride + (int64_t)row * DIM + lane * EPL;
#pragma unroll
      for (int j = 0; j < EPL; ++j) store_elem(a.out, a.out_dtype, to + j, load_elem(a.h.data, a.h.dtype, from + j));
      continue;
    }
    const uint32_t* words = reinterpret_cast<const uint32_t*>(a.h.data) + page * a.h.page_stride +
                            head * a.h.head_stride + (int64_t)row * pd;
    const float nrm = a.h.norms[page * a.h.norm_page_stride + head * a.h.norm_head_stride + row];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane * EPL + j;
      y[j] = cs_s[(__ldg(words + e / vpw) >> ((e % vpw) * a.h.bits)) & mask];
    }
    warp_butterfly<EPL>(y, lane);
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      store_elem(a.out, a.out_dtype, to + j,
                 __fmul_rn(__fmul_rn(__fmul_rn(y[j], a.s), sign_at(a.h.signs, lane * EPL + j)), nrm));
  }
}

template <int EPL>
int launch_read(const ReadArgs& a, cudaStream_t st) {
  const int64_t blocks = ((int64_t)a.batch * a.heads * a.length + kWarps - 1) / kWarps;
  const int64_t cap = (int64_t)num_sms() * 8;
  paged_read_kernel<EPL><<<(unsigned)(blocks < cap ? blocks : cap), kWarps * 32, 0, st>>>(a);
  return check_launch("tq_paged_dequantize");
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" int tq_paged_append(const tq_paged_params* p) {
  int rc = check_paged_params(p);
  if (rc) return rc;
  TQ_REQUIRE(p->tokens >= 0 && p->tokens < (1ll << 31) - 256, TQ_ERR_BAD_ARG, "tokens out of range");
  if (p->tokens == 0) return TQ_OK;
  AppendArgs a;
  memset(&a, 0, sizeof(a));
  const tq_paged_half* half[2] = {&p->k, &p->v};
  for (int i = 0; i < 2; ++i) {
    const char* what = i ? "values" : "keys";
    AppendHalf& s = a.half[i];
    if ((rc = fill_paged_half(half[i], p->dim, what, true, half[i]->format == TQ_KV_POLAR, &s.h, &s.thr))) return rc;
    s.x = half[i]->rows;
    s.x_dtype = half[i]->rows_dtype;
    TQ_REQUIRE(s.x && s.x_dtype >= TQ_F32 && s.x_dtype <= TQ_BF16, TQ_ERR_BAD_ARG,
               "%s: new rows must be given, as float32, float16 or bfloat16", what);
    TQ_REQUIRE(s.h.format != TQ_KV_DENSE || s.x_dtype == s.h.dtype, TQ_ERR_BAD_ARG, "%s: new rows must have the pages' type", what);
    s.batch_stride = half[i]->rows_batch_stride;
    s.head_stride = half[i]->rows_head_stride;
    s.token_stride = half[i]->rows_token_stride;
  }
  if ((rc = fill_page_view(p, &a.view))) return rc;
  a.batch = p->batch;
  a.heads = p->n_kv_heads;
  a.tokens = (int)p->tokens;
  a.starts = p->seq_lens;
  a.counts = p->counts;
  cudaStream_t st = (cudaStream_t)p->stream;
  switch (p->dim) {
    case 32: return launch_append<1>(a, st);
    case 64: return launch_append<2>(a, st);
    case 128: return launch_append<4>(a, st);
    default: return launch_append<8>(a, st);
  }
}

extern "C" int tq_paged_dequantize(const tq_paged_params* p) {
  int rc = check_paged_params(p);
  if (rc) return rc;
  TQ_REQUIRE(p->tokens >= 0 && p->tokens < (1ll << 31) - 256, TQ_ERR_BAD_ARG, "length out of range");
  TQ_REQUIRE(p->out_dtype >= TQ_F32 && p->out_dtype <= TQ_BF16, TQ_ERR_BAD_ARG, "bad out_dtype");
  if (p->tokens == 0) return TQ_OK;
  TQ_REQUIRE(p->out, TQ_ERR_BAD_ARG, "NULL output");
  ReadArgs a;
  memset(&a, 0, sizeof(a));
  if ((rc = fill_paged_half(&p->v, p->dim, "pages", false, p->v.format == TQ_KV_POLAR, &a.h, nullptr))) return rc;
  if ((rc = fill_page_view(p, &a.view))) return rc;
  a.s = (float)(1.0 / sqrt((double)p->dim));
  for (int i = 0; i < 16; ++i) a.h.cent.v[i] *= a.s;
  a.batch = p->batch;
  a.heads = p->n_kv_heads;
  a.length = p->tokens;
  a.lens = p->seq_lens;
  a.out = p->out;
  a.out_dtype = p->out_dtype;
  cudaStream_t st = (cudaStream_t)p->stream;
  switch (p->dim) {
    case 32: return launch_read<1>(a, st);
    case 64: return launch_read<2>(a, st);
    case 128: return launch_read<4>(a, st);
    default: return launch_read<8>(a, st);
  }
}
