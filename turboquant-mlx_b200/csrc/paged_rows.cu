// Paged caches: quantize-on-insert of new rows into pages, and pages read back as dense rows.
#include <math.h>
#include <string.h>

#include <type_traits>

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
// One token for each of 32 sequences, 8 heads: 3.5 us, a launch's latency.
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

// ---- two 32-bit floats at once ---------------------------------------------------------------------------------
// Packed add / mul / fma round each half exactly like the scalar operation, in one instruction.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float lo2(f2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi2(f2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// The 32 sign bits of a stretch of elements, laid out for 16-bit pairs: the even element of pair k at bit k, the odd one at
// 16 + k, so that one shift and one mask put a pair's signs at bits 15 and 31.
__device__ __forceinline__ uint32_t spread_signs(uint32_t w) {
  uint32_t r = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) r |= (((w >> (2 * k)) & 1u) << k) | (((w >> (2 * k + 1)) & 1u) << (16 + k));
  return r;
}
// Raw butterfly of a vector of 128 spread over two threads (q = 0, 1): v[i] holds elements i and i + 32 of the thread's
// 64, so that the stages 1 .. 16 are packed; the same sums and differences as a sequential butterfly (a - b as
// fma(b, -1, a): one rounding, the same).
__device__ __forceinline__ void butterfly_pairs(f2 (&v)[32], int q) {
  const f2 minus = pack2(-1.f, -1.f);
#pragma unroll
  for (int h = 1; h < 32; h <<= 1)
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if ((j & h) == 0) {
        const f2 a = v[j], b = v[j + h];
        v[j] = add2(a, b);
        v[j + h] = fma2(b, minus, a);
      }
  const float sg = q ? -1.f : 1.f;
  const f2 sg2 = pack2(sg, sg);
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float a = lo2(v[j]), b = hi2(v[j]);
    const float s = __fadd_rn(a, b), d = __fsub_rn(a, b);
    const f2 other = pack2(__shfl_xor_sync(0xffffffffu, s, 1), __shfl_xor_sync(0xffffffffu, d, 1));
    v[j] = fma2(pack2(s, d), sg2, other);            // lower thread: mine + other, upper: other - mine
  }
}

// ---- insert of many tokens: head_dim 128, 3 / 4-bit codes (or 16-bit dense keys), 16-bit rows -----------------------
// Six prompts of up to 5000 tokens, 8 heads, 3-bit: 59 us = 1.7 TB/s.  The exact 32-bit arithmetic (23 instructions per
// element) is 26 us of that at full issue; the rest is latency, which 16 warps per SM at 128 registers (and 16 spilled
// bytes per thread) do not cover, and half-rate instructions.  The work is cut to what the format asks for: two threads
// per vector, packed pairs (elements i and i + 32 of a
// thread's 64) for squares, division and butterfly, and one table lookup per code instead of a search: a monotone map
// puts the rotated value into one of kBuckets buckets that hold at most one threshold each (the host makes sure), and the
// bucket's entry says how many thresholds lie below and which one to compare with.  A copy of the table per lane: no
// bank conflicts.
// A warp takes 16 consecutive tokens of one head, whose rows are neighbours in their page.
constexpr int kBuckets = 64;
constexpr int kSplitTokens = 16;
struct BucketMap {
  float mul, add;                    // v = saturate(x * mul + add); bucket = round(v * (kBuckets - 1))
  float thr[kBuckets];               // the threshold inside the bucket, +inf: none
  uint8_t below[kBuckets];           // thresholds in lower buckets
};
struct SplitArgs {
  AppendArgs a;
  BucketMap map[2];
};
__host__ __device__ inline float bucket_float(float x, float mul, float add) {
#ifdef __CUDA_ARCH__
  return fmaf(__saturatef(fmaf(x, mul, add)), (float)(kBuckets - 1), 8388608.f);
#else
  const float v = fmaf(x, mul, add);
  return fmaf(v > 0.f ? (v < 1.f ? v : 1.f) : 0.f, (float)(kBuckets - 1), 8388608.f);     // 2^23 + bucket
#endif
}

// Encodes 16 tokens of one head (n of them real).  rows / norms: where each token's words and norm go; `together`: the
// rows are one stretch of memory.
template <typename T, int BITS>
__device__ __forceinline__ void encode_tokens(const AppendHalf& s, const BucketMap& map, uint32_t tab_lane, const uint32_t (&spread)[2],
                                              uint32_t* stage, uint32_t* const* rows, float* const* norms, bool together,
                                              const uint16_t* src0, int n, int lane) {
  constexpr int PD = packed_words(128, BITS);
  const int q = lane & 1, vs = lane >> 1;
  // lanes behind the last token repeat it and store nothing
  const uint4* src = reinterpret_cast<const uint4*>(src0 + min(vs, n - 1) * s.token_stride) + 8 * q;
  f2 x[32];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 wa = __ldg(src + c), wb = __ldg(src + 4 + c);                  // elements 8 c .. and 32 + 8 c ..
    const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = 8 * c + 2 * k;
      const uint32_t fa = ua[k] ^ ((spread[0] << (15 - e / 2)) & 0x80008000u);        // signs of the pair
      const uint32_t fb = ub[k] ^ ((spread[1] << (15 - e / 2)) & 0x80008000u);
      if (std::is_same<T, __half>::value) {
        const __half2 ha = *reinterpret_cast<const __half2*>(&fa), hb = *reinterpret_cast<const __half2*>(&fb);
        x[e] = pack2(__low2float(ha), __low2float(hb));
        x[e + 1] = pack2(__high2float(ha), __high2float(hb));
      } else {
        x[e] = pack2(__uint_as_float(fa << 16), __uint_as_float(fb << 16));
        x[e + 1] = pack2(__uint_as_float(fa & 0xffff0000u), __uint_as_float(fb & 0xffff0000u));
      }
    }
  }
  // sum of squares by the pairwise tree in natural order (squares of 16-bit values are exact in 32 bits, so the fma
  // rounds once, like the tree's first addition)
  f2 ss[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) ss[i] = fma2(x[2 * i + 1], x[2 * i + 1], mul2(x[2 * i], x[2 * i]));
#pragma unroll
  for (int h = 1; h < 16; h <<= 1)
#pragma unroll
    for (int i = 0; i < 16; i += 2 * h) ss[i] = add2(ss[i], ss[i + h]);
  float sum = __fadd_rn(lo2(ss[0]), hi2(ss[0]));
  sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 1));
  const float nrm = __fsqrt_rn(sum), safe = fmaxf(nrm, 1e-8f);
  if (safe < 1e30f) {
    // x / safe, correctly rounded: with a numerator of at most 11 bits one residual correction of x * RN(1 / safe) is
    // enough (div_rn of quantize_fast.cu says why)
    const float y = __frcp_rn(safe);
    const f2 y2 = pack2(y, y), nb = pack2(-safe, -safe);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const f2 d = mul2(x[i], y2);
      x[i] = fma2(fma2(nb, d, x[i]), y2, d);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = pack2(__fdiv_rn(lo2(x[i]), safe), __fdiv_rn(hi2(x[i]), safe));
  }
  butterfly_pairs(x, q);
  // codes -> this thread's bit string (64 codes)
  constexpr int DW = 2 * BITS;
  uint32_t dense[DW];
#pragma unroll
  for (int w = 0; w < DW; ++w) dense[w] = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const float v = i < 32 ? lo2(x[i & 31]) : hi2(x[i & 31]);
    const uint32_t at = (__float_as_uint(bucket_float(v, map.mul, map.add)) << 8) + tab_lane;     // 2^23's exponent is shifted out
    uint32_t thr, below;
    asm("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(thr), "=r"(below) : "r"(at));
    const int bit = i * BITS, w = bit >> 5, sh = bit & 31;
    if (sh + BITS > 32) {                                   // the code straddles two words
      const uint32_t code = below + (v > __uint_as_float(thr) ? 1u : 0u);
      dense[w] += code << sh;
      dense[w + 1] += code >> (32 - sh);
    } else {                                                // fields never overlap: + is |
      dense[w] += below << sh;
      if (v > __uint_as_float(thr)) dense[w] += 1u << sh;
    }
  }
  if (BITS == 4) {
    if (vs < n) {
      uint4* to = reinterpret_cast<uint4*>(rows[vs] + DW * q);
      to[0] = make_uint4(dense[0], dense[1], dense[2], dense[3]);
      to[1] = make_uint4(dense[DW - 4], dense[DW - 3], dense[DW - 2], dense[DW - 1]);
    }
  } else {
    // this thread's 192 bits -> 30-bit words: the first thread's are words 0 .. 5 and the low 12 bits of word 6, the
    // second's the high 18 bits of word 6 and words 7 .. 12
    const uint32_t low12 = __shfl_xor_sync(0xffffffffu, dense[DW - 1] >> 20, 1);
    uint32_t* to = stage + vs * PD;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      const int b0 = 30 * k, b1 = 18 + 30 * k;               // first bit of word k (first thread), of word 7 + k (second)
      const uint32_t w0 = __funnelshift_r(dense[b0 >> 5], (b0 >> 5) + 1 < DW ? dense[((b0 >> 5) + 1) % DW] : 0u, b0 & 31);
      const uint32_t w1 = __funnelshift_r(dense[b1 >> 5], (b1 >> 5) + 1 < DW ? dense[((b1 >> 5) + 1) % DW] : 0u, b1 & 31);
      to[q ? 7 + k : k] = (q ? w1 : w0) & 0x3fffffffu;
    }
    if (q) to[6] = low12 | ((dense[0] & 0x3ffffu) << 12);
    __syncwarp();
    if (together) {
      uint32_t* dst = rows[0];
#pragma unroll
      for (int k = 0; k < (kSplitTokens * PD + 31) / 32; ++k) {
        const int i = 32 * k + lane;
        if (i < n * PD) dst[i] = stage[i];
      }
    } else {
      for (int i = lane; i < n * PD; i += 32) rows[i / PD][i % PD] = stage[i];
    }
  }
  if (q == 0 && vs < n) *norms[vs] = nrm;
  __syncwarp();
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32, 2)
paged_append_split_kernel(const __grid_constant__ SplitArgs p) {
  __shared__ __align__(256) uint2 table[2][kBuckets * 32];
  __shared__ uint32_t stage_s[kWarps][kSplitTokens * 13];
  __shared__ uint32_t* rows_s[kWarps][kSplitTokens];
  __shared__ float* norms_s[kWarps][kSplitTokens];
  constexpr int kEntries = 256;
  __shared__ int prefix[kEntries + 1];
  const AppendArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane & 1;
#pragma unroll
  for (int which = 0; which < 2; ++which)
    if (a.half[which].h.format == TQ_KV_POLAR)
      for (int i = threadIdx.x; i < kBuckets * 32; i += kWarps * 32)
        table[which][i] = make_uint2(__float_as_uint(p.map[which].thr[i >> 5]), p.map[which].below[i >> 5]);
  __syncthreads();
  // Units of work: (sequence, half, head, 16 tokens), only those that exist: prefix[e] = chunks of 16 tokens in the
  // sequences in front of entry e (kEntries entries of `per` sequences each).
  const int per = (a.batch + kEntries - 1) / kEntries, entries = (a.batch + per - 1) / per;
  auto chunks_of = [&](int b) {
    const int count = min(a.tokens, a.counts ? __ldg(a.counts + b) : a.tokens);
    return (max(count, 0) + kSplitTokens - 1) / kSplitTokens;
  };
  for (int e = threadIdx.x; e < entries; e += kWarps * 32) {
    int c = 0;
    for (int b = e * per; b < min(a.batch, (e + 1) * per); ++b) c += chunks_of(b);
    prefix[e + 1] = c;
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
  if (warp == 0)
    for (int e0 = 1, carry = 0; e0 <= entries; e0 += 32) {
      const int e = e0 + lane;
      int c = e <= entries ? prefix[e] : 0;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, c, k);
        if (lane >= k) c += o;
      }
      c += carry;
      if (e <= entries) prefix[e] = c;
      carry = __shfl_sync(0xffffffffu, c, 31);
    }
  __syncthreads();
  const uint32_t spread[2][2] = {
      {spread_signs(a.half[0].h.signs.w[2 * q]), spread_signs(a.half[0].h.signs.w[2 * q + 1])},
      {spread_signs(a.half[1].h.signs.w[2 * q]), spread_signs(a.half[1].h.signs.w[2 * q + 1])}};
  const uint32_t rows2 = 2 * a.heads, units = (uint32_t)prefix[entries] * rows2;      // below 2^31: the launcher has checked
  for (uint32_t u = blockIdx.x * kWarps + warp; u < units; u += gridDim.x * kWarps) {
    int e = 0, hi = entries - 1;
    while (e < hi) {                           // last entry that does not begin behind u
      const int mid = (e + hi + 1) / 2;
      if ((uint32_t)prefix[mid] * rows2 <= u) e = mid;
      else hi = mid - 1;
    }
    uint32_t rest = u - (uint32_t)prefix[e] * rows2;
    int b = e * per;
    uint32_t chunks = chunks_of(b);
    while (rest >= chunks * rows2) {
      rest -= chunks * rows2;
      chunks = chunks_of(++b);
    }
    const int hr = (int)(rest / chunks), t0 = (int)(rest - (uint32_t)hr * chunks) * kSplitTokens;
    const int which = hr / a.heads, head = hr - which * a.heads;
    const int count = min(a.tokens, a.counts ? __ldg(a.counts + b) : a.tokens);
    const int n = min(kSplitTokens, count - t0);
    int row = 0;
    const int page = append_place(a, b, t0 + min(lane, n - 1), &row);        // lane = token
    const bool all = __all_sync(0xffffffffu, page >= 0);
    const bool together = __all_sync(0xffffffffu, page == __shfl_sync(0xffffffffu, page, 0));
    {
      const AppendHalf& s = a.half[which];
      const uint16_t* src = reinterpret_cast<const uint16_t*>(s.x) + b * s.batch_stride + head * s.head_stride + t0 * s.token_stride;
      if (lane < kSplitTokens) {
        uint32_t* to = nullptr;
        if (page >= 0) {
          if (s.h.format == TQ_KV_DENSE)
            to = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(s.h.data) + page * s.h.page_stride +
                                             head * s.h.head_stride + (int64_t)row * 128);
          else
            to = reinterpret_cast<uint32_t*>(s.h.data) + page * s.h.page_stride + head * s.h.head_stride +
                 row * packed_words(128, s.h.bits);
          norms_s[warp][lane] = s.h.norms + page * s.h.norm_page_stride + head * s.h.norm_head_stride + row;
        }
        rows_s[warp][lane] = to;
      }
      __syncwarp();
      if (s.h.format == TQ_KV_DENSE) {
        for (int i = lane; i < n * 16; i += 32) {          // 16 chunks of 16 bytes per row
          const int r = i >> 4, c = i & 15;
          uint4* to = reinterpret_cast<uint4*>(rows_s[warp][r]);
          if (to) to[c] = __ldg(reinterpret_cast<const uint4*>(src + r * s.token_stride) + c);
        }
      } else if (all) {
        const uint32_t tab_lane = (uint32_t)__cvta_generic_to_shared(table[which]) + lane * 8;
        const uint32_t sg[2] = {which ? spread[1][0] : spread[0][0], which ? spread[1][1] : spread[0][1]};
        if (s.h.bits == 3)
          encode_tokens<T, 3>(s, p.map[which], tab_lane, sg, stage_s[warp], rows_s[warp], norms_s[warp], together, src, n, lane);
        else
          encode_tokens<T, 4>(s, p.map[which], tab_lane, sg, stage_s[warp], rows_s[warp], norms_s[warp], together, src, n, lane);
      } else {
        // some token has no place (reported): the others one by one
        for (int r = 0; r < n; ++r) {
          const int pg = __shfl_sync(0xffffffffu, page, r), rw = __shfl_sync(0xffffffffu, row, r);
          if (pg < 0) continue;
          float x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = load_elem(src, s.x_dtype, r * s.token_stride + lane * 4 + j);
          uint8_t* idx = reinterpret_cast<uint8_t*>(stage_s[warp]);
          if (s.h.bits == 3) encode_row<4, 3>(s, x, idx, pg, head, rw, lane);
          else encode_row<4, 4>(s, x, idx, pg, head, rw, lane);
        }
      }
      __syncwarp();
    }
  }
}

// False when some bucket would hold two thresholds (a codebook with levels very close to each other).
bool make_buckets(const Table16& thr, int n, BucketMap* m) {
  const double lo = thr.v[0], hi = thr.v[n - 1], span = hi - lo;
  if (!(span > 0) || !(span < 1e30)) return false;
  // thresholds from bucket 1 to kBuckets - 2
  const double inv = (kBuckets - 3) / span;
  m->mul = (float)(inv / (kBuckets - 1));
  m->add = (float)((1.0 - lo * inv) / (kBuckets - 1));
  for (int k = 0; k < kBuckets; ++k) {
    m->thr[k] = INFINITY;
    m->below[k] = 0;
  }
  for (int i = 0; i < n; ++i) {
    const int k = (int)(bucket_float(thr.v[i], m->mul, m->add) - 8388608.f);
    if (k < 0 || k >= kBuckets || m->thr[k] != INFINITY) return false;
    m->thr[k] = thr.v[i];
    for (int j = k + 1; j < kBuckets; ++j) ++m->below[j];
  }
  return true;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Whether a half of an insert qualifies for the kernel above.
bool split_supported(const AppendHalf& s, BucketMap* map) {
  if (s.x_dtype == TQ_F32 || !aligned16(s.x) || s.batch_stride % 8 || s.head_stride % 8 || s.token_stride % 8) return false;
  if (s.h.format == TQ_KV_DENSE) return aligned16(s.h.data) && s.h.page_stride % 8 == 0 && s.h.head_stride % 8 == 0;
  if (s.h.bits != 3 && s.h.bits != 4) return false;
  if (s.h.bits == 4 && (!aligned16(s.h.data) || s.h.page_stride % 4 || s.h.head_stride % 4)) return false;
  return make_buckets(s.thr, (1 << s.h.bits) - 1, map);
}

int launch_append_split(const SplitArgs& p, cudaStream_t st) {
  const int64_t units = (int64_t)p.a.batch * 2 * p.a.heads * ((p.a.tokens + kSplitTokens - 1) / kSplitTokens);
  const int64_t blocks = (units + kWarps - 1) / kWarps, cap = (int64_t)num_sms() * 2;
  const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
  if (p.a.half[0].x_dtype == TQ_F16) paged_append_split_kernel<__half><<<grid, kWarps * 32, 0, st>>>(p);
  else paged_append_split_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, st>>>(p);
  return check_launch("tq_paged_append (split)");
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
// contiguous decoder, so both give the same bits.  Rows behind a sequence, or of a page it does not hold, are zero.
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
    const int page = pos < n ? a.view.entry(b, pos) : -1;
    const bool wrong = page < -1 || page >= a.view.n_pages;
    if (wrong && lane == 0) atomicExch(a.view.status, 1);
    if (page < 0 || wrong) {         // behind the sequence, or no page held: zero; a page outside the pool: NaN
      const float x = wrong ? __int_as_float(0x7fc00000) : 0.f;
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

// Head_dim 128, 3 / 4-bit codes, 16-bit output: two threads per row, packed pairs (elements i and i + 32 of a thread's
// 64).  The codes of such a pair are put side by side bit field by bit field, so that one table entry (a copy per half
// warp lane: conflict free) is the packed pair of scaled centroids; the same butterfly, and ((x * s) * sign) * norm with
// the sign applied to the rounded result (rounding is symmetric).  Rows leave through shared memory, so that every
// store instruction covers two whole rows.  8 prefixes of up to 16384 tokens, 8 heads, 4-bit codes 67 us = 4.6 TB/s
// (0.70 of the copy peak; a warp per row, 32-bit output: 282 us for 1.8 times the bytes): HBM, then the shared-memory pipe,
// which the table, the butterfly's cross-thread stage and the output exchange have in common.
constexpr int kReadRows = 16;
template <typename T, int BITS>
__global__ void __launch_bounds__(kWarps * 32, 2)
paged_read_split_kernel(const __grid_constant__ ReadArgs a) {
  constexpr int ENTRIES = 1 << (2 * BITS), DW = 2 * BITS, PD = packed_words(128, BITS);
  extern __shared__ __align__(256) uint8_t dyn[];
  uint2* table = reinterpret_cast<uint2*>(dyn);                                   // [entry][16 copies]
  uint8_t* out_s = dyn + ENTRIES * 128 + (threadIdx.x >> 5) * (kReadRows * 256);  // the warp's rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane & 1, vs = lane >> 1;
  for (int i = threadIdx.x; i < ENTRIES * 16; i += kWarps * 32) {
    const int e = i >> 4;
    table[i] = make_uint2(__float_as_uint(a.h.cent.v[e & ((1 << BITS) - 1)]), __float_as_uint(a.h.cent.v[e >> BITS]));
  }
  __syncthreads();
  const uint32_t tab = (uint32_t)__cvta_generic_to_shared(dyn) + (lane & 15) * 8;
  const uint32_t out_at = (uint32_t)__cvta_generic_to_shared(out_s);
  const uint32_t spread[2] = {spread_signs(a.h.signs.w[2 * q]), spread_signs(a.h.signs.w[2 * q + 1])};
  const f2 s2 = pack2(a.s, a.s);
  const int64_t chunks = (a.length + kReadRows - 1) / kReadRows, units = (int64_t)a.batch * a.heads * chunks;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + warp; u < units; u += (int64_t)gridDim.x * kWarps) {
    const int64_t bh = u / chunks;
    const int p0 = (int)(u - bh * chunks) * kReadRows, b = (int)(bh / a.heads), head = (int)(bh - (int64_t)b * a.heads);
    const int n = min(__ldg(a.lens + b), a.view.capacity());
    const int pos = p0 + vs;
    const int last = (int)min((int64_t)kReadRows, a.length - p0);                  // rows of this chunk in the output
    uint4* out = reinterpret_cast<uint4*>(a.out) + (bh * a.length + p0) * 16;
    if (p0 >= n) {                       // the whole chunk lies behind the sequence
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (2 * k + (lane >> 4) < last) out[k * 32 + lane] = make_uint4(0, 0, 0, 0);
      continue;
    }
    int page = pos < n && vs < last ? a.view.entry(b, pos) : -1;
    const bool missing = page < -1 || page >= a.view.n_pages;        // outside the pool; -1: no page held, zeros
    if (missing) page = -1;
    if (missing && q == 0) atomicExch(a.view.status, 1);
    uint32_t dense[DW + 1];
    float nrm = 0.f;
#pragma unroll
    for (int w = 0; w <= DW; ++w) dense[w] = 0;
    if (page >= 0) {
      const int row = pos & ((1 << a.view.page_shift) - 1);
      const uint32_t* words = reinterpret_cast<const uint32_t*>(a.h.data) + page * a.h.page_stride + head * a.h.head_stride +
                              (int64_t)row * PD;
      nrm = __ldg(a.h.norms + page * a.h.norm_page_stride + head * a.h.norm_head_stride + row);
      if (BITS == 4) {
        const uint4 w0 = __ldg(reinterpret_cast<const uint4*>(words + DW * q)), w1 = __ldg(reinterpret_cast<const uint4*>(words + DW * q) + 1);
        dense[0] = w0.x; dense[1] = w0.y; dense[2] = w0.z; dense[3] = w0.w;
        dense[DW - 4] = w1.x; dense[DW - 3] = w1.y; dense[DW - 2] = w1.z; dense[DW - 1] = w1.w;
      } else {
        // this thread's 64 codes = bits [192 q, 192 q + 192) of the string of 30-bit words: words 6 q .. 6 q + 6 from bit 12 q
        uint32_t w[7];
#pragma unroll
        for (int k = 0; k < 7; ++k) w[k] = __ldg(words + 6 * q + k);
        // seven 30-bit words -> six 32-bit ones starting 12 q bits in
#pragma unroll
        for (int k = 0; k < 6; ++k) {
          const int bit = 32 * k, w0 = bit / 30, o0 = bit % 30;                    // q = 0
          uint32_t d0 = w[w0] >> o0 | w[w0 + 1] << (30 - o0);
          if (60 - o0 < 32 && w0 + 2 < 7) d0 |= w[w0 + 2] << (60 - o0);
          const int bit1 = 32 * k + 12, w1 = bit1 / 30, o1 = bit1 % 30;            // q = 1
          uint32_t d1 = w[w1] >> o1;
          if (w1 + 1 < 7) d1 |= w[w1 + 1] << (30 - o1);
          if (60 - o1 < 32 && w1 + 2 < 7) d1 |= w[w1 + 2] << (60 - o1);
          dense[k] = q ? d1 : d0;
        }
      }
    }
    // pairs (i, i + 32): 3-bit codes: both halves of the thread's string are 96 bits = 3 words; 4-bit: 128 bits = 4 words
    constexpr int HW = DW / 2;
    f2 x[32];
    if (BITS == 4) {
#pragma unroll
      for (int w = 0; w < HW; ++w) {
        const uint32_t ev = (dense[w] & 0x0F0F0F0Fu) | ((dense[w + HW] << 4) & 0xF0F0F0F0u);
        const uint32_t od = ((dense[w] >> 4) & 0x0F0F0F0Fu) | (dense[w + HW] & 0xF0F0F0F0u);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t f = ((k & 1) ? od : ev) >> (8 * (k >> 1)) & 0xFFu;
          asm("ld.shared.b64 %0, [%1];" : "=l"(x[8 * w + k]) : "r"(tab + f * 128));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int bit = 3 * i, w = bit >> 5, sh = bit & 31;
        const uint32_t ca = sh + 3 <= 32 ? dense[w] >> sh : __funnelshift_r(dense[w], dense[w + 1], sh);
        const uint32_t cb = sh + 3 <= 32 ? dense[w + HW] >> sh : __funnelshift_r(dense[w + HW], dense[w + HW + 1], sh);
        const uint32_t f = (ca & 7u) | ((cb & 7u) << 3);
        asm("ld.shared.b64 %0, [%1];" : "=l"(x[i]) : "r"(tab + f * 128));
      }
    }
    butterfly_pairs(x, q);
    // a row behind the sequence has norm 0 and no signs: zeros; one without a page is NaN
    const float nq = missing ? __int_as_float(0x7fc00000) : nrm;
    const f2 n2 = pack2(nq, nq);
    const uint32_t fl[2] = {page >= 0 ? spread[0] : 0u, page >= 0 ? spread[1] : 0u};
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = mul2(mul2(x[i], s2), n2);
    // (the centroids of a row of norm 0 may be negative: x * 0 = -0; adding 0 clears it)
    const f2 zero2 = pack2(0.f, 0.f);
    if (__any_sync(0xffffffffu, page < 0)) {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = page < 0 ? add2(x[i], zero2) : x[i];
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = 8 * c + 2 * k;
          const float y0 = half ? hi2(x[e]) : lo2(x[e]), y1 = half ? hi2(x[e + 1]) : lo2(x[e + 1]);
          uint32_t h;
          if (std::is_same<T, __half>::value) {
            const __half2 v = __floats2half2_rn(y0, y1);
            h = *reinterpret_cast<const uint32_t*>(&v);
          } else {
            const __nv_bfloat162 v = __floats2bfloat162_rn(y0, y1);
            h = *reinterpret_cast<const uint32_t*>(&v);
          }
          pk[k] = h ^ ((fl[half] << (15 - e / 2)) & 0x80008000u);      // signs of elements e and e + 1
        }
        const int chunk = 8 * q + 4 * half + c;              // 16-byte chunk of the row; places are swizzled against conflicts
        const uint32_t at = out_at + vs * 256 + (chunk & 8) * 16 + ((chunk & 7) ^ ((2 * vs + q) & 7)) * 16;
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]) : "memory");
      }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = 2 * k + (lane >> 4), chunk = lane & 15;
      uint4 v;
      const uint32_t at = out_at + r * 256 + (chunk & 8) * 16 + ((chunk & 7) ^ ((2 * r + (chunk >> 3)) & 7)) * 16;
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
      if (r < last) out[r * 16 + chunk] = v;
    }
    __syncwarp();
  }
}

template <typename T, int BITS>
int launch_read_split(const ReadArgs& a, cudaStream_t st) {
  constexpr int smem = (1 << (2 * BITS)) * 128 + kWarps * kReadRows * 256;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_read_split_kernel<T, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_error(TQ_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  const int64_t units = (int64_t)a.batch * a.heads * ((a.length + kReadRows - 1) / kReadRows);
  const int64_t blocks = (units + kWarps - 1) / kWarps, cap = (int64_t)num_sms() * 2;
  paged_read_split_kernel<T, BITS><<<(unsigned)(blocks < cap ? blocks : cap), kWarps * 32, smem, st>>>(a);
  return check_launch("tq_paged_dequantize (split)");
}

bool read_split_supported(const ReadArgs& a, int dim) {
  if (dim != 128 || a.h.format != TQ_KV_POLAR || (a.h.bits != 3 && a.h.bits != 4) || a.out_dtype == TQ_F32) return false;
  if (!aligned16(a.out)) return false;
  return a.h.bits == 3 || (aligned16(a.h.data) && a.h.page_stride % 4 == 0 && a.h.head_stride % 4 == 0);
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
  // From 16 tokens on a warp's worth of neighbouring rows exists: two threads per vector (six prompts of up to 5000
  // tokens, 8 heads, 3-bit: 59 us against 184 with a warp per row).
  const int64_t units = (int64_t)a.batch * a.heads * ((a.tokens + kSplitTokens - 1) / kSplitTokens);
  if (p->dim == 128 && a.tokens >= kSplitTokens && a.half[0].x_dtype == a.half[1].x_dtype && units < (1ll << 28)) {
    SplitArgs sp;
    memset(&sp, 0, sizeof(sp));
    if (split_supported(a.half[0], &sp.map[0]) && split_supported(a.half[1], &sp.map[1])) {
      sp.a = a;
      return launch_append_split(sp, st);
    }
  }
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
  if (read_split_supported(a, p->dim)) {
    if (a.out_dtype == TQ_F16) return a.h.bits == 3 ? launch_read_split<__half, 3>(a, st) : launch_read_split<__half, 4>(a, st);
    return a.h.bits == 3 ? launch_read_split<__nv_bfloat16, 3>(a, st) : launch_read_split<__nv_bfloat16, 4>(a, st);
  }
  switch (p->dim) {
    case 32: return launch_read<1>(a, st);
    case 64: return launch_read<2>(a, st);
    case 128: return launch_read<4>(a, st);
    default: return launch_read<8>(a, st);
  }
}
