// Fused PolarQuant encode for head_dim 128, TPV = 1, 2 or 4 threads per vector (default 2).
//
// Thread q of a group holds elements [EPT q, EPT q + EPT), EPT = 128 / TPV: log2(EPT) stages run in
// registers and log2(TPV) through warp shuffles, the sum of squares follows the same
// pairwise tree (in-thread, then the partners), so results are
// bit-identical to the general warp-per-vector kernel and to the CPU oracle.
// Compared with one thread per vector (all 128 values in registers) the body is
// a quarter of the size and uses ~a third of the registers: that version was
// bound by instruction fetch (top stall "no instruction", ~4000 unrolled
// instructions at 255 registers, one or two warps per scheduler).
//   load   : straight from global, 64 B (16-bit input) or 128 B (fp32) per thread;
//            a warp covers 8 consecutive rows, every byte of every line is used.
//   divide : x / max(norm, 1e-8) correctly rounded: reciprocal + two FMA residual
//            corrections (the sequence behind IEEE division), slow path for
//            extreme norms.
//   compare: binary search over the thresholds on the raw butterfly output.
//   store  : each thread packs its codes into a dense bit string; the threads of a
//            vector exchange the strings through shared memory and cut them into
//            the 30-bit (3-bit codes) words of the storage format; the rows of the
//            warp's consecutive vectors leave as 128-bit stores.
// Requirements (checked by the launcher): dim 128, bits 3 or 4, contiguous
// input rows, 16-byte aligned input.
#include <type_traits>

#include "common.cuh"

namespace tq {
namespace {

constexpr int kDimF = 128;
constexpr int kWarps = 8;            // warps per CTA; each warp encodes 8 vectors per pass

struct FastQuantArgs {
  const void* x;
  int64_t n_vecs;
  uint32_t n_inner;
  uint32_t* packed;
  int64_t packed_outer_stride;
  float* norms;
  int64_t norms_outer_stride;
  SignMask signs;
  Table16 thr;
};

// Correctly rounded a / b given y = RN(1 / b); a, b and the quotient in the normal
// range: Markstein's residual correction.  Scaled to a, b in [1, 2): |b y - 1| <= b 2^-25,
// so q = RN(a y) is within 0.5 + a / 2 ulp of a / b and the corrected value, before it is
// rounded, is off by |a / b - q| |b y - 1|.  Rounding it is wrong only if that passes a
// midpoint m.  a - b m is a nonzero multiple of 2^-47 (2^-48 for a quotient below 1), so
// a / b is d >= 2^-24 / b ulp away from m; while q is half an ulp from m, r is exact and the
// error is (1/2 + d) b 2^-25 ulp, less than d since b < 2.  A numerator of at most 11
// significant bits (fp16 / bf16 inputs) keeps q there (0.5 + a / 2 < 1.5 - 2^-11), so one
// correction rounds correctly; a general float32 numerator may start 1.5 ulp away and takes a
// second one.
template <bool NARROW_NUMERATOR>
__device__ __forceinline__ float div_rn(float a, float b, float y) {
  float q = __fmul_rn(a, y);
  float r = __fmaf_rn(-b, q, a);
  q = __fmaf_rn(r, y, q);
  if (!NARROW_NUMERATOR) {
    r = __fmaf_rn(-b, q, a);
    q = __fmaf_rn(r, y, q);
  }
  return q;
}

// Adds code(x) << SH into `word` (fields never overlap, so += is |=): binary search
// over the thresholds, the three (four) result bits added as immediates.
template <int BITS, int SH>
__device__ __forceinline__ void add_code(uint32_t& word, float x, const Table16& T) {
  if (BITS == 3) {
    const bool p2 = x > T.v[3];
    const float ta = p2 ? T.v[5] : T.v[1];
    const bool p1 = x > ta;
    const float tb = p2 ? (p1 ? T.v[6] : T.v[4]) : (p1 ? T.v[2] : T.v[0]);
    const bool p0 = x > tb;
    if (p2) word += 4u << SH;
    if (p1) word += 2u << SH;
    if (p0) word += 1u << SH;
  } else {
    const bool p3 = x > T.v[7];
    const float ta = p3 ? T.v[11] : T.v[3];
    const bool p2 = x > ta;
    const float tb = p3 ? (p2 ? T.v[13] : T.v[9]) : (p2 ? T.v[5] : T.v[1]);
    const bool p1 = x > tb;
    const float t_hi = p2 ? (p1 ? T.v[14] : T.v[12]) : (p1 ? T.v[10] : T.v[8]);
    const float t_lo = p2 ? (p1 ? T.v[6] : T.v[4]) : (p1 ? T.v[2] : T.v[0]);
    const bool p0 = x > (p3 ? t_hi : t_lo);
    if (p3) word += 8u << SH;
    if (p2) word += 4u << SH;
    if (p1) word += 2u << SH;
    if (p0) word += 1u << SH;
  }
}
template <int BITS>
__device__ __forceinline__ uint32_t code_of(float x, const Table16& T) {
  uint32_t c = 0;
  add_code<BITS, 0>(c, x, T);
  return c;
}

// TPV threads per vector (1, 2 or 4), EPT = 128 / TPV elements per thread.
template <typename T, int BITS, int TPV>
__global__ void __launch_bounds__(kWarps * 32)
quantize_split_kernel(const FastQuantArgs a) {
  constexpr int ESZ = sizeof(T);
  constexpr int EPT = kDimF / TPV;
  constexpr int VPWARP = 32 / TPV;              // vectors per warp pass
  constexpr int QB = EPT * ESZ;                 // bytes of a row held by one thread
  constexpr int NLD = QB / 16;                  // 16-byte loads per thread
  constexpr int PDIM = packed_words(kDimF, BITS);
  constexpr int DW = EPT * BITS / 32;           // dense words per thread
  __shared__ uint32_t dense_s[BITS == 3 ? kWarps : 1][VPWARP][TPV * DW + 1];
  // 3-bit rows: the 13 words of the warp's VPWARP consecutive vectors, stored as 16-byte vectors
  __shared__ __align__(16) uint32_t rows_s[BITS == 3 ? kWarps : 1][VPWARP * PDIM];
  // lets a kernel launched behind this one with programmatic stream serialization be scheduled
  // now; it waits for this grid's completion before it reads anything written here
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q = lane % TPV, vs = lane / TPV;
  const int64_t wg = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t wstride = (int64_t)gridDim.x * kWarps;
  // 16-bit inputs: the signs of this thread's elements, 16 element pairs per word with the even
  // element's bit at position k and the odd one's at 16 + k, so that one shift and one mask give the
  // flip mask (bits 15 and 31) of a packed pair
  constexpr int NSW = ESZ == 2 ? (EPT + 31) / 32 : 1;
  uint32_t spread[NSW];
  if (ESZ == 2) {
#pragma unroll
    for (int w = 0; w < NSW; ++w) {
      const uint32_t sw = a.signs.w[(EPT * q) / 32 + w];
      uint32_t sp = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) sp |= (((sw >> (2 * k)) & 1u) << k) | (((sw >> (2 * k + 1)) & 1u) << (16 + k));
      spread[w] = sp;
    }
  }
  const float sg_upper[3] = {(q & 1) ? -1.0f : 1.0f, (q & 2) ? -1.0f : 1.0f, (q & 4) ? -1.0f : 1.0f};

  for (int64_t vb = wg * VPWARP; vb < a.n_vecs; vb += wstride * VPWARP) {
    const int64_t v = vb + vs;
    const bool valid = v < a.n_vecs;
    const int64_t vl = valid ? v : a.n_vecs - 1;          // tail lanes recompute the last vector
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.x) +
                                                      vl * (kDimF * ESZ) + q * QB);
    float x[EPT];
    {
      uint4 w[NLD];
#pragma unroll
      for (int c = 0; c < NLD; ++c) w[c] = __ldg(src + c);
#pragma unroll
      for (int c = 0; c < NLD; ++c) {
        const uint32_t ww[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (ESZ == 2) {
            // flip the signs of both packed 16-bit values at once, then widen
            const int e = c * 8 + 2 * k;
            const int pair = e / 2;
            const uint32_t f = ww[k] ^ ((spread[pair / 16] << (15 - pair % 16)) & 0x80008000u);
            if (std::is_same<T, __half>::value) {
              const __half2 h = *reinterpret_cast<const __half2*>(&f);
              x[e] = __low2float(h);
              x[e + 1] = __high2float(h);
            } else {
              x[e] = __uint_as_float(f << 16);
              x[e + 1] = __uint_as_float(f & 0xffff0000u);
            }
          } else {
            x[c * 4 + k] = __uint_as_float(ww[k] ^ sign_bit_at(a.signs, EPT * q + c * 4 + k));
          }
        }
      }
    }
    // sum of squares: pairwise tree in natural order (in-thread, then partners 1, 2)
    float s[EPT / 2];
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      if (ESZ == 2)   // squares of 16-bit inputs are exact in float32: one rounding, as in the tree
        s[i] = __fmaf_rn(x[2 * i + 1], x[2 * i + 1], __fmul_rn(x[2 * i], x[2 * i]));
      else
        s[i] = __fadd_rn(__fmul_rn(x[2 * i], x[2 * i]), __fmul_rn(x[2 * i + 1], x[2 * i + 1]));
    }
#pragma unroll
    for (int h = 1; h < EPT / 2; h <<= 1) {
#pragma unroll
      for (int i = 0; i < EPT / 2; i += 2 * h) s[i] = __fadd_rn(s[i], s[i + h]);
    }
    float ss = s[0];
#pragma unroll
    for (int k = 1; k < TPV; k <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, k));
    const float nrm = __fsqrt_rn(ss);
    const float safe = fmaxf(nrm, 1e-8f);
    if (safe > 1e-30f && safe < 1e30f) {
      const float y = __frcp_rn(safe);
#pragma unroll
      for (int i = 0; i < EPT; ++i) x[i] = div_rn<ESZ == 2>(x[i], safe, y);
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i) x[i] = __fdiv_rn(x[i], safe);
    }
    // raw Walsh-Hadamard butterfly: stages below EPT in registers, the rest across partners
#pragma unroll
    for (int h = 1; h < EPT; h <<= 1) {
#pragma unroll
      for (int j = 0; j < EPT; ++j) {
        if ((j & h) == 0) {
          const float p = x[j], r = x[j + h];
          x[j] = __fadd_rn(p, r);
          x[j + h] = __fsub_rn(p, r);
        }
      }
    }
#pragma unroll
    for (int k = 1, ki = 0; k < TPV; k <<= 1, ++ki) {
      // upper partner: o - x = fma(x, -1, o), rounded exactly like the subtraction it replaces
#pragma unroll
      for (int j = 0; j < EPT; ++j) x[j] = __fmaf_rn(x[j], sg_upper[ki], __shfl_xor_sync(0xffffffffu, x[j], k));
    }
    // codes -> dense bit string of this thread (EPT * BITS bits)
    uint32_t dense[DW];
#pragma unroll
    for (int w = 0; w < DW; ++w) dense[w] = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      constexpr int kNoStraddle = 32 - BITS;
      const int bit = i * BITS, w = bit >> 5, sh = bit & 31;
      if (sh <= kNoStraddle) {
        // shift amount is a compile-time constant after unrolling; dispatch to the immediate form
        switch (sh) {
#define TQ_CASE(S) case S: add_code<BITS, S>(dense[w], x[i], a.thr); break;
          TQ_CASE(0) TQ_CASE(1) TQ_CASE(2) TQ_CASE(3) TQ_CASE(4) TQ_CASE(5) TQ_CASE(6) TQ_CASE(7)
          TQ_CASE(8) TQ_CASE(9) TQ_CASE(10) TQ_CASE(11) TQ_CASE(12) TQ_CASE(13) TQ_CASE(14) TQ_CASE(15)
          TQ_CASE(16) TQ_CASE(17) TQ_CASE(18) TQ_CASE(19) TQ_CASE(20) TQ_CASE(21) TQ_CASE(22) TQ_CASE(23)
          TQ_CASE(24) TQ_CASE(25) TQ_CASE(26) TQ_CASE(27) TQ_CASE(28) TQ_CASE(29)
#undef TQ_CASE
          default: break;
        }
      } else {   // the code straddles two dense words
        const uint32_t c = code_of<BITS>(x[i], a.thr);
        dense[w] |= c << sh;
        dense[w + 1] |= c >> (32 - sh);
      }
    }
    const uint32_t o_idx = (uint32_t)vl / a.n_inner, i_idx = (uint32_t)vl - o_idx * a.n_inner;
    uint32_t* prow = a.packed + (int64_t)o_idx * a.packed_outer_stride + (int64_t)i_idx * PDIM;
    if (BITS == 4) {
      if (valid) {
#pragma unroll
        for (int w = 0; w < DW; ++w) prow[DW * q + w] = dense[w];
      }
    } else {
      // the vector's 384-bit string -> thirteen 30-bit words
      uint32_t* ds = dense_s[warp][vs];
#pragma unroll
      for (int w = 0; w < DW; ++w) ds[DW * q + w] = dense[w];
      if (q == 0) ds[TPV * DW] = 0;
      __syncwarp();
      // the warp's vectors are consecutive; when their rows are too (same outer index, 16-byte
      // aligned start, all valid) they leave as 128-bit stores, otherwise word by word
      const uint32_t o_first = (uint32_t)vb / a.n_inner;
      const uint32_t i_first = (uint32_t)vb - o_first * a.n_inner;
      uint32_t* row_first = a.packed + (int64_t)o_first * a.packed_outer_stride + (int64_t)i_first * PDIM;
      const bool vec_store = vb + VPWARP <= a.n_vecs && i_first + VPWARP <= a.n_inner &&
                             (reinterpret_cast<uintptr_t>(row_first) & 15) == 0 && (VPWARP * PDIM) % 4 == 0;
#pragma unroll
      for (int k = 0; k < (PDIM + TPV - 1) / TPV; ++k) {
        const int w = q + TPV * k;
        if (w < PDIM) {
          const int bit = 30 * w, dw = bit >> 5, sh = bit & 31;
          const uint32_t word = __funnelshift_r(ds[dw], ds[dw + 1], sh) & 0x3fffffffu;
          if (vec_store) rows_s[warp][vs * PDIM + w] = word;
          else if (valid) prow[w] = word;
        }
      }
      __syncwarp();
      if (vec_store) {
        uint4* dst = reinterpret_cast<uint4*>(row_first);
        const uint4* src = reinterpret_cast<const uint4*>(rows_s[warp]);
#pragma unroll
        for (int c = lane; c < VPWARP * PDIM / 4; c += 32) dst[c] = src[c];
        __syncwarp();
      }
    }
    if (valid && q == 0) a.norms[(int64_t)o_idx * a.norms_outer_stride + i_idx] = nrm;
  }
}

template <typename T, int BITS, int TPV>
int launch_tpv(const FastQuantArgs& a, cudaStream_t st) {
  const int per_block = (32 / TPV) * kWarps;
  const int64_t groups = (a.n_vecs + per_block - 1) / per_block;
  const int64_t cap = (int64_t)num_sms() * 8;
  const int grid = (int)(groups < cap ? groups : cap);
  quantize_split_kernel<T, BITS, TPV><<<grid, kWarps * 32, 0, st>>>(a);
  return check_launch("tq_quantize (split per vector)");
}

template <typename T, int BITS>
int launch_fast(const FastQuantArgs& a, cudaStream_t st) {
  return launch_tpv<T, BITS, 2>(a, st);   // 2 threads per vector measured fastest on B200 (1: +28 %, 4: +9 %)
}

}  // namespace

// Returns TQ_ERR_UNSUPPORTED (without touching the error string) when the
// arguments do not qualify, so the caller can fall back to the general kernel.
int try_launch_quantize_fast(const void* x, int x_dtype, int64_t n_outer, int64_t n_inner,
                             int64_t x_outer_stride, int dim, int bits, const SignMask& signs,
                             const Table16& thr, uint32_t* packed, int64_t packed_outer_stride,
                             float* norms, int64_t norms_outer_stride, cudaStream_t st) {
  if (dim != kDimF || (bits != 3 && bits != 4)) return TQ_ERR_UNSUPPORTED;
  if (x_outer_stride != n_inner * dim) return TQ_ERR_UNSUPPORTED;            // rows must be contiguous
  if ((reinterpret_cast<uintptr_t>(x) & 15u) != 0) return TQ_ERR_UNSUPPORTED;
  const int64_t n_vecs = n_outer * n_inner;
  if (n_vecs < 1024 || n_vecs >= (1LL << 31) || n_inner >= (1LL << 31)) return TQ_ERR_UNSUPPORTED;
  FastQuantArgs a;
  a.x = x;
  a.n_vecs = n_vecs;
  a.n_inner = (uint32_t)n_inner;
  a.packed = packed;
  a.packed_outer_stride = packed_outer_stride;
  a.norms = norms;
  a.norms_outer_stride = norms_outer_stride;
  a.signs = signs;
  a.thr = thr;
#define TQ_FAST(T)                                                                   \
  return bits == 3 ? launch_fast<T, 3>(a, st) : launch_fast<T, 4>(a, st)
  switch (x_dtype) {
    case TQ_F32: TQ_FAST(float);
    case TQ_F16: TQ_FAST(__half);
    case TQ_BF16: TQ_FAST(__nv_bfloat16);
    default: return TQ_ERR_UNSUPPORTED;
  }
#undef TQ_FAST
}

}  // namespace tq
