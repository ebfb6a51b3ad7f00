// fp32-accurate matrix products from fp16 pairs on the tensor cores (gemm_f16.cu), the engine of the
// cross entropy over a large vocabulary and of the layers checkpointed in 8 bits.
//   x * s = hi + lo,  hi = fp16(x * s), lo = fp16(x * s - hi),  s a power of two from the largest
//   finite |x| of the operand so that it lands in [2^14, 2^15)
// hi and lo hold 22 bits of every element down to 2^-15 of the largest one; smaller ones are exact to
// 2^-40 of it.  a*b = a_hi*b_hi + a_lo*b_hi + a_hi*b_lo (+ a_lo*b_lo, 2^-24 of the product, dropped).
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace eb {

// An operand laid out row-major with leading dimension ld (a multiple of 8), 16-byte aligned.
struct HalfPair {
  const __half *hi = nullptr;
  const __half *lo = nullptr;       // NULL: the operand is exact in hi
  int64_t ld = 0;
  const uint32_t *amax = nullptr;   // device: bits of the largest finite |x| (the scale s follows from it); NULL: s = 1
};

enum F16Epilogue {
  F16_STORE = 0,     // C = act(v + bias) or C += v
  F16_STATS = 1,     // per row and 128 columns: (max, sum of 2^(l - max)) of l = (v + bias) log2 e; the target's l
  F16_DLOGITS = 2    // d = (2^((v + bias) log2 e - lse) - [column == target]) * coef, stored as an fp16 pair scaled by 2^15
};
constexpr int F16_D_EXP = 15;
constexpr float F16_D_SCALE = 32768.f;      // 2^F16_D_EXP

struct F16Gemm {
  int64_t M = 0, N = 0, K = 0;
  HalfPair a, b;
  const float *alpha_dev = nullptr;   // optional device scalar multiplied into v, and 2^alpha_exp
  int alpha_exp = 0;
  const float *bias = nullptr;        // [N]
  // F16_STORE
  float *C = nullptr;
  int64_t ldc = 0;
  int act = 0;
  bool accumulate = false;            // C += v (no bias, no act)
  float *partial = nullptr;           // work space of gemm_f16_partial_bytes(M, N, K) bytes
  // F16_STATS and F16_DLOGITS
  const float *target = nullptr;      // [M] class numbers; this product's columns are classes n_base ...
  int64_t n_base = 0;                 // (a multiple of 256)
  float2 *stats = nullptr;            // F16_STATS: [2 * ceil(V / 256)][M] (max, sum)
  float *target_logit = nullptr;      // F16_STATS: [M], in units of log2 e too
  const float *lse = nullptr, *coef = nullptr;   // F16_DLOGITS: [M]; lse in units of log2 e
  __half *d_hi = nullptr, *d_lo = nullptr;       // F16_DLOGITS: [M][ld_d]
  int64_t ld_d = 0;
  float *colsum_part = nullptr;       // F16_DLOGITS, optional: [ceil(M / 32)][N] sums over 32 rows of d (times 2^15)
};

// C[M, N] = A B: a_mn = false: A is stored [M, K]; true: [K, M].  b_mn = true: B is stored [K, N]; false: [N, K].
int launch_gemm_f16(const F16Gemm &g, bool a_mn, bool b_mn, int epilogue, cudaStream_t s);
// Work space of an F16_STORE product (0 when its reduction is not cut into ranges).
size_t gemm_f16_partial_bytes(int64_t M, int64_t N, int64_t K);
bool gemm_f16_available();

// One fp32 array of the passes below: [rows, cols], leading dimension ld. `target` (optional, [rows]):
// rows with target < 0 do not count in the maximum and become zero in the pair.
struct HalfJob {
  const float *x = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
  const float *target = nullptr;
  uint32_t *amax = nullptr;      // bits of the largest finite |x|
  __half *hi = nullptr, *lo = nullptr;
  int64_t ld_out = 0;
};
// amax[0] = max(amax[0], bits of the largest finite |x|) of up to two arrays in one launch; *amax starts at 0.
int launch_amax(const HalfJob &a, const HalfJob *b, cudaStream_t s);
// The fp16 pairs of up to two arrays in one launch.
int launch_half_split(const HalfJob &a, const HalfJob *b, cudaStream_t s);

// out[n] = the sum of the rows of part [parts][N], in a fixed order, times scale, times alpha (a device scalar, NULL: 1).
int launch_column_sums(const float *part, int parts, int64_t N, float scale, const float *alpha, float *out, cudaStream_t s);

struct Carver {       // a caller's work space, handed out in 256-byte steps (base NULL: only measures)
  char *base;
  size_t used = 0;
  template <typename T> T *take(int64_t n) {
    T *p = reinterpret_cast<T *>(base + used);
    used += ((size_t)n * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

// Scale of an operand from its largest finite |x|: 2^(14 - floor(log2 amax)), at most 2^126 (an operand of
// values below 2^-112 keeps fewer than 22 bits, down to those of a denormal), and its inverse.
__host__ __device__ __forceinline__ int half_scale_exponent(uint32_t amax_bits) {
  if (amax_bits == 0) return 0;
  const int ex = 141 - (int)(amax_bits >> 23);
  return ex > 126 ? 126 : ex;
}
__device__ __forceinline__ float pow2f_exact(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float half_scale(const uint32_t *amax) { return amax ? pow2f_exact(half_scale_exponent(*amax)) : 1.f; }

// A sum of scaled products is (sum * f0) * f1: the operands' unscaling, `alpha` (optional device scalar) and
// 2^extra as two factors of about the same exponent, so that neither step leaves the range of fp32 unless
// the result does.
__device__ __forceinline__ void unscale_factors(const uint32_t *amax_a, const uint32_t *amax_b, const float *alpha, int extra,
                                                float &f0, float &f1) {
  int e = extra - (amax_a ? half_scale_exponent(*amax_a) : 0) - (amax_b ? half_scale_exponent(*amax_b) : 0);
  float m = 1.f;
  if (alpha) {
    m = *alpha;
    const int field = (int)(__float_as_uint(m) >> 23) & 0xFF;
    if (field != 0 && field != 0xFF) {      // (zero, denormal, infinite or NaN: the value itself)
      e += field - 127;
      m = __uint_as_float((__float_as_uint(m) & 0x807FFFFFu) | 0x3F800000u);
    }
  }
  const int e0 = e / 2, e1 = e - e0;
  f0 = m * pow2f_exact(e0 < -126 ? -126 : (e0 > 126 ? 126 : e0));
  f1 = pow2f_exact(e1 < -126 ? -126 : (e1 > 127 ? 127 : e1));
}

// hi and lo of a scaled value. An infinite or NaN value gives an infinite or NaN hi and a NaN lo.
__device__ __forceinline__ void half_pair(float v, __half &hi, __half &lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

}  // namespace eb
