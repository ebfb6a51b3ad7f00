// fp32-accurate matrix products from fp16 pairs on the tensor cores (gemm_f16.cu), the engine of the
// cross entropy over a large vocabulary and of the layers checkpointed in 8 bits.
//   x * s = hi + lo,  hi = fp16(x * s), lo = fp16(x * s - hi),  s a power of two per block of 128 x 128
//   elements that puts the block's largest finite |x| into [2^14, 2^15)
// hi and lo hold 22 bits of every element down to 2^-15 of the largest one of its block; smaller ones are
// exact to 2^-40 of it.  a*b = a_hi*b_hi + a_lo*b_hi + a_hi*b_lo (+ a_lo*b_lo, 2^-24 of the product, dropped).
// The blocks' scales come out again where the accumulators are added in fp32: a run of 64 or 128 of K lies in one
// block of each operand, and a tile's sums are held in units of its largest product of unscaling factors (what
// lies 2^-126 below that drops out). A scale per array would need the array's maximum first, one more pass.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace eb {

constexpr int HALF_BLOCK = 128;

// An operand laid out row-major with leading dimension ld (a multiple of 8), 16-byte aligned.
struct HalfPair {
  const __half *hi = nullptr;
  const __half *lo = nullptr;       // NULL: the operand is exact in hi
  int64_t ld = 0;
  const int *e = nullptr;           // scale exponents [row blocks][e_ld] (s = 2^e); NULL: 1
  int64_t e_ld = 0;
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
  const float *alpha_dev = nullptr;   // F16_STORE: optional device scalar multiplied into v, and 2^alpha_exp
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

// The 8-bit form of an activation (keep8.cu): q [rows][cols rounded up to 32], then e + 127 [rows][ldq / 32].
struct Kept {
  int8_t *q = nullptr;
  uint8_t *e = nullptr;
  int64_t ldq = 0, lde = 0;
};
__host__ __device__ inline Kept kept_view(void *p, int64_t rows, int64_t cols) {
  Kept k;
  k.ldq = (cols + 31) / 32 * 32;
  k.lde = k.ldq / 32;
  k.q = static_cast<int8_t *>(p);
  k.e = static_cast<uint8_t *>(p) + rows * k.ldq;
  return k;
}

// One array of the pass that makes operands: read once, block by block.
struct HalfJob {
  int64_t rows = 0, cols = 0;
  const float *x = nullptr;          // [rows][ld], or NULL: `kept`
  int64_t ld = 0;
  Kept kept;
  const float *target = nullptr;     // [rows], optional: rows with target < 0 read as zero
  int act = 0;                       // != 0: x times act'(out), out contiguous fp32, or NULL: `out_kept`
  const float *out = nullptr;
  Kept out_kept;
  __half *hi = nullptr, *lo = nullptr;   // the pair (hi NULL: none; lo NULL: exact in hi)
  int64_t ld_out = 0;
  int *e = nullptr;                  // the blocks' scale exponents, [ceil(rows / 128)][ceil(cols / 128)]
  Kept keep;                         // q != NULL: the 8-bit form is written too
  int keep_sign = 0;
  float *sums = nullptr;             // optional: [ceil(rows / 128)][cols] sums over 128 rows
};
inline int64_t half_blocks(int64_t n) { return ceil_div(n, HALF_BLOCK); }
// Up to three arrays in one launch.
int launch_half_split(const HalfJob *jobs, int n, cudaStream_t s);

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

// Scale exponent of a block from its largest finite |x|: 14 - floor(log2 amax), at most 126 (a block of
// values below 2^-112 keeps fewer than 22 bits, down to those of a denormal). A block of zeros has 126: it must
// not set the unit of a tile whose other blocks are tiny.
__host__ __device__ __forceinline__ int half_scale_exponent(uint32_t amax_bits) {
  const int ex = 141 - (int)(amax_bits >> 23);
  return ex > 126 ? 126 : ex;
}
__device__ __forceinline__ float pow2f_exact(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }   // -126 <= e <= 127

// alpha (optional device scalar) times 2^extra as two factors of about the same exponent, so that (v * f0) * f1
// leaves the range of fp32 only where the result does.
__device__ __forceinline__ void alpha_factors(const float *alpha, int extra, float &f0, float &f1) {
  int e = extra;
  float m = 1.f;
  if (alpha) {
    m = *alpha;
    const int field = (int)(__float_as_uint(m) >> 23) & 0xFF;
    if (field != 0 && field != 0xFF) {      // (zero, denormal, infinite or NaN: the value itself)
      e += field - 127;
      m = __uint_as_float((__float_as_uint(m) & 0x807FFFFFu) | 0x3F800000u);
    }
  }
  const int e0 = max(-126, min(126, e / 2)), e1 = max(-126, min(127, e - e0));
  f0 = m * pow2f_exact(e0);
  f1 = pow2f_exact(e1);
}

// hi and lo of a scaled value. An infinite or NaN value gives an infinite or NaN hi and a NaN lo.
__device__ __forceinline__ void half_pair(float v, __half &hi, __half &lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

}  // namespace eb
