// Softmax cross entropy of x W + b over a large vocabulary, with its gradients, in pieces of the
// vocabulary: no array of all the logits exists at any time.
//   l = x W + b, lse_m = log sum_v exp(l_mv), loss_m = lse_m - l_m,t(m)
//   d_mv = (exp(l_mv - lse_m) - [v == t(m)]) g_m,  dx = d W^T,  dW = x^T d,  db = sum_m d_m
// Forward: the product's epilogue reduces every 128 logits of a row to a maximum and a sum of
// exponentials (8 bytes instead of 512); a second kernel joins them per row. Backward: per piece of the
// vocabulary the logits are formed again, d leaves the epilogue as an fp16 pair (|d| <= 1, a fixed
// scale), and feeds the two gradient products of the piece. 8 M K V multiply-adds instead of the 6
// that kept logits would take, at 4 (M + K) bytes of work space per column of a piece.
// Large problems run on the fp16-pair tensor-core kernel (gemm_f16.cuh), small ones on the fp32 kernels.
// The reference's one loss is mse (endia/functional/loss_ops/mse_op.mojo:18-20); this is the
// classification loss beside it.
#include "gemm_f16.cuh"
#include "gemm.cuh"
#include <math.h>

using namespace eb;

namespace eb {

// state: [0] rows that count, [1] and [2] the scales' maxima of x and W (bits), [4 ...) lse per row, then
// lse log2 e per row. Inside, logits are in units of log2 e: exponentials are powers of two.
constexpr double CE_LOG2E = 1.4426950408889634, CE_LN2 = 0.6931471805599453;
constexpr int CE_STATE_HEAD = 4;
// Work space for one piece of the vocabulary (the d pair and W's pair, 4 bytes each per element).
constexpr int64_t CE_PIECE_BYTES = (int64_t)256 << 20;
constexpr int64_t CE_MIN_PIECE = 1024;
constexpr int CE_MAX_CLASSES = 1 << 24;    // class numbers are float32 values

// A class number that names no class: the row's loss and gradients become NaN.
__device__ __forceinline__ bool ce_invalid(float t, int V) { return !(t < (float)V) || t != floorf(t); }

// ------------------------------------------------------------------------------------- forward, second part
// Rows of a CTA: 32; its 16 warps take the parts of a row's (max, sum) in turn, lanes along the rows.
__global__ void __launch_bounds__(512)
ce_rows_kernel(const float2 *__restrict__ stats, int parts, const float *__restrict__ target,
               const float *__restrict__ target_logit, int M, int V, float *__restrict__ lse, float *__restrict__ lse2,
               float *__restrict__ row_loss) {
  __shared__ float2 part[16][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int m = (int)blockIdx.x * 32 + lane;
  float mx = -INFINITY, sum = 0.f;
  if (m < M) {
    for (int p0 = w; p0 < parts; p0 += 16 * 8) {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p0 + 16 * u < parts ? __ldcs(stats + (int64_t)(p0 + 16 * u) * M + m) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float nm = fmaxf(mx, v[u].x);
        if (nm > -INFINITY) sum = sum * exp2f(mx - nm) + v[u].y * exp2f(v[u].x - nm);
        else sum += v[u].y;      // (0, or NaN)
        mx = nm;
      }
    }
  }
  part[w][lane] = make_float2(mx, sum);
  __syncthreads();
  if (w == 0 && m < M) {
    for (int i = 1; i < 16; ++i) {
      const float2 v = part[i][lane];
      const float nm = fmaxf(mx, v.x);
      if (nm > -INFINITY) sum = sum * exp2f(mx - nm) + v.y * exp2f(v.x - nm);
      else sum += v.y;
      mx = nm;
    }
    const float t = __ldg(target + m);
    const double l2 = (double)mx + (double)log2f(sum);
    lse[m] = (float)(l2 * CE_LN2);
    lse2[m] = (float)l2;
    row_loss[m] = t < 0.f ? 0.f : (ce_invalid(t, V) ? NAN : (float)((l2 - (double)target_logit[m]) * CE_LN2));
  }
}

// loss[0] = sum of the rows' losses (over the number of rows that count, when mean), in a fixed order.
__global__ void __launch_bounds__(1024)
ce_loss_kernel(const float *__restrict__ row_loss, const float *__restrict__ target, int M, int mean,
               float *__restrict__ loss, float *__restrict__ count_out) {
  __shared__ float ps[32];
  __shared__ int pc[32];
  float s = 0.f;
  int c = 0;
  for (int m = threadIdx.x; m < M; m += 1024) {
    s += row_loss[m];
    c += !(target[m] < 0.f);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if ((threadIdx.x & 31) == 0) { ps[threadIdx.x >> 5] = s; pc[threadIdx.x >> 5] = c; }
  __syncthreads();
  if (threadIdx.x < 32) {
    s = ps[threadIdx.x];
    c = pc[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if (threadIdx.x == 0) {
      if (loss) loss[0] = c == 0 ? 0.f : (mean ? s / (float)c : s);
      count_out[0] = (float)c;
    }
  }
}

// ------------------------------------------------------------------------------------ backward, first part
// The incoming gradient g as a row coefficient in [-1, 1] and one factor:
//   scalar g (a sum or a mean): coef = 1, factor = g or g / count
//   one g per row: coef = g_m / 2^e with 2^e >= max |g|, factor = 2^e
// coef = 0: the row is left out; NaN: its target names no class. alpha = { factor, factor / 2^15 }.
__global__ void __launch_bounds__(1024)
ce_coef_kernel(const float *__restrict__ g, int per_row, int mean, const float *__restrict__ count,
               const float *__restrict__ target, int M, int V, float *__restrict__ coef, float *__restrict__ alpha) {
  __shared__ uint32_t pm[32];
  uint32_t best = 0;
  if (per_row) {
    for (int m = threadIdx.x; m < M; m += 1024) {
      const uint32_t b = __float_as_uint(g[m]) & 0x7FFFFFFFu;
      if (!(target[m] < 0.f) && b < 0x7F800000u && b > best) best = b;
    }
    best = __reduce_max_sync(0xffffffffu, best);
    if ((threadIdx.x & 31) == 0) pm[threadIdx.x >> 5] = best;
    __syncthreads();
    best = __reduce_max_sync(0xffffffffu, pm[threadIdx.x & 31]);
  }
  int e = best ? (int)(best >> 23) - 126 : 0;      // 2^e > max |g|
  e = e < -100 ? -100 : (e > 120 ? 120 : e);
  const float down = pow2f_exact(-e);
  for (int m = threadIdx.x; m < M; m += 1024) {
    const float t = target[m];
    coef[m] = t < 0.f ? 0.f : (ce_invalid(t, V) ? NAN : (per_row ? g[m] * down : 1.f));
  }
  if (threadIdx.x == 0) {
    const float f = per_row ? pow2f_exact(e) : (mean ? (count[0] > 0.f ? g[0] / count[0] : 0.f) : g[0]);
    alpha[0] = f;
    alpha[1] = f * (1.f / F16_D_SCALE);
  }
}

// ------------------------------------------------------------------------------------ small problems, fp32
// (max, sum) and the target's logit of one row of a piece; one CTA per row.
__global__ void __launch_bounds__(256)
ce_piece_stats_kernel(const float *__restrict__ l, int64_t ld, int N, int n_base, const float *__restrict__ target, int M,
                      float2 *__restrict__ stats, float *__restrict__ target_logit) {
  __shared__ float sh[8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int m = (int)blockIdx.x; m < M; m += (int)gridDim.x) {
    const float *row = l + (int64_t)m * ld;
    float mx = -INFINITY;
    for (int n = threadIdx.x; n < N; n += 256) mx = fmaxf(mx, row[n] * (float)CE_LOG2E);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    __syncthreads();
    if (lane == 0) sh[w] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sh[i]);
    float s = 0.f;
    for (int n = threadIdx.x; n < N; n += 256) {
      const float v = row[n] * (float)CE_LOG2E;
      s += v == -INFINITY ? 0.f : exp2f(v - mx);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (lane == 0) sh[w] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      s = 0.f;
      for (int i = 0; i < 8; ++i) s += sh[i];
      stats[m] = make_float2(mx, s);
      const float t = target[m];
      if (t >= (float)n_base && t < (float)(n_base + N)) target_logit[m] = row[(int)t - n_base] * (float)CE_LOG2E;
    }
  }
}

// logits -> d, in place (with the whole gradient factor; fp32 needs no scale).
__global__ void __launch_bounds__(256)
ce_piece_d_kernel(float *__restrict__ l, int64_t ld, int N, int n_base, const float *__restrict__ target, int M,
                  const float *__restrict__ lse, const float *__restrict__ coef, const float *__restrict__ alpha) {
  const int64_t total = (int64_t)M * N, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int m = (int)(i / N), n = (int)(i - (int64_t)m * N);
    const float c = coef[m];
    const float e = exp2f(l[(int64_t)m * ld + n] * (float)CE_LOG2E - lse[m]) - (target[m] == (float)(n_base + n) ? 1.f : 0.f);
    l[(int64_t)m * ld + n] = c == 0.f ? 0.f : e * (c * __ldg(alpha));
  }
}

// x with the rows that are left out as zeros.
__global__ void __launch_bounds__(256)
ce_rows_copy_kernel(const float *__restrict__ x, int64_t ld, const float *__restrict__ target, int M, int K, float *__restrict__ out) {
  const int64_t total = (int64_t)M * K, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t m = i / K;
    out[i] = target[m] < 0.f ? 0.f : x[m * ld + (i - m * K)];
  }
}

__global__ void __launch_bounds__(256)
ce_colsum_kernel(const float *__restrict__ d, int64_t ld, int M, int N, float *__restrict__ db) {
  const int n = (int)(blockIdx.x * blockDim.x + threadIdx.x);
  if (n >= N) return;
  float s = 0.f;
#pragma unroll 8
  for (int m = 0; m < M; ++m) s += d[(int64_t)m * ld + n];
  db[n] = s;
}

// The fp32 kernels take what is too small to fill the tensor-core kernel: few classes and few
// multiply-adds, or, without gradients, at most 8 rows (one pass over W).
static bool ce_small(int64_t M, int64_t K, int64_t V, bool backward) {
  if (!gemm_f16_available()) return true;
  if (!backward && M <= 8) return true;
  return V <= 4096 && M * K <= ((int64_t)1 << 24) / V;
}

// Columns per piece: equal pieces (multiples of 256) whose work space stays near CE_PIECE_BYTES.
static int64_t ce_piece(int64_t bytes_per_column, int64_t V) {
  int64_t most = CE_PIECE_BYTES / bytes_per_column;
  if (most < CE_MIN_PIECE) most = CE_MIN_PIECE;
  const int64_t pieces = ceil_div(V, most);
  return ceil_div(ceil_div(V, pieces), 256) * 256;
}

struct CeForward { float2 *stats; float *tl, *rows, *logits, *unused; __half *xh, *xl, *wh, *wl; int64_t piece, parts, ldx; };
static size_t ce_carve_forward(int64_t M, int64_t K, int64_t V, char *base, CeForward &f) {
  Carver c{base};
  f = CeForward{};
  f.tl = c.take<float>(M);
  f.rows = c.take<float>(M);
  if (ce_small(M, K, V, false)) {
    f.piece = ce_piece(4 * M, V);
    f.parts = ceil_div(V, f.piece);
    f.logits = c.take<float>(M * f.piece);
  } else {
    f.piece = ce_piece(4 * K, V);
    f.parts = 2 * ceil_div(V, 256);
    f.ldx = ceil_div(K, 8) * 8;
    f.xh = c.take<__half>(M * f.ldx); f.xl = c.take<__half>(M * f.ldx);
    f.wh = c.take<__half>(K * f.piece); f.wl = c.take<__half>(K * f.piece);
  }
  f.stats = c.take<float2>(M * f.parts);
  return c.used;
}

struct CeBackward { float *coef, *alpha, *partial, *part_sums, *d, *x0; uint32_t *amax; __half *xh, *xl, *wh, *wl, *dh, *dl; int64_t piece, ldx; };
static size_t ce_carve_backward(int64_t M, int64_t K, int64_t V, char *base, CeBackward &f) {
  Carver c{base};
  f = CeBackward{};
  f.coef = c.take<float>(M);
  f.alpha = c.take<float>(2);
  f.amax = c.take<uint32_t>(2);
  if (ce_small(M, K, V, true)) {
    f.piece = ce_piece(4 * M, V);
    f.d = c.take<float>(M * f.piece);
    f.x0 = c.take<float>(M * K);
  } else {
    f.piece = ce_piece(4 * (M + K), V);
    f.ldx = ceil_div(K, 8) * 8;
    f.xh = c.take<__half>(M * f.ldx); f.xl = c.take<__half>(M * f.ldx);
    f.wh = c.take<__half>(K * f.piece); f.wl = c.take<__half>(K * f.piece);
    f.dh = c.take<__half>(M * f.piece); f.dl = c.take<__half>(M * f.piece);
    f.part_sums = c.take<float>(ceil_div(M, 32) * f.piece);
    size_t a = gemm_f16_partial_bytes(M, K, f.piece), b = gemm_f16_partial_bytes(K, f.piece, M);
    const int64_t last = V - (ceil_div(V, f.piece) - 1) * f.piece;      // the last piece may be cut otherwise
    const size_t a2 = gemm_f16_partial_bytes(M, K, last), b2 = gemm_f16_partial_bytes(K, last, M);
    a = a > a2 ? a : a2; b = b > b2 ? b : b2;
    f.partial = reinterpret_cast<float *>(c.take<char>((int64_t)(a > b ? a : b)));
  }
  return c.used;
}

static int ce_check(const float *x, int64_t ldx, const float *W, int64_t ldw, const float *target, int64_t M, int64_t K,
                    int64_t V, int reduction, const void *scratch) {
  EB_REQUIRE(M >= 0 && K >= 1 && V >= 1, ENDIA_B200_EINVAL, "linear_ce: needs M >= 0, K >= 1, V >= 1");
  EB_REQUIRE(V <= CE_MAX_CLASSES, ENDIA_B200_ELIMIT, "linear_ce: at most 2^24 classes (class numbers are float32 values)");
  EB_REQUIRE(M <= (1 << 27) && K <= (1 << 27), ENDIA_B200_ELIMIT, "linear_ce: M and K must stay below 2^27");
  EB_REQUIRE(M == 0 || (x && W && target), ENDIA_B200_EINVAL, "linear_ce: NULL pointer");
  EB_REQUIRE(M == 0 || (ldx >= K && ldw >= V), ENDIA_B200_EINVAL, "linear_ce: leading dimension too small (ldx %lld, ldw %lld)",
             (long long)ldx, (long long)ldw);
  EB_REQUIRE((reinterpret_cast<uintptr_t>(scratch) & 255) == 0, ENDIA_B200_EINVAL, "linear_ce: scratch must be 256-byte aligned");
  EB_REQUIRE(reduction >= ENDIA_B200_LOSS_MEAN && reduction <= ENDIA_B200_LOSS_NONE, ENDIA_B200_EINVAL,
             "linear_ce: unknown reduction %d", reduction);
  return ENDIA_B200_OK;
}

}  // namespace eb

extern "C" {

size_t endia_b200_linear_ce_state_bytes(int64_t M) { return M < 0 ? 0 : sizeof(float) * (size_t)(CE_STATE_HEAD + 2 * M); }

size_t endia_b200_linear_ce_scratch_bytes(int64_t M, int64_t K, int64_t V, int32_t backward) {
  if (M <= 0 || K <= 0 || V <= 0 || V > CE_MAX_CLASSES || M > (1 << 27) || K > (1 << 27)) return 256;
  CeForward f;
  CeBackward b;
  return backward ? ce_carve_backward(M, K, V, nullptr, b) : ce_carve_forward(M, K, V, nullptr, f);
}

int endia_b200_linear_ce_fwd(const float *x, int64_t ldx, const float *W, int64_t ldw, const float *bias,
                             const float *target, int64_t M, int64_t K, int64_t V, int32_t reduction, float *loss,
                             float *state, void *scratch, void *stream) {
  int st = require_device();
  if (st) return st;
  if ((st = ce_check(x, ldx, W, ldw, target, M, K, V, reduction, scratch))) return st;
  EB_REQUIRE(state && scratch && (loss || (reduction == ENDIA_B200_LOSS_NONE && M == 0)), ENDIA_B200_EINVAL,
             "linear_ce: loss, state and scratch are required");
  cudaStream_t s = as_stream(stream);
  EB_CUDA(cudaMemsetAsync(state, 0, CE_STATE_HEAD * sizeof(float), s));
  if (M == 0) {
    if (reduction != ENDIA_B200_LOSS_NONE) EB_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), s));
    return ENDIA_B200_OK;
  }
  CeForward f;
  ce_carve_forward(M, K, V, static_cast<char *>(scratch), f);
  float *rows = reduction == ENDIA_B200_LOSS_NONE ? loss : f.rows;
  uint32_t *amax = reinterpret_cast<uint32_t *>(state) + 1;
  if (ce_small(M, K, V, false)) {
    for (int64_t v0 = 0, i = 0; v0 < V; v0 += f.piece, ++i) {
      const int64_t n = V - v0 < f.piece ? V - v0 : f.piece;
      if ((st = gemm_fp32(0, 0, M, n, K, x, ldx, W + v0, ldw, f.logits, f.piece, bias ? bias + v0 : nullptr, 0, 0.f, s))) return st;
      ce_piece_stats_kernel<<<(unsigned)(M < 4096 ? M : 4096), 256, 0, s>>>(f.logits, f.piece, (int)n, (int)v0, target, (int)M,
                                                                           f.stats + i * M, f.tl);
      EB_LAUNCH_CHECK();
    }
  } else {
    if ((st = launch_amax(x, M, K, ldx, target, amax, s))) return st;
    if ((st = launch_amax(W, K, V, ldw, nullptr, amax + 1, s))) return st;
    if ((st = launch_half_split(x, M, K, ldx, target, amax, f.xh, f.xl, f.ldx, s))) return st;
    for (int64_t v0 = 0; v0 < V; v0 += f.piece) {
      const int64_t n = V - v0 < f.piece ? V - v0 : f.piece;
      if ((st = launch_half_split(W + v0, K, n, ldw, nullptr, amax + 1, f.wh, f.wl, f.piece, s))) return st;
      F16Gemm g;
      g.M = M; g.N = n; g.K = K;
      g.a = HalfPair{f.xh, f.xl, f.ldx, amax};
      g.b = HalfPair{f.wh, f.wl, f.piece, amax + 1};
      g.bias = bias ? bias + v0 : nullptr;
      g.target = target; g.n_base = v0; g.stats = f.stats; g.target_logit = f.tl;
      if ((st = launch_gemm_f16(g, false, true, F16_STATS, s))) return st;
    }
  }
  ce_rows_kernel<<<(unsigned)ceil_div(M, 32), 512, 0, s>>>(f.stats, (int)f.parts, target, f.tl, (int)M, (int)V,
                                                           state + CE_STATE_HEAD, state + CE_STATE_HEAD + M, rows);
  EB_LAUNCH_CHECK();
  ce_loss_kernel<<<1, 1024, 0, s>>>(rows, target, (int)M, reduction == ENDIA_B200_LOSS_MEAN,
                                    reduction == ENDIA_B200_LOSS_NONE ? nullptr : loss, state);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

int endia_b200_linear_ce_bwd(const float *x, int64_t ldx, const float *W, int64_t ldw, const float *bias,
                             const float *target, int64_t M, int64_t K, int64_t V, int32_t reduction, const float *grad,
                             const float *state, float *dx, float *dw, float *db, void *scratch, void *stream) {
  int st = require_device();
  if (st) return st;
  if ((st = ce_check(x, ldx, W, ldw, target, M, K, V, reduction, scratch))) return st;
  EB_REQUIRE(state && scratch && (grad || M == 0), ENDIA_B200_EINVAL, "linear_ce: grad, state and scratch are required");
  if (!dx && !dw && !db) return ENDIA_B200_OK;
  cudaStream_t s = as_stream(stream);
  if (M == 0) {
    if (dw) EB_CUDA(cudaMemsetAsync(dw, 0, sizeof(float) * (size_t)K * (size_t)V, s));
    if (db) EB_CUDA(cudaMemsetAsync(db, 0, sizeof(float) * (size_t)V, s));
    return ENDIA_B200_OK;
  }
  CeBackward f;
  ce_carve_backward(M, K, V, static_cast<char *>(scratch), f);
  const float *lse = state + CE_STATE_HEAD + M;      // (in units of log2 e)
  const uint32_t *amax = reinterpret_cast<const uint32_t *>(state) + 1;
  const bool small = ce_small(M, K, V, true);
  ce_coef_kernel<<<1, 1024, 0, s>>>(grad, reduction == ENDIA_B200_LOSS_NONE, reduction == ENDIA_B200_LOSS_MEAN, state, target,
                                    (int)M, (int)V, f.coef, f.alpha);
  EB_LAUNCH_CHECK();
  if (small) {
    if (dw) {
      ce_rows_copy_kernel<<<grid_for(M * K, 256), 256, 0, s>>>(x, ldx, target, (int)M, (int)K, f.x0);
      EB_LAUNCH_CHECK();
    }
    for (int64_t v0 = 0; v0 < V; v0 += f.piece) {
      const int64_t n = V - v0 < f.piece ? V - v0 : f.piece;
      if ((st = gemm_fp32(0, 0, M, n, K, x, ldx, W + v0, ldw, f.d, f.piece, bias ? bias + v0 : nullptr, 0, 0.f, s))) return st;
      ce_piece_d_kernel<<<grid_for(M * n, 256), 256, 0, s>>>(f.d, f.piece, (int)n, (int)v0, target, (int)M, lse, f.coef, f.alpha);
      EB_LAUNCH_CHECK();
      if (dx && (st = gemm_fp32(0, 1, M, K, n, f.d, f.piece, W + v0, ldw, dx, K, nullptr, 0, v0 ? 1.f : 0.f, s))) return st;
      if (dw && (st = gemm_fp32(1, 0, K, n, M, f.x0, K, f.d, f.piece, dw + v0, V, nullptr, 0, 0.f, s))) return st;
      if (db) {
        ce_colsum_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(f.d, f.piece, (int)M, (int)n, db + v0);
        EB_LAUNCH_CHECK();
      }
    }
    return ENDIA_B200_OK;
  }
  if (ce_small(M, K, V, false)) {      // the forward pass ran in fp32 and left no scales
    EB_CUDA(cudaMemsetAsync(f.amax, 0, 2 * sizeof(uint32_t), s));
    if ((st = launch_amax(x, M, K, ldx, target, f.amax, s))) return st;
    if ((st = launch_amax(W, K, V, ldw, nullptr, f.amax + 1, s))) return st;
    amax = f.amax;
  }
  if ((st = launch_half_split(x, M, K, ldx, target, amax, f.xh, f.xl, f.ldx, s))) return st;
  for (int64_t v0 = 0; v0 < V; v0 += f.piece) {
    const int64_t n = V - v0 < f.piece ? V - v0 : f.piece;
    if ((st = launch_half_split(W + v0, K, n, ldw, nullptr, amax + 1, f.wh, f.wl, f.piece, s))) return st;
    F16Gemm g;
    g.M = M; g.N = n; g.K = K;
    g.a = HalfPair{f.xh, f.xl, f.ldx, amax};
    g.b = HalfPair{f.wh, f.wl, f.piece, amax + 1};
    g.bias = bias ? bias + v0 : nullptr;
    g.target = target; g.n_base = v0; g.lse = lse; g.coef = f.coef;
    g.d_hi = f.dh; g.d_lo = f.dl; g.ld_d = f.piece;
    g.colsum_part = db ? f.part_sums : nullptr;
    if ((st = launch_gemm_f16(g, false, true, F16_DLOGITS, s))) return st;
    const HalfPair d{f.dh, f.dl, f.piece, nullptr};
    if (dx) {      // dx += d W^T, over the pieces in order
      F16Gemm h;
      h.M = M; h.N = K; h.K = n;
      h.a = d;
      h.b = HalfPair{f.wh, f.wl, f.piece, amax + 1};
      h.alpha_dev = f.alpha + 1;
      h.C = dx; h.ldc = K; h.accumulate = v0 > 0; h.partial = f.partial;
      if ((st = launch_gemm_f16(h, false, false, F16_STORE, s))) return st;
    }
    if (dw) {
      F16Gemm h;
      h.M = K; h.N = n; h.K = M;
      h.a = HalfPair{f.xh, f.xl, f.ldx, amax};
      h.b = d;
      h.alpha_dev = f.alpha + 1;
      h.C = dw + v0; h.ldc = V; h.partial = f.partial;
      if ((st = launch_gemm_f16(h, true, true, F16_STORE, s))) return st;
    }
    if (db && (st = launch_column_sums(f.part_sums, (int)ceil_div(M, 32), n, f.alpha + 1, db + v0, s))) return st;
  }
  return ENDIA_B200_OK;
}

}  // extern "C"
