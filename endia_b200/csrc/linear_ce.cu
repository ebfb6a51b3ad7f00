// Softmax cross entropy of x W + b over a large vocabulary, with its gradients, in pieces of the
// vocabulary: no array of all the logits exists at any time.
//   l = x W + b, lse_m = log sum_v exp(l_mv), loss_m = lse_m - l_m,t(m)
//   d_mv = (exp(l_mv - lse_m) - [v == t(m)]) g_m,  dx = d W^T,  dW = x^T d,  db = sum_m d_m
// Forward: the product's epilogue reduces every 128 logits of a row to a maximum and a sum of
// exponentials (8 bytes instead of 512); a second kernel joins them per row. Backward: per piece of the
// vocabulary the logits are formed again, d leaves the epilogue as an fp16 pair (|d| <= 1, a fixed
// scale), and feeds the two gradient products of the piece. 8 M K V multiply-adds instead of the 6
// that kept logits would take, at 4 (M + K) bytes of work space per column of a piece. A step of 2048 x 1024 x
// 32768 takes 1.54 ms (265 us statistics, per piece 166 us d, 148 us dx, 157 us dW, 25 us for the pairs of W).
// The products run on the fp16-pair tensor-core kernel (gemm_f16.cuh), but that of up to 16 rows
// without a backward pass.
// The reference's one loss is mse (endia/functional/loss_ops/mse_op.mojo:18-20); this is the
// classification loss beside it.
#include "gemm_f16.cuh"
#include <math.h>

using namespace eb;

namespace eb {

// state: [0] rows that count, [1] CTAs of ce_rows_kernel that are done, [4 ...) lse per row, then lse log2 e per
// row. Inside, logits are in units of log2 e: exponentials are powers of two.
constexpr double CE_LOG2E = 1.4426950408889634, CE_LN2 = 0.6931471805599453;
constexpr int CE_STATE_HEAD = 4;
// Work space for one piece of the vocabulary (the d pair and W's pair, 4 bytes each per element). Smaller
// pieces cost rounds of tiles: 128 MiB 7 %, 64 MiB 22 % more time at 2048 x 1024 x 32768.
constexpr int64_t CE_PIECE_BYTES = (int64_t)256 << 20;
constexpr int64_t CE_MIN_PIECE = 1024;
constexpr int CE_MAX_CLASSES = 1 << 24;    // class numbers are float32 values

// A class number that names no class: the row's loss and gradients become NaN.
__device__ __forceinline__ bool ce_invalid(float t, int V) { return !(t < (float)V) || t != floorf(t); }

// ------------------------------------------------------------------------------------- forward, second part
// Joins a row's (max, sum) parts; rows of a CTA: 32, its 16 warps take the parts in turn, lanes along the
// rows. The CTA that finishes last adds up the rows' losses and the rows that count, in a fixed order.
__device__ __forceinline__ void ce_join(float &mx, float &sum, float2 v) {
  const float nm = fmaxf(mx, v.x);
  if (nm > -INFINITY) sum = sum * exp2f(mx - nm) + v.y * exp2f(v.x - nm);
  else sum += v.y;      // (0, or NaN)
  mx = nm;
}
__global__ void __launch_bounds__(512)
ce_rows_kernel(const float2 *__restrict__ stats, int parts, const float *__restrict__ target,
               const float *__restrict__ target_logit, int M, int V, float *__restrict__ state, float *row_loss,
               int mean, float *__restrict__ loss) {
  __shared__ float2 part[16][32];
  __shared__ int last;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int m = (int)blockIdx.x * 32 + lane;
  float mx = -INFINITY, sum = 0.f;
  if (m < M) {
    for (int p0 = w; p0 < parts; p0 += 16 * 8) {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p0 + 16 * u < parts ? __ldcs(stats + (int64_t)(p0 + 16 * u) * M + m) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) ce_join(mx, sum, v[u]);
    }
  }
  part[w][lane] = make_float2(mx, sum);
  __syncthreads();
  if (w == 0 && m < M) {
    for (int i = 1; i < 16; ++i) ce_join(mx, sum, part[i][lane]);
    const float t = __ldg(target + m);
    const double l2 = (double)mx + (double)log2f(sum);
    state[CE_STATE_HEAD + m] = (float)(l2 * CE_LN2);
    state[CE_STATE_HEAD + M + m] = (float)l2;
    row_loss[m] = t < 0.f ? 0.f : (ce_invalid(t, V) ? NAN : (float)((l2 - (double)target_logit[m]) * CE_LN2));
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(reinterpret_cast<unsigned int *>(state) + 1, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  float s = 0.f;
  int c = 0;
  for (int i = threadIdx.x; i < M; i += 512) {
    s += __ldcg(row_loss + i);
    c += !(__ldg(target + i) < 0.f);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if (lane == 0) part[0][w] = make_float2(s, __int_as_float(c));
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    c = 0;
    for (int i = 0; i < 16; ++i) { s += part[0][i].x; c += __float_as_int(part[0][i].y); }
    if (loss) loss[0] = c == 0 ? 0.f : (mean ? s / (float)c : s);
    state[0] = (float)c;
  }
}

// ------------------------------------------------------------------------------------ backward, first part
// The incoming gradient g as a row coefficient in [-1, 1] and one factor:
//   scalar g (a sum or a mean): coef = 1, factor = g or g / count
//   one g per row: coef = g_m / 2^e with 2^e >= max |g|, factor = 2^e
// coef = 0: the row is left out; NaN: its target names no class.
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
  e = e > 126 ? 126 : e;
  const float down = pow2f_exact(-e);
  for (int m = threadIdx.x; m < M; m += 1024) {
    const float t = target[m];
    coef[m] = t < 0.f ? 0.f : (ce_invalid(t, V) ? NAN : (per_row ? g[m] * down : 1.f));
  }
  if (threadIdx.x == 0) {
    alpha[0] = per_row ? pow2f_exact(e) : (mean ? (count[0] > 0.f ? g[0] / count[0] : 0.f) : g[0]);
  }
}

// ------------------------------------------------------------------------------------ few rows, fp32
// The statistics of up to 16 rows in one pass over W, which is all that such a call has to read: a CTA takes 128
// columns, its eight warps take the features in turn (x as [feature][row] in shared memory, four columns
// and ROWS x 4 sums a lane), and eight to sixteen loads of 128 bits a lane are in flight. The warps' sums are added in
// order, then a warp per row (two rows) reduces 128 logits as the tensor-core epilogue does. 8 rows at
// 1024 x 32768: 39 us cold (134 MB, 3.4 TB/s), against 133 us for the product of few rows of gemm_skinny.cu and its reduction.
constexpr int CE_FEW = 16, CE_FEW_K = 512;
template <int ROWS, bool VEC>
__global__ void __launch_bounds__(256)
ce_few_rows_kernel(const float *__restrict__ x, int64_t ldx, const float *__restrict__ W, int64_t ldw, const float *__restrict__ bias,
                   const float *__restrict__ target, int M, int K, int V, float2 *__restrict__ stats, float *__restrict__ target_logit) {
  __shared__ __align__(16) float xs[CE_FEW_K][ROWS];
  __shared__ float red[ROWS][128];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n0 = (int)blockIdx.x * 128;
  // this lane's four columns: consecutive, or 32 apart where rows of W are not 16-byte aligned
  int col[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) col[j] = n0 + (VEC ? 4 * lane + j : lane + 32 * j);
  float acc[ROWS][4];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[r][j] = 0.f;
  const bool inside = n0 + 128 <= V;
  for (int k0 = 0; k0 < K; k0 += CE_FEW_K) {
    const int kn = K - k0 < CE_FEW_K ? K - k0 : CE_FEW_K;
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * kn; i += 256) {
      const int r = i / kn, k = i - r * kn;
      xs[k][r] = r < M ? __ldg(x + (int64_t)r * ldx + k0 + k) : 0.f;
    }
    __syncthreads();
    // features kb, kb + 8, ... kb + 56 of this warp; the next eight are in flight while these are used
    auto load = [&](float (&v)[8][4], int kb) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int k = kb + 8 * u;
        const float *row = W + (int64_t)(k0 + k) * ldw;
        if (VEC && inside) {
          const float4 q = k < kn ? __ldcs(reinterpret_cast<const float4 *>(row + col[0])) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[u][0] = q.x; v[u][1] = q.y; v[u][2] = q.z; v[u][3] = q.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[u][j] = k < kn && col[j] < V ? __ldcs(row + col[j]) : 0.f;
        }
      }
    };
    auto use = [&](const float (&v)[8][4], int kb) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int k = kb + 8 * u;
        if (k < kn) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float xv = xs[k][r];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[r][j] = fmaf(xv, v[u][j], acc[r][j]);
          }
        }
      }
    };
    float va[8][4], vb[8][4];
    load(va, w);
    for (int kb = w; kb < kn; kb += 128) {
      load(vb, kb + 64);
      use(va, kb);
      load(va, kb + 128);
      use(vb, kb + 64);
    }
  }
  for (int src = 0; src < 8; ++src) {
    if (w == src) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[r][col[j] - n0] = src ? red[r][col[j] - n0] + acc[r][j] : acc[r][j];
    }
    __syncthreads();
  }
  for (int m = w; m < M; m += 8) {
    const float tg = __ldg(target + m);
    float l[4], mx = -INFINITY, s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + lane + 32 * j;
      l[j] = n < V ? (red[m][lane + 32 * j] + (bias ? __ldg(bias + n) : 0.f)) * (float)CE_LOG2E : -INFINITY;
      mx = fmaxf(mx, l[j]);
      if (n < V && tg == (float)n) target_logit[m] = l[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int j = 0; j < 4; ++j) s += exp2f(l[j] - base);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) stats[(int64_t)blockIdx.x * M + m] = make_float2(mx, s);
  }
}

template <int ROWS>
static int launch_few_rows(const float *x, int64_t ldx, const float *W, int64_t ldw, const float *bias, const float *target, int M,
                           int K, int V, float2 *stats, float *target_logit, cudaStream_t s) {
  const unsigned grid = (unsigned)ceil_div(V, 128);
  if (ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(W) & 15) == 0)
    ce_few_rows_kernel<ROWS, true><<<grid, 256, 0, s>>>(x, ldx, W, ldw, bias, target, M, K, V, stats, target_logit);
  else
    ce_few_rows_kernel<ROWS, false><<<grid, 256, 0, s>>>(x, ldx, W, ldw, bias, target, M, K, V, stats, target_logit);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

// Up to 16 rows a forward pass that no backward pass follows reads W once and is done (4 bytes per weight; making
// pairs first costs 16); its multiply-adds stay below the time of that read on the fp32 pipes. Where a
// backward pass follows, both take the logits from the same kernel: their common error (4e-7 of a logit,
// always towards zero) then cancels in l - lse; against an fp32 lse it stays (1.3e-6 of dx at 8 x 3584 x 640).
static bool ce_few_rows(int64_t M, bool alone) { return alone && M <= CE_FEW; }

// Columns per piece: equal pieces (multiples of 256) whose work space stays near CE_PIECE_BYTES.
static int64_t ce_piece(int64_t bytes_per_column, int64_t V) {
  int64_t most = CE_PIECE_BYTES / bytes_per_column;
  if (most < CE_MIN_PIECE) most = CE_MIN_PIECE;
  const int64_t pieces = ceil_div(V, most);
  return ceil_div(ceil_div(V, pieces), 256) * 256;
}

struct CeForward { float2 *stats; float *tl, *rows, *state; __half *xh, *xl, *wh, *wl; int *xe, *we; int64_t piece, parts, ldx; };
static size_t ce_carve_forward(int64_t M, int64_t K, int64_t V, bool alone, char *base, CeForward &f) {
  Carver c{base};
  f = CeForward{};
  f.tl = c.take<float>(M);
  f.rows = c.take<float>(M);
  if (alone) f.state = c.take<float>(CE_STATE_HEAD + 2 * M);
  if (ce_few_rows(M, alone)) {
    f.parts = ceil_div(V, 128);
  } else {
    f.piece = ce_piece(4 * K, V);
    f.parts = 2 * ceil_div(V, 256);
    f.ldx = ceil_div(K, 8) * 8;
    f.xh = c.take<__half>(M * f.ldx); f.xl = c.take<__half>(M * f.ldx);
    f.wh = c.take<__half>(K * f.piece); f.wl = c.take<__half>(K * f.piece);
    f.xe = c.take<int>(half_blocks(M) * half_blocks(K));
    f.we = c.take<int>(half_blocks(K) * half_blocks(f.piece));
  }
  f.stats = c.take<float2>(M * f.parts);
  return c.used;
}

struct CeBackward { float *coef, *alpha, *partial, *part_sums; __half *xh, *xl, *wh, *wl, *dh, *dl; int *xe, *we; int64_t piece, ldx; };
static size_t ce_carve_backward(int64_t M, int64_t K, int64_t V, char *base, CeBackward &f) {
  Carver c{base};
  f = CeBackward{};
  f.coef = c.take<float>(M);
  f.alpha = c.take<float>(1);
  f.piece = ce_piece(4 * (M + K), V);
  f.ldx = ceil_div(K, 8) * 8;
  f.xh = c.take<__half>(M * f.ldx); f.xl = c.take<__half>(M * f.ldx);
  f.wh = c.take<__half>(K * f.piece); f.wl = c.take<__half>(K * f.piece);
  f.xe = c.take<int>(half_blocks(M) * half_blocks(K));
  f.we = c.take<int>(half_blocks(K) * half_blocks(f.piece));
  f.dh = c.take<__half>(M * f.piece); f.dl = c.take<__half>(M * f.piece);
  f.part_sums = c.take<float>(ceil_div(M, 32) * f.piece);
  size_t a = gemm_f16_partial_bytes(M, K, f.piece), b = gemm_f16_partial_bytes(K, f.piece, M);
  const int64_t last = V - (ceil_div(V, f.piece) - 1) * f.piece;      // the last piece may be cut otherwise
  const size_t a2 = gemm_f16_partial_bytes(M, K, last), b2 = gemm_f16_partial_bytes(K, last, M);
  a = a > a2 ? a : a2; b = b > b2 ? b : b2;
  f.partial = reinterpret_cast<float *>(c.take<char>((int64_t)(a > b ? a : b)));
  return c.used;
}

// The passes over a piece of W (the caller sets its columns) and, with the first one, over x.
template <typename F>
static void ce_jobs(HalfJob (&jobs)[2], const float *x, int64_t ldx, const float *W, int64_t ldw, const float *target, int64_t M,
                    int64_t K, const F &f) {
  HalfJob &jw = jobs[0], &jx = jobs[1];
  jw.rows = K; jw.x = W; jw.ld = ldw; jw.hi = f.wh; jw.lo = f.wl; jw.ld_out = f.piece; jw.e = f.we;
  jx.rows = M; jx.cols = K; jx.x = x; jx.ld = ldx; jx.target = target; jx.hi = f.xh; jx.lo = f.xl; jx.ld_out = f.ldx; jx.e = f.xe;
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

size_t endia_b200_linear_ce_scratch_bytes(int64_t M, int64_t K, int64_t V, int32_t pass) {
  if (M <= 0 || K <= 0 || V <= 0 || V > CE_MAX_CLASSES || M > (1 << 27) || K > (1 << 27)) return 256;
  CeForward f;
  CeBackward b;
  return pass == 1 ? ce_carve_backward(M, K, V, nullptr, b) : ce_carve_forward(M, K, V, pass == 2, nullptr, f);
}

int endia_b200_linear_ce_fwd(const float *x, int64_t ldx, const float *W, int64_t ldw, const float *bias,
                             const float *target, int64_t M, int64_t K, int64_t V, int32_t reduction, float *loss,
                             float *state, void *scratch, void *stream) {
  int st = require_device();
  if (st) return st;
  if ((st = ce_check(x, ldx, W, ldw, target, M, K, V, reduction, scratch))) return st;
  EB_REQUIRE(scratch && (loss || (reduction == ENDIA_B200_LOSS_NONE && M == 0)), ENDIA_B200_EINVAL,
             "linear_ce: loss and scratch are required");
  cudaStream_t s = as_stream(stream);
  const bool alone = state == nullptr;
  CeForward f;
  ce_carve_forward(M, K, V, alone, static_cast<char *>(scratch), f);
  if (alone) state = f.state;
  if (M == 0) {
    if (!alone) EB_CUDA(cudaMemsetAsync(state, 0, CE_STATE_HEAD * sizeof(float), s));
    if (reduction != ENDIA_B200_LOSS_NONE) EB_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), s));
    return ENDIA_B200_OK;
  }
  EB_CUDA(cudaMemsetAsync(state, 0, CE_STATE_HEAD * sizeof(float), s));
  float *rows = reduction == ENDIA_B200_LOSS_NONE ? loss : f.rows;
  if (ce_few_rows(M, alone)) {
    const auto few = M <= 1 ? launch_few_rows<1> : M <= 2 ? launch_few_rows<2> : M <= 4 ? launch_few_rows<4>
                     : M <= 8 ? launch_few_rows<8> : launch_few_rows<CE_FEW>;
    if ((st = few(x, ldx, W, ldw, bias, target, (int)M, (int)K, (int)V, f.stats, f.tl, s))) return st;
  } else {
    HalfJob jobs[2];
    ce_jobs(jobs, x, ldx, W, ldw, target, M, K, f);
    for (int64_t v0 = 0; v0 < V; v0 += f.piece) {
      const int64_t n = V - v0 < f.piece ? V - v0 : f.piece;
      jobs[0].x = W + v0; jobs[0].cols = n;
      if ((st = launch_half_split(jobs, v0 ? 1 : 2, s))) return st;
      F16Gemm g;
      g.M = M; g.N = n; g.K = K;
      g.a = HalfPair{f.xh, f.xl, f.ldx, f.xe, half_blocks(K)};
      g.b = HalfPair{f.wh, f.wl, f.piece, f.we, half_blocks(n)};
      g.bias = bias ? bias + v0 : nullptr;
      g.target = target; g.n_base = v0; g.stats = f.stats; g.target_logit = f.tl;
      if ((st = launch_gemm_f16(g, false, true, F16_STATS, s))) return st;
    }
  }
  ce_rows_kernel<<<(unsigned)ceil_div(M, 32), 512, 0, s>>>(f.stats, (int)f.parts, target, f.tl, (int)M, (int)V, state, rows,
                                                           reduction == ENDIA_B200_LOSS_MEAN,
                                                           reduction == ENDIA_B200_LOSS_NONE ? nullptr : loss);
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
  ce_coef_kernel<<<1, 1024, 0, s>>>(grad, reduction == ENDIA_B200_LOSS_NONE, reduction == ENDIA_B200_LOSS_MEAN, state, target,
                                    (int)M, (int)V, f.coef, f.alpha);
  EB_LAUNCH_CHECK();
  HalfJob jobs[2];
  ce_jobs(jobs, x, ldx, W, ldw, target, M, K, f);
  for (int64_t v0 = 0; v0 < V; v0 += f.piece) {
    const int64_t n = V - v0 < f.piece ? V - v0 : f.piece;
    jobs[0].x = W + v0; jobs[0].cols = n;
    if ((st = launch_half_split(jobs, v0 ? 1 : 2, s))) return st;
    F16Gemm g;
    g.M = M; g.N = n; g.K = K;
    g.a = HalfPair{f.xh, f.xl, f.ldx, f.xe, half_blocks(K)};
    g.b = HalfPair{f.wh, f.wl, f.piece, f.we, half_blocks(n)};
    g.bias = bias ? bias + v0 : nullptr;
    g.target = target; g.n_base = v0; g.lse = lse; g.coef = f.coef;
    g.d_hi = f.dh; g.d_lo = f.dl; g.ld_d = f.piece;
    g.colsum_part = db ? f.part_sums : nullptr;
    if ((st = launch_gemm_f16(g, false, true, F16_DLOGITS, s))) return st;
    const HalfPair d{f.dh, f.dl, f.piece, nullptr, 0};
    if (dx) {      // dx += d W^T, over the pieces in order
      F16Gemm h;
      h.M = M; h.N = K; h.K = n;
      h.a = d;
      h.b = HalfPair{f.wh, f.wl, f.piece, f.we, half_blocks(n)};
      h.alpha_dev = f.alpha; h.alpha_exp = -F16_D_EXP;
      h.C = dx; h.ldc = K; h.accumulate = v0 > 0; h.partial = f.partial;
      if ((st = launch_gemm_f16(h, false, false, F16_STORE, s))) return st;
    }
    if (dw) {
      F16Gemm h;
      h.M = K; h.N = n; h.K = M;
      h.a = HalfPair{f.xh, f.xl, f.ldx, f.xe, half_blocks(K)};
      h.b = d;
      h.alpha_dev = f.alpha; h.alpha_exp = -F16_D_EXP;
      h.C = dw + v0; h.ldc = V; h.partial = f.partial;
      if ((st = launch_gemm_f16(h, true, true, F16_STORE, s))) return st;
    }
    if (db && (st = launch_column_sums(f.part_sums, (int)ceil_div(M, 32), n, 1.f / F16_D_SCALE, f.alpha, db + v0, s))) return st;
  }
  return ENDIA_B200_OK;
}

}  // extern "C"
