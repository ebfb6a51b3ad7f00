// Activations held in 8 bits for the backward pass, and the linear layer that uses them.
//
// Form: per row, blocks of 32 consecutive features share a power-of-two scale:
//   x ~ q * 2^e,  e the smallest integer with round(max|x| / 2^e) <= 127,  q = round(x / 2^e) in [-127, 127]
// (round half to even; -126 <= e <= 121, so that q * 2^e is finite: values beyond 127 * 2^121 become that). 8.25 bits per value, an error of at most half of 2^e, which is between
// max/127.5/2 and max/63.75/2. With keep_sign a value that is not zero gets |q| >= 1, so that the
// derivative of a ReLU taken from its kept output is the exact one. An infinite or NaN value is kept as
// q = -128 and reads back as NaN; it does not count in the block's maximum.
// Why a power of two: x / 2^e and q * 2^e are exact in fp32, and q * 2^e is exact in fp16 after one scale
// for the whole array, so the weight gradient h^T ds needs two fp16 products instead of three.
// Layout: q [rows][cols rounded up to 32], e + 127 [rows][cols / 32 rounded up] as bytes.
//
// The layer: out = act(x W + b) from x itself; for its backward pass only the kept forms are read:
//   ds = g act'(out),  dx = ds W^T,  dW = x8^T ds,  db = sum over the rows of ds.
// Two passes over memory (one per direction, half_split_kernel) and three products; a layer of 8192 x 4096 x 4096
// with mse above and a ReLU below takes 2.14 ms, of which the products are 1.53 (power-bound).
// Replaces, for such a layer, the products of matmul_vjp and the masks of relu/tanh/sigmoid
// (endia/functional/binary_ops/matmul_op.mojo:278-284, relu_op.mojo:95, tanh_op.mojo:92, sigmoid_op.mojo:98).
#include "gemm_f16.cuh"

using namespace eb;

namespace eb {

// Eight consecutive kept values of row r from column c (a multiple of 8).
__device__ __forceinline__ void kept8(const Kept &k, int64_t r, int64_t c, float (&v)[8]) {
  const uint2 w = __ldg(reinterpret_cast<const uint2 *>(k.q + r * k.ldq + c));
  const float unit = pow2f_exact((int)__ldg(k.e + r * k.lde + c / 32) - 127);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int n = (int)(int8_t)(((u < 4 ? w.x : w.y) >> (8 * (u & 3))) & 0xFFu);
    v[u] = n == -128 ? NAN : (float)n * unit;
  }
}

__global__ void __launch_bounds__(256)
kept_read_kernel(Kept k, int64_t rows, int64_t cols, float *__restrict__ out) {
  const int64_t per_row = k.ldq / 8, total = rows * per_row, step = (int64_t)gridDim.x * blockDim.x;
  const bool vec = cols % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    float v[8];
    kept8(k, r, c, v);
    float *dst = out + r * cols + c;
    if (vec && c + 8 <= cols) {
      reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) if (c + u < cols) dst[u] = v[u];
    }
  }
}

struct KeepForward { __half *xh, *xl, *wh, *wl; int *xe, *we; float *partial; int64_t ldx, ldw; };
static size_t keep_carve_forward(int64_t M, int64_t N, int64_t K, char *base, KeepForward &f) {
  Carver c{base};
  f = KeepForward{};
  f.ldx = ceil_div(K, 8) * 8; f.ldw = ceil_div(N, 8) * 8;
  f.xh = c.take<__half>(M * f.ldx); f.xl = c.take<__half>(M * f.ldx);
  f.wh = c.take<__half>(K * f.ldw); f.wl = c.take<__half>(K * f.ldw);
  f.xe = c.take<int>(half_blocks(M) * half_blocks(K));
  f.we = c.take<int>(half_blocks(K) * half_blocks(N));
  f.partial = reinterpret_cast<float *>(c.take<char>((int64_t)gemm_f16_partial_bytes(M, N, K)));
  return c.used;
}
struct KeepBackward { __half *dh, *dl, *wh, *wl, *x8; int *de, *we, *xe; float *partial, *sums; int64_t ldd, ldw, ldx; };
static size_t keep_carve_backward(int64_t M, int64_t N, int64_t K, char *base, KeepBackward &f) {
  Carver c{base};
  f = KeepBackward{};
  f.sums = c.take<float>(half_blocks(M) * N);
  f.ldd = f.ldw = ceil_div(N, 8) * 8;
  f.ldx = ceil_div(K, 8) * 8;
  f.dh = c.take<__half>(M * f.ldd); f.dl = c.take<__half>(M * f.ldd);
  f.wh = c.take<__half>(K * f.ldw); f.wl = c.take<__half>(K * f.ldw);
  f.x8 = c.take<__half>(M * f.ldx);
  f.de = c.take<int>(half_blocks(M) * half_blocks(N));
  f.we = c.take<int>(half_blocks(K) * half_blocks(N));
  f.xe = c.take<int>(half_blocks(M) * half_blocks(K));
  const size_t a = gemm_f16_partial_bytes(M, K, N), b = gemm_f16_partial_bytes(K, N, M);
  f.partial = reinterpret_cast<float *>(c.take<char>((int64_t)(a > b ? a : b)));
  return c.used;
}

static int keep_check(const char *what, int64_t M, int64_t N, int64_t K, int act, const void *scratch) {
  EB_REQUIRE(M >= 0 && N >= 0 && K >= 0, ENDIA_B200_EINVAL, "%s: negative size", what);
  EB_REQUIRE(M <= (1 << 27) && N <= (1 << 27) && K <= (1 << 27), ENDIA_B200_ELIMIT, "%s: sizes must stay below 2^27", what);
  EB_REQUIRE(act >= 0 && act <= ENDIA_B200_ACT_SIGMOID, ENDIA_B200_EINVAL, "%s: unknown activation %d", what, act);
  EB_REQUIRE(scratch && (reinterpret_cast<uintptr_t>(scratch) & 255) == 0, ENDIA_B200_EINVAL,
             "%s: scratch must be given, 256-byte aligned", what);
  return ENDIA_B200_OK;
}

// The 8-bit form of x as a part of the pass over it.
static HalfJob keep_job(const float *x, int64_t ld, int64_t rows, int64_t cols, int keep_sign, void *kept) {
  HalfJob j;
  j.rows = rows; j.cols = cols; j.x = x; j.ld = ld;
  if (kept) j.keep = kept_view(kept, rows, cols);
  j.keep_sign = keep_sign;
  return j;
}

}  // namespace eb

extern "C" {

size_t endia_b200_keep8_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return 0;
  const size_t ldq = ((size_t)cols + 31) / 32 * 32;
  return ((size_t)rows * (ldq + ldq / 32) + 255) / 256 * 256;
}

int endia_b200_keep8(const float *x, int64_t ldx, int64_t rows, int64_t cols, int32_t keep_sign, void *kept, void *stream) {
  int st = require_device();
  if (st) return st;
  EB_REQUIRE(rows >= 0 && cols >= 0, ENDIA_B200_EINVAL, "keep8: negative size");
  EB_REQUIRE(kept && (reinterpret_cast<uintptr_t>(kept) & 255) == 0, ENDIA_B200_EINVAL, "keep8: kept must be given, 256-byte aligned");
  EB_REQUIRE(rows == 0 || cols == 0 || (x && ldx >= cols), ENDIA_B200_EINVAL, "keep8: NULL input or leading dimension too small");
  const HalfJob j = keep_job(x, ldx, rows, cols, keep_sign, kept);
  return launch_half_split(&j, 1, as_stream(stream));
}

int endia_b200_keep8_read(const void *kept, int64_t rows, int64_t cols, float *out, void *stream) {
  int st = require_device();
  if (st) return st;
  EB_REQUIRE(rows >= 0 && cols >= 0, ENDIA_B200_EINVAL, "keep8_read: negative size");
  if (rows == 0 || cols == 0) return ENDIA_B200_OK;
  EB_REQUIRE(kept && out, ENDIA_B200_EINVAL, "keep8_read: NULL pointer");
  const Kept k = kept_view(const_cast<void *>(kept), rows, cols);
  kept_read_kernel<<<grid_for(rows * (k.ldq / 8), 256, 8), 256, 0, as_stream(stream)>>>(k, rows, cols, out);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

size_t endia_b200_linear_keep_scratch_bytes(int64_t M, int64_t N, int64_t K, int32_t backward) {
  if (M < 0 || N < 0 || K < 0 || M > (1 << 27) || N > (1 << 27) || K > (1 << 27)) return 256;
  if (M == 0 || N == 0 || K == 0) return 256;
  KeepForward f;
  KeepBackward b;
  return backward ? keep_carve_backward(M, N, K, nullptr, b) : keep_carve_forward(M, N, K, nullptr, f);
}

int endia_b200_linear_keep_fwd(const float *x, int64_t ldx, const float *W, int64_t ldw, const float *bias, int32_t act,
                               int64_t M, int64_t N, int64_t K, float *out, void *kept_x, int32_t keep_sign,
                               void *scratch, void *stream) {
  int st = require_device();
  if (st) return st;
  if ((st = keep_check("linear_keep", M, N, K, act, scratch))) return st;
  EB_REQUIRE(K >= 1, ENDIA_B200_EINVAL, "linear_keep: needs at least one input feature");
  EB_REQUIRE(!kept_x || (reinterpret_cast<uintptr_t>(kept_x) & 255) == 0, ENDIA_B200_EINVAL, "linear_keep: kept_x must be 256-byte aligned");
  cudaStream_t s = as_stream(stream);
  if (M == 0) return ENDIA_B200_OK;
  EB_REQUIRE(x && ldx >= K && (N == 0 || (W && out && ldw >= N)), ENDIA_B200_EINVAL, "linear_keep: NULL pointer or leading dimension too small");
  KeepForward f;
  keep_carve_forward(M, N, K, static_cast<char *>(scratch), f);
  HalfJob jobs[2] = {keep_job(x, ldx, M, K, keep_sign, kept_x), HalfJob{}};
  if (N == 0) return kept_x ? launch_half_split(jobs, 1, s) : ENDIA_B200_OK;
  HalfJob &jx = jobs[0], &jw = jobs[1];
  jx.hi = f.xh; jx.lo = f.xl; jx.ld_out = f.ldx; jx.e = f.xe;
  jw.rows = K; jw.cols = N; jw.x = W; jw.ld = ldw; jw.hi = f.wh; jw.lo = f.wl; jw.ld_out = f.ldw; jw.e = f.we;
  if ((st = launch_half_split(jobs, 2, s))) return st;
  F16Gemm g;
  g.M = M; g.N = N; g.K = K;
  g.a = HalfPair{f.xh, f.xl, f.ldx, f.xe, half_blocks(K)};
  g.b = HalfPair{f.wh, f.wl, f.ldw, f.we, half_blocks(N)};
  g.bias = bias; g.act = act; g.C = out; g.ldc = N; g.partial = f.partial;
  return launch_gemm_f16(g, false, true, F16_STORE, s);
}

int endia_b200_linear_keep_bwd(const void *kept_x, const float *W, int64_t ldw, const float *out, const void *kept_out,
                               int32_t act, const float *grad, int64_t M, int64_t N, int64_t K, float *dx, float *dw,
                               float *db, void *scratch, void *stream) {
  int st = require_device();
  if (st) return st;
  if ((st = keep_check("linear_keep", M, N, K, act, scratch))) return st;
  EB_REQUIRE(K >= 1, ENDIA_B200_EINVAL, "linear_keep: needs at least one input feature");
  cudaStream_t s = as_stream(stream);
  if (M == 0 || N == 0) {
    if (dx && M) EB_CUDA(cudaMemsetAsync(dx, 0, sizeof(float) * (size_t)M * (size_t)K, s));
    if (dw && N) EB_CUDA(cudaMemsetAsync(dw, 0, sizeof(float) * (size_t)K * (size_t)N, s));
    if (db && N) EB_CUDA(cudaMemsetAsync(db, 0, sizeof(float) * (size_t)N, s));
    return ENDIA_B200_OK;
  }
  if (!dx && !dw && !db) return ENDIA_B200_OK;
  EB_REQUIRE(grad && (!dw || kept_x) && (!dx || (W && ldw >= N)) && (act == 0 || out || kept_out), ENDIA_B200_EINVAL,
             "linear_keep: NULL pointer or leading dimension too small");
  KeepBackward f;
  keep_carve_backward(M, N, K, static_cast<char *>(scratch), f);
  // one pass over the incoming gradient (ds and its column sums), the kept input and W
  HalfJob jobs[3];
  int n = 1;
  HalfJob &jd = jobs[0];
  jd.rows = M; jd.cols = N; jd.x = grad; jd.ld = N; jd.act = act;
  if (act) {
    jd.out = out;
    if (!out) jd.out_kept = kept_view(const_cast<void *>(kept_out), M, N);
  }
  if (dx || dw) { jd.hi = f.dh; jd.lo = f.dl; jd.ld_out = f.ldd; jd.e = f.de; }
  if (db) jd.sums = f.sums;
  if (dw) {
    HalfJob &jx = jobs[n++];
    jx.rows = M; jx.cols = K; jx.kept = kept_view(const_cast<void *>(kept_x), M, K);
    jx.hi = f.x8; jx.ld_out = f.ldx; jx.e = f.xe;      // (exact in hi: q has 7 bits)
  }
  if (dx) {
    HalfJob &jw = jobs[n++];
    jw.rows = K; jw.cols = N; jw.x = W; jw.ld = ldw; jw.hi = f.wh; jw.lo = f.wl; jw.ld_out = f.ldw; jw.e = f.we;
  }
  if ((st = launch_half_split(jobs, n, s))) return st;
  if (db && (st = launch_column_sums(f.sums, (int)half_blocks(M), N, 1.f, nullptr, db, s))) return st;
  const HalfPair d{f.dh, f.dl, f.ldd, f.de, half_blocks(N)};
  if (dw) {
    F16Gemm g;
    g.M = K; g.N = N; g.K = M;
    g.a = HalfPair{f.x8, nullptr, f.ldx, f.xe, half_blocks(K)};
    g.b = d;
    g.C = dw; g.ldc = N; g.partial = f.partial;
    if ((st = launch_gemm_f16(g, true, true, F16_STORE, s))) return st;
  }
  if (dx) {
    F16Gemm g;
    g.M = M; g.N = K; g.K = N;
    g.a = d;
    g.b = HalfPair{f.wh, f.wl, f.ldw, f.we, half_blocks(N)};
    g.C = dx; g.ldc = K; g.partial = f.partial;
    if ((st = launch_gemm_f16(g, false, false, F16_STORE, s))) return st;
  }
  return ENDIA_B200_OK;
}

}  // extern "C"
