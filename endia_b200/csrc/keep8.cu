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
// Layout: a head of 256 bytes ([0]: bits of the largest finite |x|, [1]: scratch of the layer), q [rows][cols rounded up to 32],
// e + 127 [rows][cols / 32 rounded up] as bytes.
//
// The layer: out = act(x W + b) from x itself; for its backward pass only the kept forms are read:
//   ds = g act'(out),  dx = ds W^T,  dW = x8^T ds,  db = sum over the rows of ds.
// Replaces, for such a layer, the products of matmul_vjp and the masks of relu/tanh/sigmoid
// (endia/functional/binary_ops/matmul_op.mojo:278-284, relu_op.mojo:95, tanh_op.mojo:92, sigmoid_op.mojo:98).
#include "gemm_f16.cuh"
#include "gemm.cuh"

using namespace eb;

namespace eb {

struct Kept {
  uint32_t *amax;
  int8_t *q;
  uint8_t *e;
  int64_t ldq, lde;
};
__host__ __device__ static inline Kept kept_view(void *p, int64_t rows, int64_t cols) {
  Kept k;
  char *c = static_cast<char *>(p);
  k.ldq = (cols + 31) / 32 * 32;
  k.lde = k.ldq / 32;
  k.amax = reinterpret_cast<uint32_t *>(c);
  k.q = reinterpret_cast<int8_t *>(c + 256);
  k.e = reinterpret_cast<uint8_t *>(c + 256 + rows * k.ldq);
  return k;
}

// 4 lanes per block of 32, eight values each (128-bit loads where `vec`); two blocks per lane group in flight.
__device__ __forceinline__ void ld8(const float *src, int64_t left, bool vec, float (&v)[8]) {
  if (vec && left >= 8) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(src)), b = __ldg(reinterpret_cast<const float4 *>(src) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = u < left ? __ldg(src + u) : 0.f;
  }
}
__global__ void __launch_bounds__(256)
keep8_kernel(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols, int keep_sign, bool vec, Kept k) {
  constexpr int IN_FLIGHT = 2;
  const int64_t per_row = k.ldq / 8, total = rows * per_row, step = (int64_t)gridDim.x * blockDim.x;
  const bool narrow = total < ((int64_t)1 << 31);
  uint32_t best = 0;
  // (total is a multiple of 4 and whole warps stay in the loop, so that the exchanges have all their lanes)
  for (int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i0 - (threadIdx.x & 31) < total; i0 += IN_FLIGHT * step) {
    float v[IN_FLIGHT][8];
    int64_t row[IN_FLIGHT], col[IN_FLIGHT];
#pragma unroll
    for (int f = 0; f < IN_FLIGHT; ++f) {
      const int64_t i = i0 + f * step;
      const bool in = i < total;
      row[f] = !in ? -1 : (narrow ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row);
      col[f] = in ? (i - row[f] * per_row) * 8 : 0;
      ld8(x + (in ? row[f] * ld : 0) + col[f], in ? cols - col[f] : 0, vec, v[f]);
    }
#pragma unroll
    for (int f = 0; f < IN_FLIGHT; ++f) {
      uint32_t mx = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t b = __float_as_uint(v[f][u]) & 0x7FFFFFFFu;
        if (b < 0x7F800000u && b > mx) mx = b;
      }
#pragma unroll
      for (int o = 2; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor_sync(0xffffffffu, mx, o);
        mx = b > mx ? b : mx;
      }
      best = mx > best ? mx : best;
      // max / 2^e < 127.5: 127.5 = 64 * 1.9921875
      int e = (int)(mx >> 23) - 127 - 6 + ((mx & 0x7FFFFFu) >= 0x7F0000u ? 1 : 0);
      e = e < -126 ? -126 : (e > 121 ? 121 : e);
      const float down = pow2f_exact(-e);
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t b = __float_as_uint(v[f][u]) & 0x7FFFFFFFu;
        int n = b < 0x7F800000u ? max(-127, min(127, __float2int_rn(v[f][u] * down))) : -128;
        if (keep_sign && n == 0 && b != 0) n = v[f][u] < 0.f ? -1 : 1;
        w[u >> 2] |= ((uint32_t)n & 0xFFu) << (8 * (u & 3));
      }
      if (row[f] >= 0) {
        *reinterpret_cast<uint2 *>(k.q + row[f] * k.ldq + col[f]) = make_uint2(w[0], w[1]);
        if ((threadIdx.x & 3) == 0) k.e[row[f] * k.lde + col[f] / 32] = (uint8_t)(e + 127);
      }
    }
  }
  best = __reduce_max_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0 && best) atomicMax(k.amax, best);
}

// Eight consecutive kept values of row r from column c (a multiple of 8), times `s`.
__device__ __forceinline__ void kept8(const Kept &k, int64_t r, int64_t c, float s, float (&v)[8]) {
  const uint2 w = __ldg(reinterpret_cast<const uint2 *>(k.q + r * k.ldq + c));
  const float unit = pow2f_exact((int)__ldg(k.e + r * k.lde + c / 32) - 127);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int n = (int)(int8_t)(((u < 4 ? w.x : w.y) >> (8 * (u & 3))) & 0xFFu);
    v[u] = n == -128 ? NAN : ((float)n * unit) * s;
  }
}

__global__ void __launch_bounds__(256)
kept_read_kernel(Kept k, int64_t rows, int64_t cols, float *__restrict__ out) {
  const int64_t per_row = k.ldq / 8, total = rows * per_row, step = (int64_t)gridDim.x * blockDim.x;
  const bool vec = cols % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    float v[8];
    kept8(k, r, c, 1.f, v);
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

// The kept values as one fp16 operand (exact: q has 7 bits; values below 2^-24 of the array's scale
// step, 2^-38 of its largest value, round to nothing). Sixteen values per thread.
__global__ void __launch_bounds__(256)
kept_half_kernel(Kept k, int64_t rows, __half *__restrict__ out) {
  const int64_t per_row = k.ldq / 16, total = rows * per_row, step = (int64_t)gridDim.x * blockDim.x;
  const bool narrow = total < ((int64_t)1 << 31);
  const float s = half_scale(k.amax);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t r = narrow ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row, c = (i - r * per_row) * 16;
    const uint4 w = __ldg(reinterpret_cast<const uint4 *>(k.q + r * k.ldq + c));
    const float unit = pow2f_exact((int)__ldg(k.e + r * k.lde + c / 32) - 127);
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    __half h[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int n = (int)(int8_t)((ws[u >> 2] >> (8 * (u & 3))) & 0xFFu);
      h[u] = __float2half_rn(n == -128 ? NAN : ((float)n * unit) * s);
    }
    uint4 *dst = reinterpret_cast<uint4 *>(out + r * k.ldq + c);
    dst[0] = reinterpret_cast<uint4 *>(h)[0];
    dst[1] = reinterpret_cast<uint4 *>(h)[1];
  }
}

// ds = g act'(out) for eight columns; out from fp32 (`out`) or from its kept form.
struct DsArgs {
  const float *g, *out;
  Kept kept;
  int act;
  int64_t M, N;
  bool vec;
};
__device__ __forceinline__ void ds8(const DsArgs &a, int64_t r, int64_t c, float (&v)[8]) {
  const int64_t left = a.N - c;
  float o[8];
  ld8(a.g + r * a.N + c, left, a.vec, v);
  if (a.act) {
    if (a.out) ld8(a.out + r * a.N + c, left, a.vec, o);
    else kept8(a.kept, r, c, 1.f, o);
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = u < left ? v[u] * act_bwd(a.act, o[u]) : 0.f;
  }
}
// The largest finite |ds| and, in the CTAs from `split` on, the largest finite |W|.
__global__ void __launch_bounds__(256) ds_amax_kernel(DsArgs a, const float *__restrict__ W, int64_t w_rows, int64_t w_cols, int64_t ldw,
                                                      int split, uint32_t *__restrict__ amax) {
  const bool second = (int)blockIdx.x >= split;
  const int block = (int)blockIdx.x - (second ? split : 0), blocks = second ? (int)gridDim.x - split : split;
  const int64_t per_row = ((second ? w_cols : a.N) + 7) / 8, total = (second ? w_rows : a.M) * per_row, step = (int64_t)blocks * blockDim.x;
  const bool narrow = total < ((int64_t)1 << 31);
  const bool vec = ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(W) & 15) == 0;
  uint32_t best = 0;
  for (int64_t i = (int64_t)block * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t r = narrow ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row, c = (i - r * per_row) * 8;
    float v[8];
    if (second) ld8(W + r * ldw + c, w_cols - c, vec, v);
    else ds8(a, r, c, v);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t b = __float_as_uint(v[u]) & 0x7FFFFFFFu;
      if (b < 0x7F800000u && b > best) best = b;
    }
  }
  best = __reduce_max_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0 && best) atomicMax(amax + (second ? 1 : 0), best);
}
// The fp16 pair of ds and its sums over 64 rows: a CTA takes 64 rows x 128 columns.
__global__ void __launch_bounds__(256)
ds_split_kernel(DsArgs a, const uint32_t *__restrict__ amax, __half *__restrict__ hi, __half *__restrict__ lo, int64_t ld,
                float *__restrict__ sums) {
  __shared__ float sh[16][128];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 128 + tx * 8;
  const float s = half_scale(amax);
  for (int64_t t = blockIdx.y; t * 64 < a.M; t += gridDim.y) {
    float cs[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) cs[u] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = t * 64 + ty + 16 * j;
      if (r < a.M && c < a.N) {
        float v[8];
        ds8(a, r, c, v);
        __half h[8], l[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) half_pair(v[u] * s, h[u], l[u]);
        *reinterpret_cast<uint4 *>(hi + r * ld + c) = *reinterpret_cast<uint4 *>(h);
        *reinterpret_cast<uint4 *>(lo + r * ld + c) = *reinterpret_cast<uint4 *>(l);
#pragma unroll
        for (int u = 0; u < 8; ++u) cs[u] += v[u];
      }
    }
    if (sums) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 8; ++u) sh[ty][tx * 8 + u] = cs[u];
      __syncthreads();
      if (threadIdx.x < 128) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += sh[i][threadIdx.x];
        const int64_t n = (int64_t)blockIdx.x * 128 + threadIdx.x;
        if (n < a.N) sums[t * a.N + n] = v;
      }
    }
  }
}

struct KeepForward { uint32_t *amax; __half *xh, *xl, *wh, *wl; float *partial; int64_t ldx, ldw; };
static size_t keep_carve_forward(int64_t M, int64_t N, int64_t K, char *base, KeepForward &f) {
  Carver c{base};
  f = KeepForward{};
  f.amax = c.take<uint32_t>(2);
  f.ldx = ceil_div(K, 8) * 8; f.ldw = ceil_div(N, 8) * 8;
  f.xh = c.take<__half>(M * f.ldx); f.xl = c.take<__half>(M * f.ldx);
  f.wh = c.take<__half>(K * f.ldw); f.wl = c.take<__half>(K * f.ldw);
  f.partial = reinterpret_cast<float *>(c.take<char>((int64_t)gemm_f16_partial_bytes(M, N, K)));
  return c.used;
}
struct KeepBackward { uint32_t *amax; __half *dh, *dl, *wh, *wl, *x8; float *partial, *sums; int64_t ldd, ldw, ldx; };
static size_t keep_carve_backward(int64_t M, int64_t N, int64_t K, char *base, KeepBackward &f) {
  Carver c{base};
  f = KeepBackward{};
  f.amax = c.take<uint32_t>(2);
  f.sums = c.take<float>(ceil_div(M, 64) * N);
  f.ldd = f.ldw = ceil_div(N, 8) * 8;
  f.ldx = ceil_div(K, 32) * 32;
  f.dh = c.take<__half>(M * f.ldd); f.dl = c.take<__half>(M * f.ldd);
  f.wh = c.take<__half>(K * f.ldw); f.wl = c.take<__half>(K * f.ldw);
  f.x8 = c.take<__half>(M * f.ldx);
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

static int run_keep8(const float *x, int64_t ld, int64_t rows, int64_t cols, int keep_sign, void *kept, cudaStream_t s) {
  EB_CUDA(cudaMemsetAsync(kept, 0, 256, s));
  if (rows == 0 || cols == 0) return ENDIA_B200_OK;
  const Kept k = kept_view(kept, rows, cols);
  const int grid = grid_for(rows * (k.ldq / 8), 256, 8);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ld % 4 == 0 || rows == 1);
  keep8_kernel<<<grid, 256, 0, s>>>(x, ld, rows, cols, keep_sign, vec, k);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

}  // namespace eb

extern "C" {

size_t endia_b200_keep8_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return 0;
  const size_t ldq = ((size_t)cols + 31) / 32 * 32;
  return 256 + ((size_t)rows * (ldq + ldq / 32) + 255) / 256 * 256;
}

int endia_b200_keep8(const float *x, int64_t ldx, int64_t rows, int64_t cols, int32_t keep_sign, void *kept, void *stream) {
  int st = require_device();
  if (st) return st;
  EB_REQUIRE(rows >= 0 && cols >= 0, ENDIA_B200_EINVAL, "keep8: negative size");
  EB_REQUIRE(kept && (reinterpret_cast<uintptr_t>(kept) & 255) == 0, ENDIA_B200_EINVAL, "keep8: kept must be given, 256-byte aligned");
  EB_REQUIRE(rows == 0 || cols == 0 || (x && ldx >= cols), ENDIA_B200_EINVAL, "keep8: NULL input or leading dimension too small");
  return run_keep8(x, ldx, rows, cols, keep_sign, kept, as_stream(stream));
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
  if (M == 0) return kept_x ? run_keep8(x, ldx, M, K, keep_sign, kept_x, s) : ENDIA_B200_OK;
  EB_REQUIRE(x && ldx >= K && (N == 0 || (W && out && ldw >= N)), ENDIA_B200_EINVAL, "linear_keep: NULL pointer or leading dimension too small");
  if (kept_x && (st = run_keep8(x, ldx, M, K, keep_sign, kept_x, s))) return st;
  if (N == 0) return ENDIA_B200_OK;
  KeepForward f;
  keep_carve_forward(M, N, K, static_cast<char *>(scratch), f);
  // the 8-bit form has found the largest |x| already; its head, cleared with it, has room for W's
  uint32_t *amax_x = kept_x ? static_cast<uint32_t *>(kept_x) : f.amax, *amax_w = amax_x + 1;
  if (!kept_x) EB_CUDA(cudaMemsetAsync(f.amax, 0, 2 * sizeof(uint32_t), s));
  HalfJob jw{W, K, N, ldw, nullptr, amax_w, f.wh, f.wl, f.ldw};
  HalfJob jx{x, M, K, ldx, nullptr, amax_x, f.xh, f.xl, f.ldx};
  if ((st = launch_amax(jw, kept_x ? nullptr : &jx, s))) return st;
  if ((st = launch_half_split(jw, &jx, s))) return st;
  F16Gemm g;
  g.M = M; g.N = N; g.K = K;
  g.a = HalfPair{f.xh, f.xl, f.ldx, amax_x};
  g.b = HalfPair{f.wh, f.wl, f.ldw, amax_w};
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
  DsArgs a{};
  a.g = grad; a.out = act && out ? out : nullptr; a.act = act; a.M = M; a.N = N;
  if (act && !out) a.kept = kept_view(const_cast<void *>(kept_out), M, N);
  a.vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(grad) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const dim3 grid((unsigned)ceil_div(N, 128), (unsigned)(ceil_div(M, 64) < 32768 ? ceil_div(M, 64) : 32768));
  EB_CUDA(cudaMemsetAsync(f.amax, 0, 2 * sizeof(uint32_t), s));
  const int split = grid_for(M * ceil_div(N, 8), 256, 8), more = dx ? grid_for(K * ceil_div(N, 8), 256, 8) : 0;
  ds_amax_kernel<<<split + more, 256, 0, s>>>(a, W, K, N, ldw, split, f.amax);
  EB_LAUNCH_CHECK();
  ds_split_kernel<<<grid, 256, 0, s>>>(a, f.amax, f.dh, f.dl, f.ldd, db ? f.sums : nullptr);
  EB_LAUNCH_CHECK();
  if (db && (st = launch_column_sums(f.sums, (int)ceil_div(M, 64), N, 1.f, nullptr, db, s))) return st;
  const Kept kx = kept_view(const_cast<void *>(kept_x), M, K);
  const HalfPair d{f.dh, f.dl, f.ldd, f.amax};
  if (dw) {
    kept_half_kernel<<<grid_for(M * (kx.ldq / 16), 256, 8), 256, 0, s>>>(kx, M, f.x8);
    EB_LAUNCH_CHECK();
    F16Gemm g;
    g.M = K; g.N = N; g.K = M;
    g.a = HalfPair{f.x8, nullptr, f.ldx, kx.amax};
    g.b = d;
    g.C = dw; g.ldc = N; g.partial = f.partial;
    if ((st = launch_gemm_f16(g, true, true, F16_STORE, s))) return st;
  }
  if (dx) {
    const HalfJob jw{W, K, N, ldw, nullptr, f.amax + 1, f.wh, f.wl, f.ldw};
    if ((st = launch_half_split(jw, nullptr, s))) return st;
    F16Gemm g;
    g.M = M; g.N = K; g.K = N;
    g.a = d;
    g.b = HalfPair{f.wh, f.wl, f.ldw, f.amax + 1};
    g.C = dx; g.ldc = K; g.partial = f.partial;
    if ((st = launch_gemm_f16(g, false, false, F16_STORE, s))) return st;
  }
  return ENDIA_B200_OK;
}

}  // extern "C"
