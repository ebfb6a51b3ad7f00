// fp32-accurate products from fp16 pairs (see gemm_f16.cuh) and the passes that make the pairs.
//
// One persistent kernel of CTA pairs (cta_group::2), 256 x 256 tiles, as the framework's other two-CTA
// product, but with another division of the work, because what limits accuracy there is the
// accumulator: tensor memory adds with rounding toward zero, a bias that grows with the number of
// adds (1e-5 of the result after 2048 of K). Here an accumulator lives for one stage of 64 of K (two in
// some kernels, see f16_run_first):
//   - the eight correction MMAs first, into an empty accumulator (they are 2^-11 of the result, so
//     their truncation is too), then the four MMAs of hi*hi: four truncating adds in all;
//   - the epilogue warps add it to the tile's sums, which they hold in registers (128 a thread) with
//     round to nearest, while the MMAs of the next stage fill the other half of tensor memory.
// Per stage the tensor pipe is busy for 12 x 128 = 1536 cycles (1560 measured with clock stamps); the drain of 256
// columns by eight warps takes about a third of that, so it costs no tensor time. What it buys: errors of
// 2e-7 instead of 1e-5 at K = 4096, at 3 fp16 MMAs per product (tf32 + 2 bf16 take the time of 4).
// Bound by power: 2048 x 16384 x 1024 and the like run at 1.3 to 1.56 PFLOP/s of MMAs with the clock at 1.6 of
// 1.965 GHz (the measured cuBLAS bf16 rate is 1.66 in a burst, 1.38 sustained).
//   warp 0: TMA producer (one lane), warp 1: MMA issuer (one lane of the leader CTA), warps 2, 3 idle
//   warps 4-11: sums, epilogue and stores (lane quarter warp & 3, column half (warp - 4) >> 2)
// The 168 registers a thread that the launch hands out are split as 40 for the first warpgroup and 232
// for the other two (128 sums, 64 in flight from tensor memory).
// Every wait is bounded; a wait that gives up records a code, the CTA drains its copies and returns.
#include "gemm_f16.cuh"
#include "gemm.cuh"
#include "tc_ptx.cuh"

namespace eb {

constexpr int F16_BK = 64;                       // one stage: 64 of K, 128 bytes per K-major row
constexpr uint32_t F16_TILE = 128 * F16_BK * 2;  // bytes of one [128 x 64] fp16 tile
constexpr int F16_EPI_WARPS = 8;
constexpr int F16_THREADS = 384;
constexpr int F16_REGS_CONTROL = 40, F16_REGS_EPI = 232;
static_assert(F16_REGS_CONTROL * 128 + F16_REGS_EPI * 256 <= 168 * F16_THREADS, "registers of the launch");

struct F16Maps {
  CUtensorMap a_hi, a_lo, b_hi, b_lo;
  CUtensorMap c;           // F16_STORE: C or the work space, boxes of [32 rows][32 floats]
  CUtensorMap d_hi, d_lo;  // F16_DLOGITS: boxes of [32 rows][32 halfs]
};

struct F16Params {
  int M, N;
  int pairs_m, tiles_n, group_m, ksplit, nkb;   // nkb: stages of 64 of K in all
  const int *ea, *eb;            // the operands' scale exponents, leading dimensions and last blocks along m and n
  int64_t ea_ld, eb_ld;
  int a_last, b_last;
  const float *alpha_dev;
  int alpha_exp;
  const float *bias;
  float *C;
  int64_t ldc;
  int act, accumulate, vec_c;    // vec_c: C goes out by bulk tensor stores
  int part_rows;                 // > 0: range r of K stores its bare sums to rows [r * part_rows, ...) behind maps.c
  const float *target;
  int64_t n_base;
  float2 *stats;
  float *target_logit;
  const float *lse, *coef;
  float *colsum_part;
};

// K-major tile [128 rows][64 k]: 128-byte rows, 128-byte swizzle, 8-row groups 1024 bytes apart.
// MN-major tile: two boxes of [64 k][64 rows] 8192 bytes apart, 8-k-row groups 1024 bytes apart.
template <bool MN>
__device__ __forceinline__ uint64_t f16_desc(uint32_t addr) {
  return MN ? smem_desc(addr, 8192, 1024, 2) : smem_desc(addr, 16, 1024, 2);
}
template <bool MN>
__device__ __forceinline__ void f16_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int row0, int k0) {
  if constexpr (MN) {
    tma_load_2d_pair(dst, map, bar, row0, k0);
    tma_load_2d_pair(dst + 8192u, map, bar, row0 + 64, k0);
  } else {
    tma_load_2d_pair(dst, map, bar, k0, row0);
  }
}

// A run: the stages that one accumulator sums before it is drained; stage i of a tile of n is the first
// or the last of its run. Stored products of two pairs have runs of one stage. Runs of two:
//   - the logit kernels: their epilogue (exponentials of a whole tile) outlasts the two stages that the MMAs can
//     run ahead with runs of one (2048 x 1024 x 32768: statistics 294 -> 262 us, d 177 -> 162 us)
//   - products with an exact operand: a stage is 1024 cycles of MMAs there, shorter than a drain and its
//     hand-over (layer 8192 x 4096 x 4096, the whole step: 2.22 -> 2.18 ms)
// Expected loss to truncation, 4.3e-8 of the running sum per add: 1.1e-7 of the result with runs of one,
// 3.7e-7 (2.8e-7 with an exact operand) with runs of two, where the second stage's corrections add to the
// full sum. A stored product of two pairs gains 1 to 2 % from runs of two and keeps the smaller error.
template <int PROD, int EPI>
__device__ __forceinline__ bool f16_run_first(int i) { return (PROD == 3 && EPI == F16_STORE) || (i & 1) == 0; }
template <int PROD, int EPI>
__device__ __forceinline__ bool f16_run_last(int i, int n) { return (PROD == 3 && EPI == F16_STORE) || (i & 1) == 1 || i == n - 1; }

// Column sums over a warp's 32 rows: v[j] of lane r is row r, column j; returns, in lane L, the sum of
// column L. Halves the columns a lane is responsible for in each of five exchanges.
__device__ __forceinline__ float warp_colsum32(float (&v)[32], int lane) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    const bool up = (lane & w) != 0;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float send = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
    }
  }
  return v[0];
}

constexpr float LOG2E = 1.4426950408889634f;
// 2^x in one instruction (results below 2^-126 are zero)
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two fp32 lanes per instruction: (a0, a1) = (x0, x1) * s + (a0, a1), and products and sums of the kind.
__device__ __forceinline__ void fma2(float &a0, float &a1, float x0, float x1, float s) {
  asm("{\n\t.reg .b64 a, x, f;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 x, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\t"
      "fma.rn.f32x2 a, x, f, a;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(x0), "f"(x1), "f"(s));
}
__device__ __forceinline__ void scale_add2(float &a0, float &a1, float s, float b0, float b1) {      // a = a * s + b
  asm("{\n\t.reg .b64 a, b, f;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%3, %4};\n\tmov.b64 f, {%2, %2};\n\t"
      "fma.rn.f32x2 a, a, f, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(s), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul2(float &a0, float &a1, float s) {
  asm("{\n\t.reg .b64 a, f;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 f, {%2, %2};\n\tmul.rn.f32x2 a, a, f;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(s));
}
__device__ __forceinline__ void add2(float &a0, float &a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void sts128u(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// PROD: 3 = both operands are pairs, 2 = A is exact in its hi part.
template <bool A_MN, bool B_MN, int PROD, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F16_THREADS, 1)
gemm_f16_kernel(const __grid_constant__ F16Maps maps, const F16Params p) {
  constexpr int STAGES = PROD == 3 ? 3 : 4;
  constexpr uint32_t A_BYTES = (PROD == 3 ? 2 : 1) * F16_TILE, STAGE_BYTES = A_BYTES + 2 * F16_TILE;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t smem_base = (smem_u32(smem) + 1023u) & ~1023u;
  const uint32_t epi_base = smem_base + STAGES * STAGE_BYTES;
  const uint32_t bars = epi_base + F16_EPI_WARPS * 4096u;
  __shared__ uint32_t tmem_slot;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int num_pairs = (int)(gridDim.x >> 1), pair_id = (int)(blockIdx.x >> 1);
  const int tiles_mn = p.pairs_m * p.tiles_n, num_items = tiles_mn * p.ksplit;
  auto k_range = [&](int t, int &kb0, int &kb1) {      // (ranges of whole blocks of 128, none empty)
    const int part = t / tiles_mn, blocks = (p.nkb + 1) / 2;
    kb0 = 2 * (int)((int64_t)blocks * part / p.ksplit);
    kb1 = 2 * (int)((int64_t)blocks * (part + 1) / p.ksplit);
    kb1 = kb1 < p.nkb ? kb1 : p.nkb;
  };
  // groups of group_m row pairs, the column tiles of a group one after the other: the pairs that run at
  // the same time share a few bands of A and tiles of B in L2
  auto tile_origin = [&](int w, int &m0, int &n0) {
    const int t = w % tiles_mn;
    const int group = t / (p.group_m * p.tiles_n);
    const int gm0 = group * p.group_m;
    const int gh = p.pairs_m - gm0 < p.group_m ? p.pairs_m - gm0 : p.group_m;
    const int rem = t - group * (p.group_m * p.tiles_n);
    m0 = (gm0 + rem % gh) * 256 + (int)rank * 128;
    n0 = (rem / gh) * 256;
  };
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto acc_full = [&](int b) { return bars + 8u * (2 * STAGES + b); };
  auto acc_empty = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 2 * F16_EPI_WARPS); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F16_REGS_CONTROL));
  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = pair_id; t < num_items && ok; t += num_pairs) {
        int m0, n0, kb, kb1;
        tile_origin(t, m0, n0);
        k_range(t, kb, kb1);
        const int nh0 = n0 + (int)rank * 128;
        for (; kb < kb1; ++kb, ++it) {
          const int s = (int)(it % STAGES);
          if (it >= STAGES && !mbar_wait(empty_bar(s), ((it / STAGES) - 1) & 1, 51)) { ok = false; break; }
          const uint32_t st = smem_base + s * STAGE_BYTES, sb = st + A_BYTES;
          if (leader) mbar_expect_tx(full_bar(s), 2 * STAGE_BYTES);   // both CTAs' bytes
          const uint32_t fb = map_to_cta(full_bar(s), 0);
          const int k0 = kb * F16_BK;
          f16_load<A_MN>(st, &maps.a_hi, fb, m0, k0);
          if constexpr (PROD == 3) f16_load<A_MN>(st + F16_TILE, &maps.a_lo, fb, m0, k0);
          f16_load<B_MN>(sb, &maps.b_hi, fb, nh0, k0);
          f16_load<B_MN>(sb + F16_TILE, &maps.b_lo, fb, nh0, k0);
        }
      }
      if (!ok && leader) {
        // copies in flight (of both CTAs) get a bounded chance to land before the pair exits
        for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j)
          mbar_wait(full_bar((int)(j % STAGES)), (j / STAGES) & 1, 52);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // fp32 accumulator, fp16 A and B (format 0), majors, N >> 3, M >> 4
      const uint32_t idesc = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                             ((uint32_t)(256 >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
      // 16 of K further: 32 bytes along a K-major row, 16 k-rows (2048 bytes) of an MN-major box
      constexpr uint64_t A_STEP = A_MN ? 128 : 2, B_STEP = B_MN ? 128 : 2;
      // descriptors of stage 0; a stage further is STAGE_BYTES, in 16-byte units (addresses stay below 2^18)
      const uint64_t ah0 = f16_desc<A_MN>(smem_base), al0 = f16_desc<A_MN>(smem_base + F16_TILE);
      const uint64_t bh0 = f16_desc<B_MN>(smem_base + A_BYTES), bl0 = f16_desc<B_MN>(smem_base + A_BYTES + F16_TILE);
      uint32_t j = 0, s = 0, s_phase = 0;      // runs so far; ring position
      bool ok = true;
      for (int t = pair_id; t < num_items && ok; t += num_pairs) {
        int kb0, kb1;
        k_range(t, kb0, kb1);
        const int n = kb1 - kb0;
        for (int i = 0; i < n; ++i) {
          const bool first = f16_run_first<PROD, EPI>(i), last = f16_run_last<PROD, EPI>(i, n);
          const uint32_t b = j & 1;
          if (!mbar_wait(full_bar((int)s), s_phase, 54)) { ok = false; break; }
          if (first && j >= 2 && !mbar_wait(acc_empty((int)b), ((j >> 1) - 1) & 1, 53)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + 256u * b, more = first ? 0u : 1u;
          const uint64_t off = (uint64_t)(s * (STAGE_BYTES >> 4));
          const uint64_t ah = ah0 + off, bh = bh0 + off, bl = bl0 + off;
          if constexpr (PROD == 3) {
            const uint64_t al = al0 + off;
            tc_mma_16bit_pair(d, al, bh, idesc, more);
#pragma unroll
            for (int ks = 1; ks < F16_BK / 16; ++ks) tc_mma_16bit_pair(d, al + ks * A_STEP, bh + ks * B_STEP, idesc, 1u);
          }
          tc_mma_16bit_pair(d, ah, bl, idesc, PROD == 3 ? 1u : more);
#pragma unroll
          for (int ks = 1; ks < F16_BK / 16; ++ks) tc_mma_16bit_pair(d, ah + ks * A_STEP, bl + ks * B_STEP, idesc, 1u);
#pragma unroll
          for (int ks = 0; ks < F16_BK / 16; ++ks) tc_mma_16bit_pair(d, ah + ks * A_STEP, bh + ks * B_STEP, idesc, 1u);
          tc_commit_pair(empty_bar((int)s));
          if (last) { tc_commit_pair(acc_full((int)b)); ++j; }
          if (++s == STAGES) { s = 0; s_phase ^= 1; }
        }
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F16_REGS_EPI));
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t ebuf = epi_base + (uint32_t)(warp - 4) * 4096u;
    const uint32_t row_addr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * 128);
    const uint32_t empty_leader[2] = {map_to_cta(acc_empty(0), 0), map_to_cta(acc_empty(1), 0)};
    uint32_t j = 0;
    bool ok = true;
    for (int t = pair_id; t < num_items && ok; t += num_pairs) {
      int m0, n0, kb, kb1;
      tile_origin(t, m0, n0);
      k_range(t, kb, kb1);
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // the scale exponents along K of this CTA's block of A and this warp's block of B
      const int64_t mblk = min(m0 >> 7, p.a_last), nblk = min((n0 + half * 128) >> 7, p.b_last);
      const int *ea = p.ea ? p.ea + (A_MN ? mblk : mblk * p.ea_ld) : nullptr, *eb = p.eb ? p.eb + (B_MN ? nblk : nblk * p.eb_ld) : nullptr;
      auto unscale_of = [&](int kblk) {
        return -((ea ? __ldg(ea + (A_MN ? kblk * p.ea_ld : kblk)) : 0) + (eb ? __ldg(eb + (B_MN ? kblk * p.eb_ld : kblk)) : 0));
      };
      // the tile's unit: the largest unscaling exponent along K
      int unit = -1000;
      for (int k = (kb >> 1) + lane; 2 * k < kb1; k += 32) unit = max(unit, unscale_of(k));
      unit = __reduce_max_sync(0xffffffffu, unit);
      for (int i = 0, n = kb1 - kb; i < n; ++i) {
        if (!f16_run_last<PROD, EPI>(i, n)) continue;
        const uint32_t b = j & 1;
        const int e = unscale_of((kb + i) >> 1) - unit;      // <= 0
        if (!mbar_wait(acc_full((int)b), (j >> 1) & 1, 55)) { ok = false; break; }
        tc_fence_after();
        const float s0 = e < -126 ? 0.f : pow2f_exact(e);
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          uint32_t r0[32], r1[32];
          tc_ld32(row_addr + 256u * b + (uint32_t)(32 * c), r0);
          tc_ld32(row_addr + 256u * b + (uint32_t)(32 * c + 32), r1);
          tc_wait_ld();
          if (c == 2) {       // the last values have left tensor memory
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(empty_leader[b]);
          }
#pragma unroll
          for (int u = 0; u < 32; u += 2) {
            fma2(acc[32 * c + u], acc[32 * c + u + 1], __uint_as_float(r0[u]), __uint_as_float(r0[u + 1]), s0);
            fma2(acc[32 * c + 32 + u], acc[32 * c + 33 + u], __uint_as_float(r1[u]), __uint_as_float(r1[u + 1]), s0);
          }
        }
        ++j;
      }
      if (!ok) break;
      const int nb = n0 + half * 128;            // this warp's first column
      const int mq = m0 + q * 32, m = mq + lane; // its first row, this lane's row

      if constexpr (EPI == F16_STORE) {
        const bool parts = p.part_rows > 0;
        float f0, f1;      // (the parts' alpha comes with their sum)
        alpha_factors(parts ? nullptr : p.alpha_dev, unit + (parts ? 0 : p.alpha_exp), f0, f1);
        const int row_off = parts ? (t / tiles_mn) * p.part_rows : 0;
        const bool bulk = parts || p.vec_c;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int nc = nb + 32 * c;
          if (nc < p.N && mq < p.M) {            // (uniform over the warp)
            const float bv = (!parts && p.bias && nc + lane < p.N) ? __ldg(p.bias + nc + lane) : 0.f;
            if (bulk) {                          // the previous chunk's store has read the buffer
              if (lane == 0) bulk_wait_read0();
              __syncwarp();
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              float4 v = make_float4(acc[32 * c + 4 * u], acc[32 * c + 4 * u + 1], acc[32 * c + 4 * u + 2], acc[32 * c + 4 * u + 3]);
              v.x = (v.x * f0) * f1; v.y = (v.y * f0) * f1; v.z = (v.z * f0) * f1; v.w = (v.w * f0) * f1;
              sts128(ebuf + (uint32_t)lane * 128u + (uint32_t)((u ^ (lane & 7)) * 16), v);
            }
            __syncwarp();
            if (!parts && (p.bias || p.act || !bulk)) {
              // lanes along the row: bias and activation, and the stores where C has no 16-byte rows
              const uint32_t col = (uint32_t)(lane >> 2), sub = (uint32_t)(lane & 3) * 4u;
#pragma unroll 4
              for (int r = 0; r < 32; ++r) {
                const uint32_t a = ebuf + (uint32_t)r * 128u + ((col ^ (uint32_t)(r & 7)) * 16u) + sub;
                float v;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
                v += bv;
                if (p.act) v = act_fwd(p.act, v);
                if (bulk) {
                  asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
                } else if (mq + r < p.M && nc + lane < p.N) {
                  float *cp = p.C + (int64_t)(mq + r) * p.ldc + nc + lane;
                  *cp = p.accumulate ? *cp + v : v;
                }
              }
            }
            if (bulk) {
              fence_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (p.accumulate && !parts) tma_reduce_add_2d(&maps.c, ebuf, nc, mq);
                else tma_store_2d(&maps.c, ebuf, nc, mq + row_off);
                bulk_commit();
              }
            } else {
              __syncwarp();
            }
          }
        }
      } else {
        const bool row_ok = m < p.M;
        const float tg = row_ok ? __ldg(p.target + m) : -1.f;
        const int64_t v0 = p.n_base + nb;
        // this lane's target among the warp's 128 columns, or -1
        const int tl = (tg >= (float)v0 && tg < (float)(v0 + 128)) ? (int)((int64_t)tg - v0) : -1;
        const bool any_target = __any_sync(0xffffffffu, tl >= 0);
        // Logits in units of log2 e, so that an exponential is one MUFU operation on a difference: a rounding of
        // 2^-24 of the logit, as in any fp32 logit. (One factor: a unit beyond its range belongs to logits below
        // 2^-80, or to sums that fp32 does not hold.)
        const float to_log2 = pow2f_exact(max(-126, min(126, unit))) * LOG2E;
        float bv[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) bv[c] = p.bias && nb + 32 * c + lane < p.N ? __ldg(p.bias + nb + 32 * c + lane) * LOG2E : 0.f;
        if constexpr (EPI == F16_STATS) {
          if (p.bias) {
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = fmaf(acc[i], to_log2, __shfl_sync(0xffffffffu, bv[i >> 5], i & 31));
          } else {
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] *= to_log2;
          }
          if (nb + 128 > p.N) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (nb + i >= p.N) acc[i] = -INFINITY;
          }
          if (any_target) {
            float tv = 0.f;
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i == tl) tv = acc[i];
            if (tl >= 0) p.target_logit[m] = tv;
          }
          // maximum and sum of exponentials, four chains each; -inf columns (banned classes) add 0, a NaN
          // makes the sum NaN
          float mx4[4] = {acc[0], acc[1], acc[2], acc[3]}, s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 4; i < 128; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], acc[i]);
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          const float base = mx == -INFINITY ? 0.f : mx;      // (a row of -inf: 2^-inf = 0)
#pragma unroll
          for (int i = 0; i < 128; ++i) s4[i & 3] += exp2_fast(acc[i] - base);
          if (row_ok) p.stats[(v0 >> 7) * (int64_t)p.M + m] = make_float2(mx, (s4[0] + s4[1]) + (s4[2] + s4[3]));
        } else {
          const float lse = row_ok ? __ldg(p.lse + m) : 0.f, cf = row_ok ? __ldg(p.coef + m) : 0.f;
          const bool any_dead = __any_sync(0xffffffffu, cf == 0.f);
          const float cs = cf * F16_D_SCALE;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int nc = nb + 32 * c;
            if (nc >= p.N || mq >= p.M) continue;      // (uniform over the warp)
            float v[32];
            // p = 2^(l - lse), d = (p - [target]) coef
            if (p.bias) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = exp2_fast(fmaf(acc[32 * c + i], to_log2, __shfl_sync(0xffffffffu, bv[c], i) - lse));
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                v[i] = acc[32 * c + i];
                v[i + 1] = acc[32 * c + i + 1];
                scale_add2(v[i], v[i + 1], to_log2, -lse, -lse);
                v[i] = exp2_fast(v[i]);
                v[i + 1] = exp2_fast(v[i + 1]);
              }
            }
            if (any_target) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (32 * c + i == tl) v[i] -= 1.f;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) mul2(v[i], v[i + 1], cs);
            if (any_dead) {      // rows that are left out: exactly zero, whatever their logits are
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = cf == 0.f ? 0.f : v[i];
            }
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const __half2 h = __floats2half2_rn(v[2 * u], v[2 * u + 1]);
              const float2 hf = __half22float2(h);
              float l0 = v[2 * u], l1 = v[2 * u + 1];
              add2(l0, l1, -hf.x, -hf.y);
              const __half2 l = __floats2half2_rn(l0, l1);
              hi[u] = *reinterpret_cast<const uint32_t *>(&h);
              lo[u] = *reinterpret_cast<const uint32_t *>(&l);
            }
            // both parts of [32 rows][32 columns] through the warp's buffer, 64-byte rows, 64-byte swizzle
            if (lane == 0) bulk_wait_read0();      // the previous chunk's stores have read it
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint32_t at = ebuf + (uint32_t)lane * 64u + (uint32_t)((u ^ ((lane >> 1) & 3)) * 16);
              sts128u(at, hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]);
              sts128u(at + 2048u, lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.d_hi, ebuf, nc, mq);
              tma_store_2d(&maps.d_lo, ebuf + 2048u, nc, mq);
              bulk_commit();
            }
            if (p.colsum_part) {
              const float s = warp_colsum32(v, lane);
              if (nc + lane < p.N) p.colsum_part[(int64_t)(mq >> 5) * p.N + nc + lane] = s;
            }
          }
        }
      }
    }
    if (lane == 0) bulk_wait0();   // the stores have left shared memory and are complete
  }
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// C = act(alpha * sum over the ranges of K, in order, + bias), or C += it. Four consecutive columns per
// thread (the rows of the work space are 16-byte aligned).
__global__ void __launch_bounds__(256)
gemm_f16_finish_kernel(const F16Params p, const float *__restrict__ partial, int64_t ld_partial, int64_t slice, int parts) {
  float f0, f1;
  alpha_factors(p.alpha_dev, p.alpha_exp, f0, f1);
  const uint32_t per_row = (uint32_t)((p.N + 3) / 4);
  const int64_t total = (int64_t)p.M * per_row, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t m = total < ((int64_t)1 << 31) ? (int64_t)((uint32_t)i / per_row) : i / per_row;
    const int n = (int)(i - m * per_row) * 4;
    const float *src = partial + m * ld_partial + n;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 4) {
      float4 t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        t[u] = s0 + u < parts ? __ldcs(reinterpret_cast<const float4 *>(src + (int64_t)(s0 + u) * slice)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 4; ++u) { v[0] += t[u].x; v[1] += t[u].y; v[2] += t[u].z; v[3] += t[u].w; }
    }
    float *c = p.C + m * p.ldc + n;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k < p.N) {
        v[k] = (v[k] * f0) * f1 + (p.bias ? __ldg(p.bias + n + k) : 0.f);
        if (p.act) v[k] = act_fwd(p.act, v[k]);
        if (p.accumulate) v[k] += c[k];
      }
    }
    if (p.vec_c && n + 4 <= p.N) {
      *reinterpret_cast<float4 *>(c) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < p.N) c[k] = v[k];
    }
  }
}

// out[n] = alpha * scale * sum over the parts [parts][N], in a fixed order: 32 columns per CTA, its eight warps take
// the parts in turn with eight loads in flight.
__global__ void __launch_bounds__(256)
column_sums_kernel(const float *__restrict__ part, int parts, int64_t N, float scale, const float *__restrict__ alpha,
                   float *__restrict__ out) {
  __shared__ float sh[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (n < N) {
    for (int r0 = w; r0 < parts; r0 += 64) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = r0 + 8 * u < parts ? __ldg(part + (int64_t)(r0 + 8 * u) * N + n) : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  }
  sh[w][lane] = s;
  __syncthreads();
  if (w == 0 && n < N) {
    for (int i = 1; i < 8; ++i) s += sh[i][lane];
    s *= scale;
    out[n] = alpha ? s * __ldg(alpha) : s;
  }
}

int launch_column_sums(const float *part, int parts, int64_t N, float scale, const float *alpha, float *out, cudaStream_t s) {
  column_sums_kernel<<<(unsigned)ceil_div(N, 32), 256, 0, s>>>(part, parts, N, scale, alpha, out);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

// ---------------------------------------------------------------------------- passes over fp32 arrays
// One CTA of 512 threads per block of 128 x 128: a warp takes 8 rows 16 apart, a lane four columns, so that the
// block stays in registers between its maximum and its pair; every array is read once. With two CTAs per SM
// 128 KB are in flight on each. Bound by HBM: 286 MB (W of 1024 x 32768 and x of 2048 x 1024) in 50-52 us, 5.4 TB/s.
struct HalfJobs {
  HalfJob job[3];
  bool vec[3], vec_out[3];     // 128-bit reads of x and of out
  int begin[3];                // first CTA of each array
  int n;
};
// Four values of a kept array, from column c (a multiple of 4).
__device__ __forceinline__ void kept4(const Kept &k, int64_t r, int64_t c, float (&v)[4]) {
  const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(k.q + r * k.ldq + c));
  const float unit = pow2f_exact((int)__ldg(k.e + r * k.lde + (c >> 5)) - 127);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int n = (int)(int8_t)((w >> (8 * u)) & 0xFFu);
    v[u] = n == -128 ? NAN : (float)n * unit;
  }
}
__device__ __forceinline__ void load4(const float *src, int64_t left, bool vec, float (&v)[4]) {
  if (vec && left >= 4) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(src));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? __ldg(src + i) : 0.f;
  }
}
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// PLAIN: pairs of fp32 arrays and nothing else (fewer registers).
template <bool PLAIN>
__global__ void __launch_bounds__(512, 2) half_split_kernel(const __grid_constant__ HalfJobs jobs) {
  __shared__ uint32_t wmax[16];
  __shared__ float part[16][HALF_BLOCK];
  const int which = jobs.n > 2 && (int)blockIdx.x >= jobs.begin[2] ? 2 : (jobs.n > 1 && (int)blockIdx.x >= jobs.begin[1] ? 1 : 0);
  const HalfJob &j = jobs.job[which];
  const bool vec = jobs.vec[which], vec_out = jobs.vec_out[which];
  const int block = (int)blockIdx.x - jobs.begin[which], bcols = (int)((j.cols + HALF_BLOCK - 1) / HALF_BLOCK);
  const int rb = block / bcols, cb = block - rb * bcols;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)cb * HALF_BLOCK + 4 * lane, left = j.cols - c;
  const int64_t row0 = (int64_t)rb * HALF_BLOCK + w;      // this warp's rows: row0 + 16 i
  bool live[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) live[i] = row0 + 16 * i < j.rows && left > 0 && !(j.target && __ldg(j.target + row0 + 16 * i) < 0.f);
  float v[8][4];
  // (the eight loads are issued together: nothing uses one of them before the last is on its way)
  if (!PLAIN && !j.x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (live[i]) kept4(j.kept, row0 + 16 * i, c, v[i]);
      else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
  } else if (vec && (cb + 1) * HALF_BLOCK <= j.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 t = live[i] ? __ldg(reinterpret_cast<const float4 *>(j.x + (row0 + 16 * i) * j.ld + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) v[i][u] = live[i] && u < left ? __ldg(j.x + (row0 + 16 * i) * j.ld + c + u) : 0.f;
  }
  if (!PLAIN && j.act) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (live[i]) {
        float o[4];
        if (j.out) load4(j.out + (row0 + 16 * i) * j.cols + c, left, vec_out, o);
        else kept4(j.out_kept, row0 + 16 * i, c, o);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[i][u] = u < left ? v[i][u] * act_bwd(j.act, o[u]) : 0.f;
      }
    }
  }
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int u = 0; u < 4; ++u) best = max(best, finite_bits(v[i][u]));
  if (!PLAIN && j.keep.q) {
    // the 8-bit form (keep8.cu): 8 lanes share a scale
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = row0 + 16 * i;
      uint32_t mx = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) mx = max(mx, finite_bits(v[i][u]));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // max / 2^e < 127.5: 127.5 = 64 * 1.9921875
      int e = (int)(mx >> 23) - 127 - 6 + ((mx & 0x7FFFFFu) >= 0x7F0000u ? 1 : 0);
      e = e < -126 ? -126 : (e > 121 ? 121 : e);
      const float down = pow2f_exact(-e);
      uint32_t q = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t b = __float_as_uint(v[i][u]) & 0x7FFFFFFFu;
        int n = b < 0x7F800000u ? max(-127, min(127, __float2int_rn(v[i][u] * down))) : -128;
        if (j.keep_sign && n == 0 && b != 0) n = v[i][u] < 0.f ? -1 : 1;
        q |= ((uint32_t)n & 0xFFu) << (8 * u);
      }
      if (r < j.rows && c < j.keep.ldq) {
        *reinterpret_cast<uint32_t *>(j.keep.q + r * j.keep.ldq + c) = q;
        if ((lane & 7) == 0) j.keep.e[r * j.keep.lde + (c >> 5)] = (uint8_t)(e + 127);
      }
    }
  }
  if (PLAIN || j.hi) {
    best = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) wmax[w] = best;
    __syncthreads();
    best = __reduce_max_sync(0xffffffffu, wmax[lane & 15]);
    const int ex = half_scale_exponent(best);
    if (threadIdx.x == 0) j.e[block] = ex;
    const float s = pow2f_exact(ex);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = row0 + 16 * i;
      if (r < j.rows && left > 0) {        // (ld_out covers whole groups of 4)
        __half h[4], l[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) half_pair(v[i][u] * s, h[u], l[u]);
        *reinterpret_cast<uint2 *>(j.hi + r * j.ld_out + c) = *reinterpret_cast<uint2 *>(h);
        if (PLAIN || j.lo) *reinterpret_cast<uint2 *>(j.lo + r * j.ld_out + c) = *reinterpret_cast<uint2 *>(l);
      }
    }
  }
  if (!PLAIN && j.sums) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float t = v[0][u];
#pragma unroll
      for (int i = 1; i < 8; ++i) t += v[i][u];
      part[w][4 * lane + u] = t;
    }
    __syncthreads();
    if (threadIdx.x < HALF_BLOCK) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) t += part[i][threadIdx.x];
      const int64_t n = (int64_t)cb * HALF_BLOCK + threadIdx.x;
      if (n < j.cols) j.sums[rb * j.cols + n] = t;
    }
  }
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int launch_half_split(const HalfJob *jobs, int n, cudaStream_t s) {
  HalfJobs a;
  bool plain = true;
  int64_t grid = 0;
  a.n = 0;
  for (int i = 0; i < n; ++i) {
    if (jobs[i].rows <= 0 || jobs[i].cols <= 0) continue;
    a.job[a.n] = jobs[i];
    a.vec[a.n] = aligned16(jobs[i].x) && (jobs[i].ld % 4 == 0 || jobs[i].rows == 1);
    a.vec_out[a.n] = aligned16(jobs[i].out) && jobs[i].cols % 4 == 0;
    a.begin[a.n] = (int)grid;
    grid += half_blocks(jobs[i].rows) * half_blocks(jobs[i].cols);
    plain = plain && jobs[i].x && jobs[i].hi && jobs[i].lo && !jobs[i].act && !jobs[i].keep.q && !jobs[i].sums;
    ++a.n;
  }
  if (grid == 0) return ENDIA_B200_OK;
  EB_REQUIRE(grid < ((int64_t)1 << 31), ENDIA_B200_ELIMIT, "fp16-pair product: operands of more than 2^45 elements");
  if (plain) half_split_kernel<true><<<(unsigned)grid, 512, 0, s>>>(a);
  else half_split_kernel<false><<<(unsigned)grid, 512, 0, s>>>(a);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

// ---------------------------------------------------------------------------------------- host side
// Tensor map of a row-major [outer, inner] array: fp16 boxes of 64 elements with the 128-byte
// swizzle for operands, of 32 with the 64-byte one for d, fp32 boxes of [32][32] for C. Elements outside read as zero and are not written.
static int make_map_16(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld, int box_outer,
                       int box_inner = 64) {
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer}, strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer}, estr[2] = {1u, 1u};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 box_inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  EB_REQUIRE(r == CUDA_SUCCESS, ENDIA_B200_ECUDA, "fp16-pair product: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return ENDIA_B200_OK;
}
static int make_map_32(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld) {
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer}, strides[1] = {(cuuint64_t)ld * 4};
  cuuint32_t box[2] = {32u, 32u}, estr[2] = {1u, 1u};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void *>(base), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  EB_REQUIRE(r == CUDA_SUCCESS, ENDIA_B200_ECUDA, "fp16-pair product: cuTensorMapEncodeTiled (C) failed with code %d", (int)r);
  return ENDIA_B200_OK;
}

bool gemm_f16_available() { return encode_fn() != nullptr; }

// Ranges of K of an F16_STORE product: when its tiles leave half of the CTA pairs idle, each tile's
// reduction is cut into up to 16 ranges of at least 512.
static int k_ranges(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ceil_div(M, 256) * ceil_div(N, 256), cap = pair_capacity();
  if (2 * tiles > cap) return 1;
  int64_t sp = cap / tiles;
  if (sp > K / 512) sp = K / 512;
  if (sp > 16) sp = 16;
  return sp >= 2 ? (int)sp : 1;
}
size_t gemm_f16_partial_bytes(int64_t M, int64_t N, int64_t K) {
  const int sp = k_ranges(M, N, K);
  return sp < 2 ? 0 : sizeof(float) * (size_t)sp * (size_t)(ceil_div(M, 256) * 256) * (size_t)(ceil_div(N, 4) * 4);
}

template <bool A_MN, bool B_MN, int PROD, int EPI>
static int launch_kernel(const F16Maps &maps, const F16Params &p, cudaStream_t s) {
  constexpr int STAGES = PROD == 3 ? 3 : 4;
  constexpr size_t SMEM = (size_t)STAGES * ((PROD == 3 ? 4 : 3) * F16_TILE) + F16_EPI_WARPS * 4096 + 1024 + 256;
  auto kern = gemm_f16_kernel<A_MN, B_MN, PROD, EPI>;
  static int max_pairs = 0;
  if (!max_pairs) {
    EB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(F16_THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int nc = 0;
    if (cudaOccupancyMaxActiveClusters(&nc, kern, &cfg) != cudaSuccess || nc <= 0) {
      cudaGetLastError();
      nc = (sm_count() > 0 ? sm_count() : 148) / 2;
    }
    max_pairs = nc < pair_capacity() ? nc : pair_capacity();
  }
  const int items = p.pairs_m * p.tiles_n * p.ksplit, pairs = items < max_pairs ? items : max_pairs;
  kern<<<dim3((unsigned)(2 * pairs)), F16_THREADS, SMEM, s>>>(maps, p);
  EB_LAUNCH_CHECK();
  return ENDIA_B200_OK;
}

int launch_gemm_f16(const F16Gemm &g, bool a_mn, bool b_mn, int epilogue, cudaStream_t s) {
  EB_REQUIRE(gemm_f16_available(), ENDIA_B200_ECUDA, "fp16-pair product: the driver has no cuTensorMapEncodeTiled");
  EB_REQUIRE(g.M >= 1 && g.N >= 1 && g.K >= 1 && g.M <= (1 << 30) && g.N <= (1 << 30) && g.K <= (1 << 30),
             ENDIA_B200_ELIMIT, "fp16-pair product: sizes must lie in [1, 2^30]");
  F16Maps maps;
  F16Params p{};
  int st;
  const int64_t a_in = a_mn ? g.M : g.K, a_out = a_mn ? g.K : g.M, b_in = b_mn ? g.N : g.K, b_out = b_mn ? g.K : g.N;
  const int a_box = a_mn ? F16_BK : 128, b_box = b_mn ? F16_BK : 128;
  const bool exact_a = g.a.lo == nullptr;
  if ((st = make_map_16(&maps.a_hi, g.a.hi, a_in, a_out, g.a.ld, a_box))) return st;
  if ((st = make_map_16(&maps.a_lo, exact_a ? g.a.hi : g.a.lo, a_in, a_out, g.a.ld, a_box))) return st;
  if ((st = make_map_16(&maps.b_hi, g.b.hi, b_in, b_out, g.b.ld, b_box))) return st;
  if ((st = make_map_16(&maps.b_lo, g.b.lo, b_in, b_out, g.b.ld, b_box))) return st;
  maps.c = maps.d_hi = maps.d_lo = maps.a_hi;
  p.M = (int)g.M; p.N = (int)g.N;
  p.pairs_m = (int)ceil_div(g.M, 256); p.tiles_n = (int)ceil_div(g.N, 256);
  p.group_m = 8;
  p.nkb = (int)ceil_div(g.K, F16_BK);
  p.ksplit = 1;
  p.ea = g.a.e; p.ea_ld = g.a.e_ld; p.a_last = (int)half_blocks(g.M) - 1;
  p.eb = g.b.e; p.eb_ld = g.b.e_ld; p.b_last = (int)half_blocks(g.N) - 1;
  p.alpha_dev = g.alpha_dev; p.alpha_exp = g.alpha_exp; p.bias = g.bias;
  p.C = g.C; p.ldc = g.ldc; p.act = g.act; p.accumulate = g.accumulate ? 1 : 0;
  p.target = g.target; p.n_base = g.n_base; p.stats = g.stats; p.target_logit = g.target_logit;
  p.lse = g.lse; p.coef = g.coef; p.colsum_part = g.colsum_part;
  EB_REQUIRE((int64_t)p.pairs_m * p.tiles_n <= (1 << 26), ENDIA_B200_ELIMIT, "fp16-pair product: too many tiles");
  if (epilogue == F16_STATS) {
    if (!a_mn && b_mn && !exact_a) return launch_kernel<false, true, 3, F16_STATS>(maps, p, s);
  } else if (epilogue == F16_DLOGITS) {
    if ((st = make_map_16(&maps.d_hi, g.d_hi, g.N, g.M, g.ld_d, 32, 32))) return st;
    if ((st = make_map_16(&maps.d_lo, g.d_lo, g.N, g.M, g.ld_d, 32, 32))) return st;
    if (!a_mn && b_mn && !exact_a) return launch_kernel<false, true, 3, F16_DLOGITS>(maps, p, s);
  } else {
    const int sp = g.partial ? k_ranges(g.M, g.N, g.K) : 1;
    const int64_t ldp = ceil_div(g.N, 4) * 4;
    p.vec_c = aligned16(g.C) && g.ldc % 4 == 0;
    if (sp > 1) {
      p.ksplit = sp;
      p.part_rows = p.pairs_m * 256;
      if ((st = make_map_32(&maps.c, g.partial, g.N, (int64_t)sp * p.part_rows, ldp))) return st;
    } else if (p.vec_c) {
      if ((st = make_map_32(&maps.c, g.C, g.N, g.M, g.ldc))) return st;
    }
    if (!a_mn && b_mn && !exact_a) st = launch_kernel<false, true, 3, F16_STORE>(maps, p, s);
    else if (!a_mn && !b_mn && !exact_a) st = launch_kernel<false, false, 3, F16_STORE>(maps, p, s);
    else if (a_mn && b_mn && !exact_a) st = launch_kernel<true, true, 3, F16_STORE>(maps, p, s);
    else if (a_mn && b_mn) st = launch_kernel<true, true, 2, F16_STORE>(maps, p, s);
    else { set_error("fp16-pair product: no kernel for these layouts"); return ENDIA_B200_EINVAL; }
    if (st || sp < 2) return st;
    gemm_f16_finish_kernel<<<grid_for(g.M * ceil_div(g.N, 4), 256), 256, 0, s>>>(p, g.partial, ldp, (int64_t)p.part_rows * ldp, sp);
    EB_LAUNCH_CHECK();
    return ENDIA_B200_OK;
  }
  set_error("fp16-pair product: no kernel for these layouts");
  return ENDIA_B200_EINVAL;
}

int f16_status_and_clear(cudaStream_t s) {
  int h = 0;
  if (cudaStreamSynchronize(s) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&h, g_tc_status, sizeof(int)) != cudaSuccess) return -1;
  if (h) {
    int z = 0;
    cudaMemcpyToSymbol(g_tc_status, &z, sizeof(int));
  }
  return h;
}

}  // namespace eb
