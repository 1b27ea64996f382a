// Products of 4-bit operands on the block-scaled tensor instructions (layouts and formats: lowbit.cuh):
//
//   y[m, n] = epilogue( xf[m] wf[n] sum_k X[m, k] W[n, k] )      X, W = e2m1 values times their blocks' scales; xf, wf fp32 factors per row (nvfp4)
//
// for linear layers of one row to many, and for all experts of a mixture in one launch.  The epilogue adds a bias, applies an activation, a
// gate per batch and a residual; gated weights (8 gate rows, their 8 lift rows, the next 8 gate rows ...) give silu(gate) * lift.
//
// The weights are the M side of the MMA (128 rows of W per CTA, K = 64 per instruction) and rows of X its N side: the N of an MMA goes in
// steps of 16, so few rows cost little, and a tile of an expert has any number of them.  A stage of the shared-memory ring holds 256
// elements of K (one 128-byte swizzle row of codes) of both operands and their scale tiles; the issuing thread copies the scales to
// tensor memory (columns of their own per stage, free again when the stage is) and issues the MMAs that read them.
//
//   fp4_kernel<FMT, XR, EPI, PAIR>
//     XR = 16, 64, 128  single CTAs, two accumulators, so that the drain of a tile overlaps the next one's products
//     XR = 256, pairs   (cta_group::2) 256 x 256 tiles: each CTA brings 128 rows of W and half of the rows of X, and an MMA reads both: half the
//                       L2 traffic per product, which is what bounds 4-bit tiles (128 x 128: 32 KB per 8.4 Mflop).
//                       One accumulator: the scales take the rest of tensor memory; sixteen warps drain it into registers at once
//                       and hand it back before they work on it.  8192 x 24576 x 4096, nvfp4, SwiGLU: 322 us, 5.1 PFLOP/s, tensor pipe 69 % busy; loads
//                       alone 78 % of the time (8192 x 8192 x 4096: 88 of 113 us, 14.3 TB/s).  In 128-row tiles on single CTAs 478 us.
//     One row of 24576 x 4096, nvfp4: 12.6 us alone (57 MB at 4.5 TB/s), 13.8 with its quantisation before it, during which
//     the first weights come; 33 x 4096 x 12288 in four shares 10.0 us.
//     few tiles         2 or 4 CTAs (2 pairs) of a cluster share a tile along K; each finishes its part of the outputs from the sums of all
//
// All waits are bounded (ptx_sm100.cuh).  No load is a multicast.
#pragma once
#include "host_util.h"
#include "lowbit.cuh"
#include "per_device.h"

namespace omni {

struct Fp4Args {
  CUtensorMap tmW, tmWS, tmX, tmXS;
  bf16* y;
  long ldy;
  const float *wf, *xf;                       // factors of the rows of W (per expert one after another) and of X, or null
  const bf16 *bias, *residual, *gate;
  long ldr, gate_stride;
  int rows_per_gate, act;
  int M, N, K;                                // rows of X, rows of W (of an expert), contraction
  const int *tile_expert, *tile_row0, *tile_rows;        // null: one matrix, tiles of XR rows
  int max_tiles, split;                       // tiles of rows, CTAs that share a tile along K
  int by16;                                   // y and residual in pieces of 16 bytes (gates and biases are read one by one)
};

template <int FMT, int XR, bool PAIR>
struct Fp4Cfg {
  static constexpr int WORDS = FMT == FMT_MXFP4 ? 2 : 4;                       // scale words per row and stage
  static constexpr int X_ROWS = PAIR ? XR / 2 : XR;                            // rows of X in this CTA's shared memory
  static constexpr int X_TILES = XR > 128 ? 2 : 1;                             // scale tiles of 128 rows of X: a pair's CTAs both hold them all
  static constexpr int W_BYTES = 128 * 128, X_BYTES = X_ROWS * 128, WS_BYTES = WORDS * 512, XS_BYTES = X_TILES * WORDS * 512;
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + WS_BYTES + XS_BYTES;
  static constexpr int BOX = PAIR ? 32 : XR < 64 ? XR : 64;                    // rows of X per load
  static constexpr int ACCS = PAIR ? 1 : 2, SCALE_COLS = 4 * WORDS * (1 + X_TILES);
  static constexpr int CTAS = XR <= 16 ? 2 : 1;                                // per SM
  static constexpr int PARTS = XR == 16 ? 1 : PAIR ? 4 : 2;                    // draining warps per quadrant of tensor memory
  static constexpr int CHUNKS = XR / 16 / PARTS;                               // of 16 rows of X, per draining warp
  static constexpr int DRAIN_WARPS = 4 * PARTS, THREADS = 64 + 32 * DRAIN_WARPS;
  static constexpr int TURN_BYTES = DRAIN_WARPS * 1024;                        // 16 x 32 bf16 per draining warp
  static constexpr int STAGE_PITCH = (STAGE_BYTES + 1023) / 1024 * 1024;       // codes begin on 1024 bytes (swizzle)
  static constexpr int TMEM_COLS = 512 / CTAS;
  // an SM has 228 KB, of which every CTA takes 1 KB, up to 1 KB to begin on 1024 bytes and its barriers
  static constexpr int BY_SMEM = (228 * 1024 / CTAS - 2560 - TURN_BYTES) / STAGE_PITCH, BY_TMEM = (TMEM_COLS - ACCS * XR) / SCALE_COLS;
  static constexpr int STAGES = BY_SMEM < BY_TMEM ? BY_SMEM : BY_TMEM;
  static constexpr int SMEM_BYTES = STAGES * STAGE_PITCH + TURN_BYTES + 1024;
  static_assert(XR * 512 <= STAGES * STAGE_PITCH, "sums of a split tile lie in the ring");
};

enum Fp4Act : int { FP4_NONE = 0, FP4_GELU_TANH = 1, FP4_SILU = 2 };
// the sums; silu(gate) * lift; bias and activation where given; these and a gate and a residual
enum Fp4Epilogue : int { EPI_PLAIN = 0, EPI_GATED = 1, EPI_ACT = 2, EPI_ANY = 3 };

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x / (1 + e^-x), by a reciprocal and a power of two each good to two steps of fp32
__device__ __forceinline__ float silu_of(float x) { return x * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * x)); }
// 0.5 x (1 + tanh u) = x / (1 + e^-2u), u = sqrt(2 / pi) (x + 0.044715 x^3)
__device__ __forceinline__ float gelu_of(float x) {
  constexpr float C = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
  return x * rcp_approx(1.0f + ex2_approx(x * fmaf(C * 0.044715f, x * x, C)));
}

// One result of row m of X: weight row n of the matrix (already times both factors).
__device__ __forceinline__ float fp4_finish(const Fp4Args& a, float v, long m, int n, bool residual) {
  if (a.bias) v += __bfloat162float(a.bias[n]);
  v = a.act == FP4_SILU ? silu_of(v) : a.act == FP4_GELU_TANH ? gelu_of(v) : v;
  if (a.gate) v *= __bfloat162float(a.gate[m / a.rows_per_gate * a.gate_stride + n]);
  if (residual && a.residual) v += __bfloat162float(a.residual[m * a.ldr + n]);
  return v;
}

// eight neighbouring values of which n exist, where they do not begin on 16 bytes
__device__ __forceinline__ void store_some(bf16* p, const uint4& u, int n) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) p[e] = __ushort_as_bfloat16((unsigned short)(w[e >> 1] >> (16 * (e & 1))));
}
__device__ __forceinline__ uint4 load_some(const bf16* p, int n) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) w[e >> 1] |= (uint32_t)__bfloat16_as_ushort(p[e]) << (16 * (e & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// What a draining lane keeps of a tile, loaded while the tile is waited for: factors and biases of weight rows n0 + 8 i + lane / 4 of its warp's 32.
template <int EPI> struct Fp4Lane {
  float wf[4], bias[EPI >= EPI_ACT ? 4 : 1];
  __device__ __forceinline__ void load(const Fp4Args& a, long wf0, int n0, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 8 * i + (lane >> 2);
      wf[i] = a.wf && n < a.N ? a.wf[wf0 + n] : 1.0f;
      if (EPI >= EPI_ACT) bias[i] = a.bias && n < a.N ? __bfloat162float(a.bias[n]) : 0.0f;
    }
  }
};

// 16 rows of X by 32 rows of W out to memory.  v0, v1: the accumulator as fragments, for either half of the weight rows [8 rows of X][4], so that a lane holds
// for rows 2 (lane % 4) and the next of either eight the weight rows lane / 4 + 0, 8, 16, 24: the gate and the lift of an output are its own, factors and biases of
// weight rows stay for the tile, and the transposing matrix stores turn rounded results in 1 KB of the warp's own, from where they leave in pieces of 16
// bytes.  Residuals come in the same way.  m0: the first row, rows: how many there are; n0: the warp's first weight row; xf: the factor of row lane % 16.
// (A lane per weight row and a turn of fp32 took three times the instructions: 2463 tokens' rows of experts, 768 -> 2048, 121 us, 67 so.)
template <int EPI>
__device__ __forceinline__ void fp4_store(const Fp4Args& a, const uint32_t* v0, const uint32_t* v1, uint32_t turned, long m0, int rows, int n0,
                                          const Fp4Lane<EPI>& keep, float xf, int lane) {
  float f[4];                                                                  // factors of this lane's rows of X: eight g, column c at 2 g + c
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __shfl_sync(0xffffffffu, xf, (i >> 1) * 8 + 2 * (lane & 3) + (i & 1));
  if (EPI == EPI_GATED) {
    uint32_t o[4];                                                             // [half][eight rows]
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t* v = (h ? v1 : v0) + 4 * g;
        float r[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          r[c] = silu_of(__uint_as_float(v[c]) * keep.wf[2 * h] * f[2 * g + c]) * (__uint_as_float(v[2 + c]) * keep.wf[2 * h + 1] * f[2 * g + c]);
        o[2 * h + g] = pack_bf16(r[0], r[1]);
      }
    // 32 bytes per row of X; matrix (h, g) = (lane / 16, lane / 8 % 2)
    const int m = ((lane >> 3) & 1) * 8 + (lane & 7);
    stmatrix_x4_trans(turned + m * 32 + (((lane >> 4) ^ (m >> 2)) & 1) * 16, o[0], o[1], o[2], o[3]);
    __syncwarp();
    const int r = lane >> 1, h = lane & 1, col = n0 / 2 + h * 8;
    if (r < rows && col < a.N / 2) {
      const uint4 u = ld_shared_v4(turned + r * 32 + ((h ^ (r >> 2)) & 1) * 16);
      bf16* out = a.y + (m0 + r) * a.ldy + col;
      if (a.by16) *reinterpret_cast<uint4*>(out) = u;                          // N / 2 is a multiple of 8
      else store_some(out, u, 8);
    }
  } else {
    const int sm = ((lane >> 3) & 1) * 8 + (lane & 7), sn = lane >> 4;         // matrix (sn, eight) of a half: which row of 16 bytes this lane names
    const int rr = lane >> 2, rn = lane & 3, n = n0 + rn * 8;                  // what it moves: rows rr and rr + 8, outputs n ..
    auto at = [&](int m, int n8) { return turned + m * 64 + ((n8 ^ (m >> 1)) & 3) * 16; };
    if (EPI == EPI_ANY && a.residual) {
      uint4 u[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bf16* p = a.residual + (m0 + rr + 8 * i) * a.ldr + n;
        u[i] = make_uint4(0u, 0u, 0u, 0u);
        if (rr + 8 * i < rows && n < a.N) {
          if (a.by16) u[i] = *reinterpret_cast<const uint4*>(p);
          else u[i] = load_some(p, a.N - n);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) st_shared_v4(at(rr + 8 * i, rn), u[i]);
      __syncwarp();
    }
    float r[2][8];                                                             // [half][2 (2 s + g) + c]
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = i >> 2, g = (i >> 1) & 1, c = i & 1;
        r[h][i] = __uint_as_float((h ? v1 : v0)[4 * g + 2 * s + c]) * keep.wf[2 * h + s] * f[2 * g + c];
        if (EPI >= EPI_ACT) r[h][i] += keep.bias[2 * h + s];
      }
    if (EPI >= EPI_ACT) {
      // a step for all sixteen values at a time: they do not depend on one another, and the branches are the same for all
      if (a.act == FP4_SILU) {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i >> 3][i & 7] = silu_of(r[i >> 3][i & 7]);
      } else if (a.act == FP4_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i >> 3][i & 7] = gelu_of(r[i >> 3][i & 7]);
      }
      if (EPI == EPI_ANY && a.gate) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int h = i >> 3, s = (i >> 2) & 1, g = (i >> 1) & 1, c = i & 1;
          const int row = min(8 * g + 2 * (lane & 3) + c, rows - 1), col = min(n0 + 16 * h + 8 * s + (lane >> 2), a.N - 1);
          r[h][i & 7] *= __bfloat162float(a.gate[(m0 + row) / a.rows_per_gate * a.gate_stride + col]);
        }
      }
      if (EPI == EPI_ANY && a.residual) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t res[4];
          ldmatrix_x4_trans(at(sm, 2 * h + sn), res);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 t = unpack_bf16(res[i]);
            r[h][2 * i] += t.x;
            r[h][2 * i + 1] += t.y;
          }
        }
      }
    }
    uint32_t o[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[h][i] = pack_bf16(r[h][2 * i], r[h][2 * i + 1]);
    if (EPI == EPI_ANY && a.residual) __syncwarp();                            // everybody has read what they write over
#pragma unroll
    for (int h = 0; h < 2; ++h) stmatrix_x4_trans(at(sm, 2 * h + sn), o[h][0], o[h][1], o[h][2], o[h][3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = rr + 8 * i;
      if (r < rows && n < a.N) {
        const uint4 u = ld_shared_v4(at(r, rn));
        bf16* out = a.y + (m0 + r) * a.ldy + n;
        if (a.by16) *reinterpret_cast<uint4*>(out) = u;                        // N is a multiple of 8
        else store_some(out, u, a.N - n);
      }
    }
  }
  __syncwarp();                                                                // the next 16 rows are turned in the same place
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* tmap, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* tmap, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

constexpr int SPLIT_MOST = 4;    // CTAs or pairs that share a tile
// Stages of weights that a CTA asks for ahead of its first item.  One row of 24576 x 4096 with its quantisation: 14.2 us without, 13.8 with 4, 14.4 with 8,
// 15.8 with 16 (asked for ahead of what other CTAs need first).  64 tokens x 8 of 128 experts, 2048 -> 768 -> 2048: 51 us without, 47.5 with 4.
constexpr int PREFETCH = 4;

// a tile of rows: which expert, its first row in X and y, how many rows, and where its scales begin
struct RowTile {
  int expert, rows, scale_tile;
  long row0;
};
// Loads only, so that a role can ask for its next tile before it works on this one; expert < 0: no more tiles (used ones come first).
template <int XR>
__device__ __forceinline__ RowTile row_tile(const Fp4Args& a, int t) {
  RowTile r;
  r.scale_tile = t * (XR > 128 ? 2 : 1);      // XR = 16, 64: one tile only, or tiles of experts, whose scales begin anew
  if (a.tile_expert) {
    r.expert = a.tile_expert[t];
    r.row0 = a.tile_row0[t];
    r.rows = a.tile_rows[t];
  } else {
    r.expert = 0;
    r.row0 = (long)t * XR;
    r.rows = min(XR, a.M - t * XR);
  }
  return r;
}

template <int FMT, int XR, int EPI, bool PAIR>
__global__ void __launch_bounds__(Fp4Cfg<FMT, XR, PAIR>::THREADS, Fp4Cfg<FMT, XR, PAIR>::CTAS)
fp4_kernel(const __grid_constant__ Fp4Args a, int* status) {
  using Cfg = Fp4Cfg<FMT, XR, PAIR>;
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int STAGES = Cfg::STAGES, ACCS = Cfg::ACCS, STEP = PAIR ? 32 : 16;         // steps of an MMA's N
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES];               // pairs: in the even CTA, the bytes of both
  __shared__ __align__(8) uint64_t empty_bar[STAGES];
  __shared__ __align__(8) uint64_t tfull_bar[ACCS];
  __shared__ __align__(8) uint64_t tempty_bar[ACCS];               // pairs: in the even CTA, the warps of both
  __shared__ float xf_s[XR];                                       // split: factors of the tile's rows of X
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int SIZE = PAIR ? 2 : 1;
  const int group = SIZE * a.split, in_group = group > 1 ? (int)cluster_ctarank() : 0;  // CTAs that work on an item
  const int rank = in_group % SIZE, share = in_group / SIZE, even = share * SIZE;       // this CTA in its pair, its part of K, the pair's even CTA
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const int num_n = (a.N + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128), num_items = a.max_tiles * num_n;
  const int all_kb = (a.K + 255) / 256, kb0 = share * all_kb / a.split, kb1 = (share + 1) * all_kb / a.split;
  const int first = blockIdx.x / group, step = gridDim.x / group;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_u32(&full_bar[i]), 1);
      mbar_init(smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < ACCS; ++i) {
      mbar_init(smem_u32(&tfull_bar[i]), 1);
      mbar_init(smem_u32(&tempty_bar[i]), Cfg::DRAIN_WARPS * (PAIR ? 2 : 1));
    }
    fence_mbar_init();
    tma_prefetch_desc(&a.tmW);
    tma_prefetch_desc(&a.tmWS);
    tma_prefetch_desc(&a.tmX);
    tma_prefetch_desc(&a.tmXS);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(&tmem_base_s), Cfg::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_base_s), Cfg::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s, tmem_scales = tmem_base + ACCS * XR;
  // item -> (block of weight rows, tile of rows).  One matrix: tiles of rows first, so that neighbours share the weights and all of X, which is small in 4
  // bits, stays in L2.  Experts: blocks of weight rows first; the tiles of an expert follow one another and share its weights.
  const bool experts = a.tile_expert != nullptr;
  auto tile_of = [&](int it) { return experts ? it / num_n : it % a.max_tiles; };
  auto block_of = [&](int it) { return (experts ? it % num_n : it / a.max_tiles) * (PAIR ? 2 : 1) + rank; };

  auto tile_at = [&](int it) { return row_tile<XR>(a, tile_of(min(it, num_items - 1))); };

  // The first item's weights into L2 while the kernel before (the rows' quantiser) runs out.  Experts: the plan ran before that kernel, which let this one start
  // only when it had waited for the plan itself; what is asked for is in bounds or not fetched, whatever the table holds.
  if (warp == 0 && first < num_items && elect_one()) {
    const int expert = experts ? __ldcg(a.tile_expert + tile_of(first)) : 0;
    for (int kb = kb0; expert >= 0 && kb < kb1 && kb < kb0 + PREFETCH; ++kb) {
      tma_prefetch_3d(&a.tmW, kb * 128, block_of(first) * 128, expert);
      tma_prefetch_4d(&a.tmWS, 0, kb * Cfg::WORDS, block_of(first), expert);
    }
  }
  __syncwarp();
  pdl_begin();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      RowTile next = tile_at(first);
      for (int it = first; it < num_items; it += step) {
        const RowTile t = next;
        if (t.expert < 0) break;
        next = tile_at(it + step);
        const int nb = block_of(it), mine = PAIR ? (t.rows + 31) / 32 * 16 : t.rows, boxes = (mine + Cfg::BOX - 1) / Cfg::BOX;
        const int x0 = (int)t.row0 + rank * mine;
        const uint32_t bytes = Cfg::W_BYTES + boxes * Cfg::BOX * 128 + Cfg::WS_BYTES + Cfg::XS_BYTES;
        for (int kb = kb0; kb < kb1; ++kb) {
          mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1, &s_abort, status, ERR_WAIT_EMPTY);
          const uint32_t s = smem_base + stage * Cfg::STAGE_PITCH, sx = s + Cfg::W_BYTES, sws = sx + Cfg::X_BYTES, sxs = sws + Cfg::WS_BYTES;
          if (PAIR) {
            if (rank == 0) mbar_expect_tx(smem_u32(&full_bar[stage]), 2 * bytes);
            const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), even);
            tma_load_3d_pair(s, &a.tmW, fb, kb * 128, nb * 128, t.expert);
            tma_load_4d_pair(sws, &a.tmWS, fb, 0, kb * Cfg::WORDS, nb, t.expert);
            for (int b = 0; b < boxes; ++b) tma_load_2d_pair(sx + b * Cfg::BOX * 128, &a.tmX, fb, kb * 128, x0 + b * Cfg::BOX);
            tma_load_3d_pair(sxs, &a.tmXS, fb, 0, kb * Cfg::WORDS, t.scale_tile);
          } else {
            const uint32_t fb = smem_u32(&full_bar[stage]);
            mbar_expect_tx(fb, bytes);
            tma_load_3d(s, &a.tmW, fb, kb * 128, nb * 128, t.expert);
            tma_load_4d(sws, &a.tmWS, fb, 0, kb * Cfg::WORDS, nb, t.expert);
            for (int b = 0; b < boxes; ++b) tma_load_2d(sx + b * Cfg::BOX * 128, &a.tmX, fb, kb * 128, x0 + b * Cfg::BOX);
            tma_load_3d(sxs, &a.tmXS, fb, 0, kb * Cfg::WORDS, t.scale_tile);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      RowTile next = tile_at(first);
      for (int it = first; it < num_items; it += step) {
        const RowTile t = next;
        if (t.expert < 0) break;
        next = tile_at(it + step);
        const uint32_t n = (t.rows + STEP - 1) / STEP * STEP;
        const uint32_t idesc = fp4_idesc<FMT>(PAIR ? 256 : 128, n, 0);
        mbar_wait(smem_u32(&tempty_bar[acc]), acc_phase ^ 1, &s_abort, status, ERR_WAIT_TMEM_EMPTY);
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * XR;
        for (int kb = kb0; kb < kb1; ++kb) {
          mbar_wait(smem_u32(&full_bar[stage]), phase, &s_abort, status, ERR_WAIT_FULL);
          tc_fence_after_sync();
          const uint32_t s = smem_base + stage * Cfg::STAGE_PITCH, sx = s + Cfg::W_BYTES, sws = sx + Cfg::X_BYTES, sxs = sws + Cfg::WS_BYTES;
          const uint64_t w_desc = umma_desc_kmajor_sw128(s), x_desc = umma_desc_kmajor_sw128(sx);
          // a word of W's scales: 4 columns; of X's: 4 per 128 rows, side by side
          const uint32_t w_cols = tmem_scales + stage * Cfg::SCALE_COLS, x_cols = w_cols + 4 * Cfg::WORDS;
#pragma unroll
          for (int w = 0; w < Cfg::WORDS; ++w) {
            scales_to_tmem<PAIR>(w_cols + 4 * w, scale_tile_desc(sws + w * 512));
#pragma unroll
            for (int h = 0; h < Cfg::X_TILES; ++h)
              scales_to_tmem<PAIR>(x_cols + 4 * (Cfg::X_TILES * w + h), scale_tile_desc(sxs + (h * Cfg::WORDS + w) * 512));
          }
          const int steps = min(4, (a.K - kb * 256 + 63) / 64);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= steps) break;
            const int w = FMT == FMT_MXFP4 ? k / 2 : k;
            const uint32_t id = FMT == FMT_MXFP4 ? (k & 1) * 2 : 0;
            mma_fp4_ss<FMT, PAIR>(d_tmem, w_desc + 2 * k, x_desc + 2 * k, idesc | (id << 4) | (id << 29), w_cols + 4 * w,
                                  x_cols + 4 * Cfg::X_TILES * w, kb != kb0 || k != 0);
          }
          if (PAIR) {
            tc_commit_pair(mapa_shared(smem_u32(&empty_bar[stage]), even));
            tc_commit_pair(mapa_shared(smem_u32(&empty_bar[stage]), even + 1));
          } else {
            tc_commit(smem_u32(&empty_bar[stage]));
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (PAIR) {
          tc_commit_pair(mapa_shared(smem_u32(&tfull_bar[acc]), even));
          tc_commit_pair(mapa_shared(smem_u32(&tfull_bar[acc]), even + 1));
        } else {
          tc_commit(smem_u32(&tfull_bar[acc]));
        }
        if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;                // quadrant of tensor memory; which share of the tile's rows of X
    const uint32_t turned = smem_base + STAGES * Cfg::STAGE_PITCH + (warp - 2) * 1024;
    int acc = 0;
    uint32_t acc_phase = 0;
    RowTile next = tile_at(first);
    for (int it = first; it < num_items; it += step) {
      const RowTile t = next;
      if (t.expert < 0) break;
      next = tile_at(it + step);
      const int n0 = block_of(it) * 128 + q * 32, c0 = part * 16 * Cfg::CHUNKS;
      Fp4Lane<EPI> keep;
      keep.load(a, (long)t.expert * a.N, n0, lane);
      float xf[Cfg::CHUNKS];
#pragma unroll
      for (int i = 0; i < Cfg::CHUNKS; ++i) {
        const int r = c0 + i * 16 + (lane & 15);
        xf[i] = a.xf && r < t.rows ? a.xf[t.row0 + r] : 1.0f;
      }
      float wf = 1.0f;
      if (a.split > 1) {                                           // what finishing will need, while the tile is waited for
        if (a.wf && n0 + lane < a.N) wf = a.wf[n0 + lane];
        if (q == 0)
          for (int r = c0 + lane; r < min(t.rows, c0 + 16 * Cfg::CHUNKS); r += 32) xf_s[r] = a.xf ? a.xf[t.row0 + r] : 1.0f;
      }
      mbar_wait(smem_u32(&tfull_bar[acc]), acc_phase, &s_abort, status, ERR_WAIT_TMEM_FULL);
      tc_fence_after_sync();
      const uint32_t at = tmem_base + ((uint32_t)(q * 32) << 16) + acc * XR + c0, half = 16u << 16;
      if (a.split > 1) {
        // this CTA's sums to its ring, which its products no longer read, as blocks [owner][row of X][width]
        const int width = 128 / a.split, n = q * 32 + lane;
        float* to = reinterpret_cast<float*>(smem) + (n / width * t.rows + c0) * width + n % width;
#pragma unroll 1
        for (int c = 0; c < 16 * Cfg::CHUNKS && c0 + c < t.rows; c += 16) {
          uint32_t v[16];
          tmem_ld_32x16(tmem_base + ((uint32_t)(q * 32) << 16) + c0 + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + c + j < t.rows) to[(c + j) * width] = __uint_as_float(v[j]) * wf;
        }
        break;
      }
      if constexpr (PAIR) {
        // 64 of the 256 rows per warp, into registers; then the accumulator is free.  With a gate or a residual in two steps, for want of registers (18 warps leave
        // 96 a thread): 2390 x 8192 x 2048 with a residual 40 us, in one step 52; with a bias and GELU, which have a form of their own, 34 and 29.
        constexpr int STEPS = EPI == EPI_ANY ? 2 : 1, PER = Cfg::CHUNKS / STEPS;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          uint32_t v[2][8 * PER];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (PER == 4) tmem_ld_16x256_x8(at + h * half, v[h]);
            else tmem_ld_16x256_x4(at + h * half + j * 16 * PER, v[h]);
          tmem_wait_ld();
          if (j == STEPS - 1) {
            tc_fence_before_sync();
            __syncwarp();
            // relaxed: a release waits for the stores of the tile before, 8192 x 24576 x 4096 375 -> 322 us without, 2463 tokens of experts 182 -> 161
            if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&tempty_bar[acc]), even));
          }
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int c = c0 + (j * PER + i) * 16;
            if (c < t.rows) fp4_store<EPI>(a, v[0] + 8 * i, v[1] + 8 * i, turned, t.row0 + c, t.rows - c, n0, keep, xf[j * PER + i], lane);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < Cfg::CHUNKS; ++i) {
          const int c = c0 + i * 16;
          if (c >= t.rows) break;
          uint32_t v[2][8];
          tmem_ld_16x256_x2(at + i * 16, v[0]);
          tmem_ld_16x256_x2(at + i * 16 + half, v[1]);
          tmem_wait_ld();
          fp4_store<EPI>(a, v[0], v[1], turned, t.row0 + c, t.rows - c, n0, keep, xf[i], lane);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[acc]));
      }
      if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
    }
  }

  if (a.split > 1) {
    // Every CTA finishes 128 / split of the weight rows (at least 16: a gate group and its lift rows), all rows of X.  Sums lie in the rings as blocks
    // [owner][row of X][width]; the owner reads its block of every CTA where it lies and adds them in the order of the shares.
    __syncwarp();
    cluster_sync_all();
    if (first < num_items) {
      const RowTile t = tile_at(first);
      const int width = 128 / a.split, n0 = block_of(first) * 128 + share * width, outs = GATED ? width / 2 : width, quads = outs / 4, total = t.rows * quads;
      const uint32_t block = smem_base + share * t.rows * width * 4;
      auto column = [&](int o) { return GATED ? o / 8 * 16 + o % 8 : o; };       // of the block, where output o (or its gate) stands
      constexpr int COLS = GATED ? 2 : 1;                                        // gate and lift
      for (int i0 = threadIdx.x; i0 < total; i0 += 2 * blockDim.x) {             // four outputs of two rows at a time
        float sums[2][COLS][4];
        uint2 res[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = i0 + u * blockDim.x, r = i / quads, o = (i - r * quads) * 4;
          if (EPI == EPI_ANY && a.residual && a.by16 && i < total && n0 + o < a.N) res[u] = *reinterpret_cast<const uint2*>(a.residual + (t.row0 + r) * a.ldr + n0 + o);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int k = 0; k < COLS; ++k) {
            const int i = i0 + u * blockDim.x, r = i / quads, o = (i - r * quads) * 4;
            float4 v[SPLIT_MOST];
#pragma unroll
            for (int c = 0; c < SPLIT_MOST; ++c)
              v[c] = c < a.split && i < total ? ld_cluster_f32x4(mapa_shared(block + (r * width + column(o) + 8 * k) * 4, c * SIZE + rank)) : make_float4(0.f, 0.f, 0.f, 0.f);
            float(&s)[4] = sums[u][k];
            s[0] = v[0].x; s[1] = v[0].y; s[2] = v[0].z; s[3] = v[0].w;
#pragma unroll
            for (int c = 1; c < SPLIT_MOST; ++c) { s[0] += v[c].x; s[1] += v[c].y; s[2] += v[c].z; s[3] += v[c].w; }
          }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = i0 + u * blockDim.x, r = i / quads, o = (i - r * quads) * 4;
          if (i >= total || n0 + column(o) >= a.N) continue;
          const long m = t.row0 + r;
          const float f = xf_s[r];
          bf16* out = a.y + m * a.ldy + (GATED ? n0 / 2 : n0) + o;
          const int left = a.N - n0 - o;                                         // outputs that exist (gated: all)
          float(&s)[4] = sums[u][0];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[e] *= f;
            if (GATED) s[e] = silu_of(s[e]) * (sums[u][COLS - 1][e] * f);
            else if (EPI >= EPI_ACT && e < left) s[e] = fp4_finish(a, s[e], m, n0 + o + e, !a.by16);
          }
          if (EPI == EPI_ANY && a.residual && a.by16) {
            const float2 lo = unpack_bf16(res[u].x), hi = unpack_bf16(res[u].y);
            s[0] += lo.x; s[1] += lo.y; s[2] += hi.x; s[3] += hi.y;
          }
          if (a.by16) *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
          else
            for (int e = 0; e < 4 && (GATED || e < left); ++e) out[e] = __float2bfloat16(s[e]);
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (s_abort) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  if (group > 1) cluster_sync_all();            // nobody leaves while another may still signal it or copy from it
  if (warp == 1) {
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
    else tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// --------------------------------------------------------------------------------------------------------------- host
static int make_map(CUtensorMap* out, const void* p, CUtensorMapDataType dt, int dims, const uint64_t* size, const uint64_t* pitch, const uint32_t* box,
                    CUtensorMapSwizzle swizzle) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return RC_NO_DRIVER;
  if (reinterpret_cast<uintptr_t>(p) & 15) return RC_BAD_ARG;
  cuuint64_t gd[4], gs[3];
  cuuint32_t bx[4], es[4];
  for (int i = 0; i < dims; ++i) {
    gd[i] = size[i]; bx[i] = box[i]; es[i] = 1;
    if (i + 1 < dims) {
      if (pitch[i] & 15) return RC_BAD_ARG;
      gs[i] = pitch[i];
    }
  }
  const CUresult r = enc(out, dt, dims, const_cast<void*>(p), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? RC_OK : RC_TMAP;
}

struct Fp4Operands {
  const void *w, *ws, *x, *xs;
  int experts;
  long x_rows, xs_tiles;         // rows of X, its scale tiles of 128 rows
};

// How many pairs of a kernel run at once on the current device: a persistent kernel of more would leave its last ones to a round of their own.
static int resident_pairs(PerDevice& known, const void* kernel, int threads, int smem) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int half = sm_count() / 2;
  const int n = known.get(dev, half, [&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * half);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) clusters = 0;
    (void)cudaGetLastError();
    return clusters;
  });
  return n < half ? n : half;
}

template <int FMT, int XR, int EPI, bool PAIR>
static int launch_fp4(Fp4Args& a, const Fp4Operands& o, int* status, cudaStream_t stream) {
  using Cfg = Fp4Cfg<FMT, XR, PAIR>;
  const uint64_t K2 = a.K / 2, words = scale_words(FMT, a.K), blocks = (a.N + 127) / 128;
  const uint64_t wd[3] = {K2, (uint64_t)a.N, (uint64_t)o.experts}, wp[2] = {K2, K2 * a.N};
  const uint32_t wb[3] = {128, 128, 1};
  if (int rc = make_map(&a.tmW, o.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, wd, wp, wb, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  const uint64_t wsd[4] = {128, words, blocks, (uint64_t)o.experts}, wsp[3] = {512, 512 * words, 512 * words * blocks};
  const uint32_t wsb[4] = {128, Cfg::WORDS, 1, 1};
  if (int rc = make_map(&a.tmWS, o.ws, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, wsd, wsp, wsb, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
  const uint64_t xd[2] = {K2, (uint64_t)o.x_rows}, xp[1] = {K2};
  const uint32_t xb[2] = {128, Cfg::BOX};
  if (int rc = make_map(&a.tmX, o.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, xd, xp, xb, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  const uint64_t xsd[3] = {128, words, (uint64_t)o.xs_tiles}, xsp[2] = {512, 512 * words};
  const uint32_t xsb[3] = {128, Cfg::WORDS, Cfg::X_TILES};
  if (int rc = make_map(&a.tmXS, o.xs, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, xsd, xsp, xsb, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;

  static unsigned long long prepared = 0;
  static PerDevice pairs;
  auto* kernel = fp4_kernel<FMT, XR, EPI, PAIR>;
  if (int e = ensure_dynamic_smem((const void*)kernel, Cfg::SMEM_BYTES, prepared)) return e;
  const long items = (long)a.max_tiles * ((a.N + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128));
  const int group = (PAIR ? 2 : 1) * a.split, most = PAIR ? resident_pairs(pairs, (const void*)kernel, Cfg::THREADS, Cfg::SMEM_BYTES) : Cfg::CTAS * sm_count();
  const long run = a.split > 1 ? items : items < most ? items : most;
  if (run <= 0 || run * group > 0x7fffffffL) return RC_BAD_ARG;
  return launch_with(true, group, kernel, (unsigned)(run * group), Cfg::THREADS, Cfg::SMEM_BYTES, stream, a, status);
}

template <int FMT, int EPI>
static int launch_rows_of(Fp4Args& a, const Fp4Operands& o, int tile, int* status, cudaStream_t s) {
  switch (tile) {
    case 16: return launch_fp4<FMT, 16, EPI, false>(a, o, status, s);
    case 64: return launch_fp4<FMT, 64, EPI, false>(a, o, status, s);
    case 128: return launch_fp4<FMT, 128, EPI, false>(a, o, status, s);
    case 256: return launch_fp4<FMT, 256, EPI, true>(a, o, status, s);
    default: return RC_BAD_ARG;
  }
}

template <int FMT>
static int launch_epi(Fp4Args& a, const Fp4Operands& o, bool gated, int tile, int* status, cudaStream_t s) {
  if (gated) return launch_rows_of<FMT, EPI_GATED>(a, o, tile, status, s);
  if (a.gate || a.residual) return launch_rows_of<FMT, EPI_ANY>(a, o, tile, status, s);
  return a.bias || a.act ? launch_rows_of<FMT, EPI_ACT>(a, o, tile, status, s) : launch_rows_of<FMT, EPI_PLAIN>(a, o, tile, status, s);
}
static int launch_any(Fp4Args& a, const Fp4Operands& o, int fmt, bool gated, int tile, int* status, cudaStream_t s) {
  if (fmt == FMT_MXFP4) return launch_epi<FMT_MXFP4>(a, o, gated, tile, status, s);
  if (fmt == FMT_NVFP4) return launch_epi<FMT_NVFP4>(a, o, gated, tile, status, s);
  return RC_BAD_ARG;
}

// Tile and split of a linear layer: the tile's rows, or a negative code.
// Up to 16 rows: two CTAs per SM with tiles of 16 (16 rows of 24576 x 4096 12.4 us, in a tile of 64 14.2); up to 64: one (64 rows 14.5, in a tile of 128 15.3).
// More than 128 rows: 128-row tiles on single CTAs or 256-row tiles on pairs, by the rounds that each take.  In a full round a block of 256 of K costs 0.4 us
// on single CTAs and 0.5 on pairs (what L2 delivers), in a last round that is not full 0.3 and 0.4.  N x K = 4096 x 4096, 512 rows 8.7 us on single
// CTAs, 10.6 on pairs; 1000 rows 13.6 and 12.0; gated 24576 x 4096, 200 rows 19.0 and 18.0, 8192 rows 478 and 322.
// Few tiles: a split saves blocks of K (0.28 us each) and costs an exchange of 1.4 us and 14 ns per row, 0.6 more in fours.  4096 x 12288, 33 rows: 15.9 us
// whole, 12.3 in two, 10.0 in four; 200 rows 16.8 whole, 14.3 in two; 4096 x 1024, 33 rows: 3.9, 5.1, 5.7.  (Clusters of 8 of these CTAs, one per SM, do
// not all find room: 22 us.)  The limit counts one CTA per SM for tiles of 16 rows too, of which two run; what a split up to that would give was not measured.
static int pick_tiles(Fp4Args& a, int force_tile, int force_split) {
  const int sms = sm_count(), kb = (a.K + 255) / 256;
  int tile = force_tile ? force_tile : a.M <= 16 ? 16 : a.M <= 64 ? 64 : 128;
  if (!force_tile && a.M > 128) {
    const long single = ((long)a.M + 127) / 128 * ((a.N + 127) / 128), pairs = ((long)a.M + 255) / 256 * ((a.N + 255) / 256), slots = sms / 2;
    if (5 * (pairs / slots) + (pairs % slots ? 4 : 0) <= 4 * (single / sms) + (single % sms ? 3 : 0)) tile = 256;
  }
  if ((tile != 16 && tile != 64 && tile != 128 && tile != 256) || (tile <= 64 && a.M > tile)) return RC_BAD_ARG;
  const bool pair = tile == 256;
  a.max_tiles = (int)(((long)a.M + tile - 1) / tile);
  const long items = (long)a.max_tiles * (pair ? (a.N + 255) / 256 : (a.N + 127) / 128);
  const int most = pair ? 2 : SPLIT_MOST, rows = a.M < tile ? a.M : tile;
  a.split = 1;
  if (force_split) {
    a.split = force_split;
  } else {
    int least = 280 * kb;
    for (int s = 2; s <= most && s <= kb && items * s <= (pair ? sms / 2 : sms); s *= 2) {
      const int cost = 280 * ((kb + s - 1) / s) + 1400 + 14 * rows + (s > 2 ? 600 : 0);
      if (cost < least) { least = cost; a.split = s; }
    }
  }
  if (a.split < 1 || a.split > most || (a.split & (a.split - 1)) || a.split > kb) return RC_BAD_ARG;
  return tile;
}

}  // namespace omni
