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
//   fp4_kernel<FMT, XR, GATED, PAIR>
//     XR = 16, 64       single CTAs, two per SM, two accumulators, so that the drain of a tile overlaps the next one's products
//     XR = 128          the same, one per SM
//     XR = 256, pairs   (cta_group::2) 256 x 256 tiles: each CTA brings 128 rows of W and half of the rows of X, and an MMA reads both: half the
//                       L2 traffic per product, which is what bounds 4-bit tiles (128 x 128: 32 KB per 8.4 Mflop).
//                       One accumulator: the scales take the rest of tensor memory; sixteen warps drain it into registers at once
//                       and hand it back before they work on it.
//     few tiles         a cluster of 2 to 8 CTAs shares a tile along K: partial sums meet in shared memory, added in the order of the ranks
//
// All waits are bounded (ptx_sm100.cuh).  No load is a multicast.
#pragma once
#include "host_util.h"
#include "lowbit.cuh"

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
  int by16;                                   // y (and residual, gate, bias) in pieces of 16 bytes
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
  static constexpr int CTAS = XR <= 64 ? 2 : 1;                                // per SM
  static constexpr int PARTS = XR == 16 ? 1 : PAIR ? 4 : 2;                    // draining warps per quadrant of tensor memory
  static constexpr int CHUNKS = XR / 16 / PARTS;                               // of 16 rows of X, per draining warp
  static constexpr int DRAIN_WARPS = 4 * PARTS, THREADS = 64 + 32 * DRAIN_WARPS;
  static constexpr int TURN_BYTES = DRAIN_WARPS * 2048;                        // 16 x 32 fp32 per draining warp
  static constexpr int STAGE_PITCH = (STAGE_BYTES + 1023) / 1024 * 1024;       // codes begin on 1024 bytes (swizzle)
  static constexpr int TMEM_COLS = 512 / CTAS;
  static constexpr int BY_SMEM = (226 * 1024 / CTAS - 1024 - TURN_BYTES) / STAGE_PITCH, BY_TMEM = (TMEM_COLS - ACCS * XR) / SCALE_COLS;
  static constexpr int STAGES = BY_SMEM < BY_TMEM ? BY_SMEM : BY_TMEM;
  static constexpr int SMEM_BYTES = STAGES * STAGE_PITCH + TURN_BYTES + 1024;
};

enum Fp4Act : int { FP4_NONE = 0, FP4_GELU_TANH = 1, FP4_SILU = 2 };

// x / (1 + e^-x); the quotient is good to 2 steps of fp32
__device__ __forceinline__ float silu_of(float x) { return __fdividef(x, 1.0f + __expf(-x)); }
// 0.5 x (1 + tanh u) = x / (1 + e^-2u)
__device__ __forceinline__ float gelu_of(float x) {
  const float u = 0.7978845608028654f * x * fmaf(0.044715f * x, x, 1.0f);
  return __fdividef(x, 1.0f + __expf(-2.0f * u));
}

// One result of row m of X: weight row n of the matrix (already times both factors).
__device__ __forceinline__ float fp4_finish(const Fp4Args& a, float v, long m, int n) {
  if (a.bias) v += __bfloat162float(a.bias[n]);
  v = a.act == FP4_SILU ? silu_of(v) : a.act == FP4_GELU_TANH ? gelu_of(v) : v;
  if (a.gate) v *= __bfloat162float(a.gate[m / a.rows_per_gate * a.gate_stride + n]);
  if (a.residual) v += __bfloat162float(a.residual[m * a.ldr + n]);
  return v;
}

__device__ __forceinline__ void add8(float (&v)[8], const uint4& u) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  v[0] += a.x; v[1] += a.y; v[2] += b.x; v[3] += b.y; v[4] += c.x; v[5] += c.y; v[6] += d.x; v[7] += d.y;
}
__device__ __forceinline__ void mul8(float (&v)[8], const uint4& u) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  v[0] *= a.x; v[1] *= a.y; v[2] *= b.x; v[3] *= b.y; v[4] *= c.x; v[5] *= c.y; v[6] *= d.x; v[7] *= d.y;
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// 16 rows of X by 32 rows of W, as a warp's accumulator lanes hold them (a lane per weight row), out to memory: turned in 2 KB of the
// warp's own, so that a lane gets eight neighbouring outputs of a row and loads and stores go in 16 bytes.  m0: the first row of X, n0: the
// warp's first weight row; rows: how many of the 16 there are; wf: the factor of this lane's weight row, xf: of row lane % 16 of X.  The
// factors were loaded before the tile was waited for, bias and residual are before the turn: a load where it is used costs its latency per
// chunk (768 -> 2048 for 2463 tokens of 128 experts 103 us, FIXME).
template <bool GATED>
__device__ __forceinline__ void fp4_store(const Fp4Args& a, const uint32_t* v, float* turned, long m0, int rows, int n0, float wf, float xf,
                                          int lane) {
  const int n = n0 + (lane & 3) * 8;
  uint4 res[2], bias8;
  if (!GATED && a.bias && a.by16 && n < a.N) bias8 = *reinterpret_cast<const uint4*>(a.bias + n);
  if (!GATED && a.residual && a.by16) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 8 + (lane >> 2);
      if (r < rows && n < a.N) res[i] = *reinterpret_cast<const uint4*>(a.residual + (m0 + r) * a.ldr + n);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) turned[i * 32 + lane] = __uint_as_float(v[i]) * wf;
  __syncwarp();
  if (GATED) {
    const int r = lane >> 1, g = (lane & 1) * 16, o = (n0 + g) / 2;
    const float f = __shfl_sync(0xffffffffu, xf, r);
    if (r < rows && o < a.N / 2) {
      const float* p = turned + r * 32 + g;
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = silu_of(p[e] * f) * (p[8 + e] * f);
      bf16* out = a.y + (m0 + r) * a.ldy + o;
      if (a.by16) *reinterpret_cast<uint4*>(out) = pack8(w);                   // N / 2 is a multiple of 8
      else
        for (int e = 0; e < 8; ++e) out[e] = __float2bfloat16(w[e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 8 + (lane >> 2);
      const float f = __shfl_sync(0xffffffffu, xf, r);
      if (r < rows && n < a.N) {
        const long m = m0 + r;
        const float4* p = reinterpret_cast<const float4*>(turned + r * 32 + (lane & 3) * 8);
        const float4 lo = p[0], hi = p[1];
        float w[8] = {lo.x * f, lo.y * f, lo.z * f, lo.w * f, hi.x * f, hi.y * f, hi.z * f, hi.w * f};
        bf16* out = a.y + m * a.ldy + n;
        if (a.by16) {
          if (a.bias) add8(w, bias8);
          if (a.act == FP4_SILU) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = silu_of(w[e]);
          } else if (a.act == FP4_GELU_TANH) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = gelu_of(w[e]);
          }
          if (a.gate) mul8(w, *reinterpret_cast<const uint4*>(a.gate + m / a.rows_per_gate * a.gate_stride + n));
          if (a.residual) add8(w, res[i]);
          *reinterpret_cast<uint4*>(out) = pack8(w);
        } else {
          for (int e = 0; e < 8 && n + e < a.N; ++e) out[e] = __float2bfloat16(fp4_finish(a, w[e], m, n + e));
        }
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* tmap, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

// a tile of rows: which expert, its first row in X and y, how many rows, and where its scales begin
struct RowTile {
  int expert, rows, scale_tile;
  long row0;
};
template <int XR>
__device__ __forceinline__ bool row_tile(const Fp4Args& a, int t, RowTile& r) {
  if (a.tile_expert) {
    r.expert = a.tile_expert[t];
    if (r.expert < 0) return false;           // used tiles come first
    r.row0 = a.tile_row0[t];
    r.rows = a.tile_rows[t];
    r.scale_tile = t * (XR > 128 ? 2 : 1);
    return true;
  }
  r.expert = 0;
  r.row0 = (long)t * XR;
  r.rows = min(XR, a.M - t * XR);
  r.scale_tile = t * (XR > 128 ? 2 : 1);      // XR = 64 has one tile only, or an expert's
  return true;
}

template <int FMT, int XR, bool GATED, bool PAIR>
__global__ void __launch_bounds__(Fp4Cfg<FMT, XR, PAIR>::THREADS, Fp4Cfg<FMT, XR, PAIR>::CTAS)
fp4_kernel(const __grid_constant__ Fp4Args a, int* status) {
  using Cfg = Fp4Cfg<FMT, XR, PAIR>;
  constexpr int STAGES = Cfg::STAGES, ACCS = Cfg::ACCS, STEP = PAIR ? 32 : 16;         // steps of an MMA's N
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[STAGES];               // pairs: in the even CTA, the bytes of both
  __shared__ __align__(8) uint64_t empty_bar[STAGES];
  __shared__ __align__(8) uint64_t tfull_bar[ACCS];
  __shared__ __align__(8) uint64_t tempty_bar[ACCS];               // pairs: in the even CTA, the warps of both
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int share = !PAIR && a.split > 1 ? (int)cluster_ctarank() : 0;                 // this CTA's part of K
  const int group = PAIR ? 2 : a.split;                                                // CTAs that work on an item
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
  if (PAIR || a.split > 1) cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s, tmem_scales = tmem_base + ACCS * XR;
  // item -> (block of weight rows, tile of rows).  One matrix: tiles of rows first, so that neighbours share the weights and all of X, which is small in 4
  // bits, stays in L2.  Experts: blocks of weight rows first; the tiles of an expert follow one another and share its weights.
  const bool experts = a.tile_expert != nullptr;
  auto tile_of = [&](int it) { return experts ? it / num_n : it % a.max_tiles; };
  auto block_of = [&](int it) { return (experts ? it % num_n : it / a.max_tiles) * (PAIR ? 2 : 1) + rank; };

  // the first stages' weights into L2 while the kernel before (the rows' quantiser) runs out
  if (!experts && warp == 0 && first < num_items && elect_one())
    for (int kb = kb0; kb < kb1 && kb < kb0 + STAGES; ++kb) tma_prefetch_3d(&a.tmW, kb * 128, block_of(first) * 128, 0);
  __syncwarp();
  pdl_begin();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int it = first; it < num_items; it += step) {
        RowTile t;
        if (!row_tile<XR>(a, tile_of(it), t)) break;
        const int nb = block_of(it), mine = PAIR ? (t.rows + 31) / 32 * 16 : t.rows, boxes = (mine + Cfg::BOX - 1) / Cfg::BOX;
        const int x0 = (int)t.row0 + rank * mine;
        const uint32_t bytes = Cfg::W_BYTES + boxes * Cfg::BOX * 128 + Cfg::WS_BYTES + Cfg::XS_BYTES;
        for (int kb = kb0; kb < kb1; ++kb) {
          mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1, &s_abort, status, ERR_WAIT_EMPTY);
          const uint32_t s = smem_base + stage * Cfg::STAGE_PITCH, sx = s + Cfg::W_BYTES, sws = sx + Cfg::X_BYTES, sxs = sws + Cfg::WS_BYTES;
          if (PAIR) {
            if (rank == 0) mbar_expect_tx(smem_u32(&full_bar[stage]), 2 * bytes);
            const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), 0);
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
      for (int it = first; it < num_items; it += step) {
        RowTile t;
        if (!row_tile<XR>(a, tile_of(it), t)) break;
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
            tc_commit_pair(mapa_shared(smem_u32(&empty_bar[stage]), 0));
            tc_commit_pair(mapa_shared(smem_u32(&empty_bar[stage]), 1));
          } else {
            tc_commit(smem_u32(&empty_bar[stage]));
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (PAIR) {
          tc_commit_pair(mapa_shared(smem_u32(&tfull_bar[acc]), 0));
          tc_commit_pair(mapa_shared(smem_u32(&tfull_bar[acc]), 1));
        } else {
          tc_commit(smem_u32(&tfull_bar[acc]));
        }
        if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;                // quadrant of tensor memory; which share of the tile's rows of X
    float* turned = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE_PITCH + (warp - 2) * 2048);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int it = first; it < num_items; it += step) {
      RowTile t;
      if (!row_tile<XR>(a, tile_of(it), t)) break;
      const int n0 = block_of(it) * 128 + q * 32, c0 = part * 16 * Cfg::CHUNKS;
      const float wf = a.wf && n0 + lane < a.N ? a.wf[(long)t.expert * a.N + n0 + lane] : 1.0f;
      float xf[Cfg::CHUNKS];
#pragma unroll
      for (int i = 0; i < Cfg::CHUNKS; ++i) {
        const int r = c0 + i * 16 + (lane & 15);
        xf[i] = a.xf && r < t.rows ? a.xf[t.row0 + r] : 1.0f;
      }
      mbar_wait(smem_u32(&tfull_bar[acc]), acc_phase, &s_abort, status, ERR_WAIT_TMEM_FULL);
      tc_fence_after_sync();
      const uint32_t at = tmem_base + ((uint32_t)(q * 32) << 16) + acc * XR + c0;
      if (PAIR) {
        // 64 of the 256 rows per warp, into registers; then the accumulator is free
        uint32_t v[Cfg::CHUNKS][16];
#pragma unroll
        for (int i = 0; i < Cfg::CHUNKS; ++i) tmem_ld_32x16(at + i * 16, v[i]);
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty_bar[acc]), 0));
#pragma unroll
        for (int i = 0; i < Cfg::CHUNKS; ++i) {
          const int c = c0 + i * 16;
          if (c < t.rows) fp4_store<GATED>(a, v[i], turned, t.row0 + c, t.rows - c, n0, wf, xf[i], lane);
        }
      } else {
        // split: this CTA's sums [row of X][128] to its ring, which nothing reads any more
        float* sums = reinterpret_cast<float*>(smem) + q * 32 + lane;
#pragma unroll
        for (int i = 0; i < Cfg::CHUNKS; ++i) {
          const int c = c0 + i * 16;
          if (c >= t.rows) break;
          uint32_t v[16];
          tmem_ld_32x16(at + i * 16, v);
          tmem_wait_ld();
          if (a.split == 1) {
            fp4_store<GATED>(a, v, turned, t.row0 + c, t.rows - c, n0, wf, xf[i], lane);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(c + j) * 128] = __uint_as_float(v[j]) * wf;
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[acc]));
      }
      if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
    }
  }

  if (!PAIR && a.split > 1) {
    __syncwarp();
    cluster_sync_all();
    RowTile t;
    if (first < num_items && row_tile<XR>(a, tile_of(first), t)) {
      // every CTA finishes 128 / split of the weight rows (at least 16: a gate group and its lift rows), all rows of X, four at a time
      const int width = 128 / a.split, base = share * width, n0 = block_of(first) * 128 + base, outs = GATED ? width / 2 : width, quads = outs / 4;
      auto sum = [&](int r, int n, float (&s)[4]) {
        float4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < a.split) v[c] = ld_cluster_f32x4(mapa_shared(smem_base + (r * 128 + base + n) * 4, c));
        s[0] = v[0].x; s[1] = v[0].y; s[2] = v[0].z; s[3] = v[0].w;
#pragma unroll
        for (int c = 1; c < 8; ++c)
          if (c < a.split) { s[0] += v[c].x; s[1] += v[c].y; s[2] += v[c].z; s[3] += v[c].w; }
      };
      for (int i = threadIdx.x; i < t.rows * quads; i += blockDim.x) {
        const int r = i / quads, o = (i - r * quads) * 4;
        const long m = t.row0 + r;
        const float f = a.xf ? a.xf[m] : 1.0f;
        float s0[4], s1[4];
        if (GATED) {
          const int n = o / 8 * 16 + o % 8;
          sum(r, n, s0);
          sum(r, n + 8, s1);
          if (n0 + n < a.N)
#pragma unroll
            for (int e = 0; e < 4; ++e) a.y[m * a.ldy + n0 / 2 + o + e] = __float2bfloat16(silu_of(s0[e] * f) * (s1[e] * f));
        } else {
          sum(r, o, s0);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + o + e < a.N) a.y[m * a.ldy + n0 + o + e] = __float2bfloat16(fp4_finish(a, s0[e] * f, m, n0 + o + e));
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
  if (PAIR || a.split > 1) cluster_sync_all();   // nobody leaves while another may still signal it or read its sums
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

// How many pairs run at once: a persistent kernel of more would leave its last ones to a round of their own.
static int resident_pairs(const void* kernel, int threads, int smem) {
  static int cached = 0;
  if (cached) return cached;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count() & ~1);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
  (void)cudaGetLastError();
  return cached = n <= 0 || n > sm_count() / 2 ? sm_count() / 2 : n;
}

template <int FMT, int XR, bool GATED, bool PAIR>
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
  auto* kernel = fp4_kernel<FMT, XR, GATED, PAIR>;
  if (int e = ensure_dynamic_smem((const void*)kernel, Cfg::SMEM_BYTES, prepared)) return e;
  const long items = (long)a.max_tiles * ((a.N + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128));
  const int group = PAIR ? 2 : a.split, most = PAIR ? resident_pairs((const void*)kernel, Cfg::THREADS, Cfg::SMEM_BYTES) : Cfg::CTAS * sm_count();
  const long run = a.split > 1 ? items : items < most ? items : most;
  if (run <= 0 || run * group > 0x7fffffffL) return RC_BAD_ARG;
  return launch_with(true, group, kernel, (unsigned)(run * group), Cfg::THREADS, Cfg::SMEM_BYTES, stream, a, status);
}

template <int FMT, bool GATED>
static int launch_rows_of(Fp4Args& a, const Fp4Operands& o, int tile, int* status, cudaStream_t s) {
  switch (tile) {
    case 16: return launch_fp4<FMT, 16, GATED, false>(a, o, status, s);
    case 64: return launch_fp4<FMT, 64, GATED, false>(a, o, status, s);
    case 128: return launch_fp4<FMT, 128, GATED, false>(a, o, status, s);
    case 256: return launch_fp4<FMT, 256, GATED, true>(a, o, status, s);
    default: return RC_BAD_ARG;
  }
}

static int launch_any(Fp4Args& a, const Fp4Operands& o, int fmt, bool gated, int tile, int* status, cudaStream_t s) {
  if (fmt == FMT_MXFP4) return gated ? launch_rows_of<FMT_MXFP4, true>(a, o, tile, status, s) : launch_rows_of<FMT_MXFP4, false>(a, o, tile, status, s);
  if (fmt == FMT_NVFP4) return gated ? launch_rows_of<FMT_NVFP4, true>(a, o, tile, status, s) : launch_rows_of<FMT_NVFP4, false>(a, o, tile, status, s);
  return RC_BAD_ARG;
}

// Tile and split of a linear layer: the tile's rows, or a negative code.
static int pick_tiles(Fp4Args& a, int force_tile, int force_split) {
  const int tile = force_tile ? force_tile : a.M <= 16 ? 16 : a.M <= 64 ? 64 : a.M <= 128 ? 128 : 256;
  if ((tile != 16 && tile != 64 && tile != 128 && tile != 256) || (tile <= 64 && a.M > tile)) return RC_BAD_ARG;
  a.max_tiles = (int)(((long)a.M + tile - 1) / tile);
  a.split = 1;
  if (tile == 256) return force_split > 1 ? RC_BAD_ARG : tile;
  const long items = (long)a.max_tiles * ((a.N + 127) / 128), slots = (tile <= 64 ? 2 : 1) * sm_count();
  const int kb = (a.K + 255) / 256;
  if (force_split) a.split = force_split;
  else
    while (a.split < 8 && items * a.split * 2 <= slots && kb >= a.split * 4) a.split *= 2;
  if (a.split < 1 || a.split > 8 || (a.split & (a.split - 1)) || a.split > kb) return RC_BAD_ARG;
  return tile;
}

}  // namespace omni
