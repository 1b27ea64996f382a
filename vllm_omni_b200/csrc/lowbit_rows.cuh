// Rows to 4 and 8 bits and back (layouts: lowbit.cuh): kernels and their launchers.
//
// All are bound by memory traffic for many rows and by one round trip for few, so a row is read once and stays in registers: eight
// elements (16 bytes) per lane and access, lanes side by side, so that a block of 16, 32 or 128 is 2, 4 or 16 neighbouring lanes and its largest
// magnitude a few shuffles.
#pragma once
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "f32x2.cuh"
#include "host_util.h"
#include "lowbit.cuh"

namespace omni {

// Where a launch's rows go.  ROWS: row r of x to row r, scales by groups of `group` rows (the experts of a weight), each from a new tile of 128 on.
// GATHER: item t is a token, its row goes to the rows row_of_pair[t * per ..] of its choices (< 0: nowhere), their scales to place_of_pair[t * per ..], which
// place_of_row keeps.  PLACED: row r to row r, scales to place_of_row[r]; rows from *n_rows on are left out.
enum RowMode : int { ROWS = 0, GATHER = 1, PLACED = 2 };
struct RowPlace {
  long group;
  const int *row_of_pair, *place_of_pair, *n_rows;
  int* place_of_row;
  int per;
};

struct RowsArgs {
  const bf16 *x, *residual, *gain;
  bf16 *total, *normed;
  long ldx, ldr, ldt, ldn, rows;
  uint8_t* codes;
  void* scales;
  float* row_scale;
  int K;
  float eps, inv_k;              // 1 / K
  RowPlace place;
};

// larger ones of two pairs of bf16 that are not negative, NaN above all
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// of eight bf16, two magnitudes side by side that hold the largest
__device__ __forceinline__ uint32_t max_pair(const uint4& u) {
  constexpr uint32_t M = 0x7fff7fffu;
  return max2(max2(u.x & M, u.y & M), max2(u.z & M, u.w & M));
}
// Largest magnitude of LANES neighbouring lanes as a 15-bit pattern: ordered like the magnitudes, infinity and NaN from 0x7f80 on.
template <int LANES>
__device__ __forceinline__ uint32_t group_top(uint32_t pair) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) pair = max2(pair, __shfl_xor_sync(0xffffffffu, pair, o));
  return max2(pair, pair >> 16) & 0xffffu;
}

// eight values to e2m1, the first in the lowest half byte (the converted bytes merge into one register)
__device__ __forceinline__ uint32_t e2m1x8(const float (&q)[8]) {
  uint32_t out;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(out) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return out;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes of a chunk (4-bit: x; fp8: x and y) and the scale of its block: a byte (4-bit), an fp32 (fp8).
struct Chunk {
  uint2 code;
  uint32_t scale;
};
// Eight elements per lane; `row_inv` (nvfp4) the reciprocal of the row's factor.  The integer pipe bounds this (8191 x 12288 to mxfp4: 78 % busy at 61 us with
// integer maxima, shifts that assemble scale words and bytes), so maxima are taken on packed pairs, products and roundings on the floating-point pipe.
template <int FMT>
__device__ __forceinline__ Chunk quantize_chunk(const uint4& u, float row_inv) {
  Chunk out;
  float v[8];
  unpack8(u, v);
  if (FMT == FMT_FP8) {
    // s = max / 448 and code = e4m3(x / s), both quotients rounded to fp32 as a division rounds them.  s: a product with 1 / 448 in two terms, good to 2^-46,
    // while 8 bits over 7 are either exact in fp32 or (binary digits of period three) 2^-28 of themselves away from halfway between two fp32 values.  x / s:
    // one step of Newton's on a product with a reciprocal, q + (x - q s) / s, whose residual is exact.  (With s by one rounded term it was a step off in
    // half of the blocks, which moved one in 190 of the values rounded to bf16; with codes from 448 x / max one in 27000 ties fell the other way.)
    const uint32_t top = group_top<16>(max_pair(u));
    constexpr float INV448 = 1.0f / 448.0f, INV448_REST = (float)(1.0 / 448.0 - (double)INV448);
    const float amax = fmaxf(__uint_as_float(top << 16), 1e-8f), scale = fmaf(amax, INV448, amax * INV448_REST), inv = rcp_fast(scale);
    const uint64_t inv2 = pack2(inv, inv), minus = pack2(-scale, -scale);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t x = pack2(v[2 * i], v[2 * i + 1]), q = mul2(x, inv2), r = fma2(fma2(q, minus, x), inv2, q);
      float lo, hi;
      unpack2(r, lo, hi);
      w[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
    }
    out.code = make_uint2(w[0], w[1]);
    out.scale = top >= 0x7f80u ? 0x7fc00000u : __float_as_uint(scale);
    return out;
  }
  const uint32_t top = group_top<FMT == FMT_MXFP4 ? 4 : 2>(max_pair(u));
  float q[8];
  if (FMT == FMT_MXFP4) {
    // the power of two two below the largest magnitude's (6 = 1.5 * 2^2 is the largest code): dividing by it is exact
    const uint32_t e = top >> 7;
    out.scale = e == 255 ? 255 : e > 2 ? e - 2 : 0;
    const float inv = __uint_as_float((254u - out.scale) << 23);     // 2^-(byte - 127); no finite block's byte is above 252
    const uint64_t inv2 = pack2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2(mul2(pack2(v[2 * i], v[2 * i + 1]), inv2), q[2 * i], q[2 * i + 1]);
  } else {
    // s = e4m3(max / 6), code = e2m1(x / s).  Both quotients are products with a reciprocal, off by a few steps of fp32, rounded to fp16 before they are
    // rounded to the format: max / 6 (8-bit mantissas) is either exactly halfway between two e4m3 values or 2^-9 of itself away, and so is x / s (8 by
    // 4 bits) for e2m1, so that the 11 bits of fp16 keep what is no tie from becoming one and restore what is.
    const __half want = __float2half_rn(__uint_as_float(top << 16) * row_inv * (1.0f / 6.0f));
    const uint32_t byte = __nv_cvt_halfraw_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
    const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
    const float inv = s > 0.f ? rcp_fast(s) : 0.f;
    const uint64_t row2 = pack2(row_inv, row_inv), inv2 = pack2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      unpack2(mul2(mul2(pack2(v[2 * i], v[2 * i + 1]), row2), inv2), lo, hi);
      const float2 f = __half22float2(__floats2half2_rn(lo, hi));
      q[2 * i] = f.x;
      q[2 * i + 1] = f.y;
    }
    out.scale = top >= 0x7f80u ? 0x7f : byte;
  }
  out.code = make_uint2(e2m1x8(q), 0u);
  return out;
}

// Where a thread's chunks go: chunk tid + i * tpr.  tpr is a multiple of 32, so that a block's first lane and its byte of the word are the same for all i.
template <int FMT> struct ChunkPlace {
  uint8_t *code, *scale;
  int code_step, scale_step, left, scales_left;                 // chunks (and of them ones with a place for a scale) from this thread's first on
  bool first;                                                   // of its block
  __device__ __forceinline__ ChunkPlace(const RowsArgs& a, long code_row, long scale_row, int tid, int tpr) {
    constexpr int PER = FMT == FMT_FP8 ? 16 : FMT == FMT_MXFP4 ? 4 : 2;
    first = tid % PER == 0;
    left = a.K / 8 - tid;
    if (FMT == FMT_FP8) {
      code = a.codes + code_row * a.K + tid * 8;
      scale = static_cast<uint8_t*>(a.scales) + (scale_row * (a.K / 128) + tid / 16) * 4;
      code_step = tpr * 8; scale_step = tpr / 16 * 4; scales_left = left;
    } else {
      const int words = scale_words(FMT, a.K);
      code = a.codes + code_row * (a.K / 2) + tid * 4;
      scale = static_cast<uint8_t*>(a.scales) + scale_word_at(scale_row, tid / (4 * PER), words) + tid / PER % 4;
      code_step = tpr * 4; scale_step = tpr / (4 * PER) * 512; scales_left = words * 4 * PER - tid;      // blocks past K in a row's last word: zeros
    }
  }
  __device__ __forceinline__ void store(const Chunk& c, int i, int tpr) const {
    if (i * tpr < left) {
      if (FMT == FMT_FP8) *reinterpret_cast<uint2*>(code + (long)i * code_step) = c.code;
      else *reinterpret_cast<uint32_t*>(code + (long)i * code_step) = c.code.x;
    }
    if (first && i * tpr < scales_left) {
      if (FMT == FMT_FP8) *reinterpret_cast<uint32_t*>(scale + (long)i * scale_step) = c.scale;
      else scale[(long)i * scale_step] = (uint8_t)c.scale;
    }
  }
};

// NV chunks per thread, blockDim.x threads (a multiple of 32) per row, blockDim.y rows per block.  One pass over a row, which stays in registers.  8191 x 12288 to
// mxfp4: 44 us (254 MB, 5.8 TB/s), integer pipe 71 % busy; to nvfp4 61 (4.2 TB/s): a row's warps meet between its loads and its codes, for the row's factor.
// With a residual, the norm, its sum and fp8, 12289 x 4096: 66 us (352 MB, 5.4 TB/s), mxfp4 61, nvfp4 68.  Without a residual 8192 x 4096 34.8, 31.5, 36.4.
template <int FMT, bool NORM, int MODE, int NV, int MOST>
__global__ void __launch_bounds__(MOST)
lowbit_rows_kernel(const RowsArgs a) {
  __shared__ uint32_t red[32];
  const int tid = threadIdx.x, sub = threadIdx.y, tpr = blockDim.x, lane = tid & 31;
  const int warps = tpr >> 5, warp0 = sub * warps, warp = warp0 + (tid >> 5);
  const long item = (long)blockIdx.x * blockDim.y + sub;
  const RowPlace& pl = a.place;
  bool live = item < a.rows;
  pdl_begin();
  uint4 u[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = tid + i * tpr;
    u[i] = live && c * 8 < a.K ? *reinterpret_cast<const uint4*>(a.x + item * a.ldx + c * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
  long scale_row = item;
  if (MODE == PLACED) {
    live = live && item < *pl.n_rows;
    scale_row = live ? pl.place_of_row[item] : 0;
  } else if (MODE == ROWS && pl.group != a.rows) {
    const long g = item / pl.group;
    scale_row = g * ((pl.group + 127) / 128 * 128) + (item - g * pl.group);
  }
  if (NORM) {
    float ss = 0.f;
    if (a.residual) {
      uint4 r[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = tid + i * tpr;
        r[i] = live && c * 8 < a.K ? *reinterpret_cast<const uint4*>(a.residual + item * a.ldr + c * 8) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float v[8], w[8];
        unpack8(u[i], v);
        unpack8(r[i], w);
        u[i] = make_uint4(pack_bf16(v[0] + w[0], v[1] + w[1]), pack_bf16(v[2] + w[2], v[3] + w[3]), pack_bf16(v[4] + w[4], v[5] + w[5]),
                          pack_bf16(v[6] + w[6], v[7] + w[7]));
      }
    }
    uint4 gain[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = tid + i * tpr;
      const bool in = live && c * 8 < a.K;
      gain[i] = in ? *reinterpret_cast<const uint4*>(a.gain + c * 8) : make_uint4(0u, 0u, 0u, 0u);
      if (a.total && in) *reinterpret_cast<uint4*>(a.total + item * a.ldt + c * 8) = u[i];
      float v[8];
      unpack8(u[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (warps > 1) {
      if (lane == 0) red[warp] = __float_as_uint(ss);
      __syncthreads();
      ss = 0.f;
      for (int w = 0; w < warps; ++w) ss += __uint_as_float(red[warp0 + w]);
      if (FMT == FMT_NVFP4) __syncthreads();
    }
    const float r = rsqrtf(ss * a.inv_k + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = tid + i * tpr;
      float v[8], g[8];
      unpack8(u[i], v);
      unpack8(gain[i], g);
      // rounded to bf16 before the blocks' scales are taken: the values a norm of its own would have stored
      u[i] = make_uint4(pack_bf16(v[0] * r * g[0], v[1] * r * g[1]), pack_bf16(v[2] * r * g[2], v[3] * r * g[3]),
                        pack_bf16(v[4] * r * g[4], v[5] * r * g[5]), pack_bf16(v[6] * r * g[6], v[7] * r * g[7]));
      if (a.normed && live && c * 8 < a.K) *reinterpret_cast<uint4*>(a.normed + item * a.ldn + c * 8) = u[i];
    }
  }
  float row_inv = 1.f, factor = 1.f;
  if (FMT == FMT_NVFP4) {
    // the row's factor: the power of two that puts the row's largest magnitude into [2^10, 2^11), its block's scale into [170, 342)
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max2(top, max_pair(u[i]));
    top = __reduce_max_sync(0xffffffffu, max2(top, top >> 16) & 0xffffu);
    if (warps > 1) {
      if (lane == 0) red[warp] = top;
      __syncthreads();
      for (int w = 0; w < warps; ++w) top = max(top, red[warp0 + w]);
    }
    const int e = (int)(top >> 7), field = top == 0 ? 127 : e > 11 ? e - 10 : 1;
    row_inv = __uint_as_float((uint32_t)(254 - field) << 23);
    factor = e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)field << 23);
  }
  Chunk c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) c[i] = quantize_chunk<FMT>(u[i], row_inv);
  if (MODE != GATHER) {
    if (!live) return;
    if (FMT == FMT_NVFP4 && tid == 0) a.row_scale[item] = factor;
    const ChunkPlace<FMT> to(a, item, scale_row, tid, tpr);
#pragma unroll
    for (int i = 0; i < NV; ++i) to.store(c[i], i, tpr);
  } else {
    // quantised once, written once per choice
    if (!live) return;
#pragma unroll 1
    for (int j0 = 0; j0 < pl.per; j0 += 4) {
      int row[4], place[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = j0 + j < pl.per;
        row[j] = in ? pl.row_of_pair[item * pl.per + j0 + j] : -1;
        place[j] = in ? pl.place_of_pair[item * pl.per + j0 + j] : 0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (row[j] < 0) continue;
        if (tid == 0) {
          pl.place_of_row[row[j]] = place[j];
          if (FMT == FMT_NVFP4) a.row_scale[row[j]] = factor;
        }
        const ChunkPlace<FMT> to(a, row[j], place[j], tid, tpr);
#pragma unroll
        for (int i = 0; i < NV; ++i) to.store(c[i], i, tpr);
      }
    }
  }
}

struct DequantArgs {
  const uint8_t* codes;
  const void* scales;
  const float* row_scale;
  void* out;
  long rows, group;
  int K, f32;
};

// Eight elements per thread, four rows on their way at a time; blockDim.x chunks by blockDim.y rows per block.  8191 x 12288 mxfp4 to bf16
// 65 to 67 us, to fp32 104: 201 and 402 MB written at 3.0 and 3.9 TB/s, codes read beside them.  A fill of the 201 MB takes 52, a copy of them 63, so that stores
// alone do not bound the bf16 form; its 16 bytes a thread are half of what the fp32 form stores.
template <int FMT>
__global__ void __launch_bounds__(256)
dequantize_kernel(const DequantArgs a) {
  pdl_begin();
  constexpr int PER = FMT == FMT_MXFP4 ? 4 : 2, DEPTH = 4;
  const int chunks = a.K / 8, words = scale_words(FMT, a.K);
  const long step = (long)gridDim.y * blockDim.y;
  for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < chunks; c += gridDim.x * blockDim.x) {
    const int block = c / PER;
    for (long row0 = (long)blockIdx.y * blockDim.y + threadIdx.y; row0 < a.rows; row0 += DEPTH * step) {
      uint2 code[DEPTH];
      float s[DEPTH];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const long row = row0 + d * step;
        code[d] = make_uint2(0u, 0u);
        s[d] = 0.f;
        if (row < a.rows) {
          if (FMT == FMT_FP8) {
            code[d] = *reinterpret_cast<const uint2*>(a.codes + row * a.K + c * 8);
            s[d] = static_cast<const float*>(a.scales)[row * (a.K / 128) + c / 16];
          } else {
            code[d].x = *reinterpret_cast<const uint32_t*>(a.codes + row * (a.K / 2) + c * 4);
            long scale_row = row;
            if (a.group != a.rows) {
              const long g = row / a.group;
              scale_row = g * ((a.group + 127) / 128 * 128) + (row - g * a.group);
            }
            const uint32_t byte = static_cast<const uint8_t*>(a.scales)[scale_word_at(scale_row, block >> 2, words) + (block & 3)];
            if (FMT == FMT_MXFP4) s[d] = __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 1u << 22 : byte << 23);
            else s[d] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3))) * a.row_scale[row];
          }
        }
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const long row = row0 + d * step;
        if (row >= a.rows) break;
        float v[8];
        if (FMT == FMT_FP8) {
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((p < 2 ? code[d].x : code[d].y) >> (16 * (p & 1))), __NV_E4M3));
            const float2 f = __half22float2(h);
            v[2 * p] = f.x * s[d];
            v[2 * p + 1] = f.y * s[d];
          }
        } else {
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const float2 f = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(code[d].x >> (8 * p)), __NV_E2M1)));
            v[2 * p] = f.x * s[d];
            v[2 * p + 1] = f.y * s[d];
          }
        }
        if (a.f32) {
          float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out) + row * a.K + c * 8);
          o[0] = make_float4(v[0], v[1], v[2], v[3]);
          o[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          *reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) + row * a.K + c * 8) =
              make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
      }
    }
  }
}

// Threads per row and chunks per thread.  Up to 512 chunks per SM, none of a row longer than that: a lane per chunk (nvfp4, us with one and with up to four
// chunks: 8 x 4096 1.75, 2.06, with the norm 2.41, 2.91; 148 x 4096 1.89, 2.23; 296 x 2048 1.88, 2.06).  Beyond: up to four, which share what a thread does
// once per row, with fewer warps to wait for (1 x 8192 2.57, 2.23, with the norm 3.94, 3.08; 296 x 4096 with the norm 3.59, 3.10; 8192 x 4096 35.0, 20.3), and no more of them than
// the row's threads need: 19704 x 768 in three 9.2 us, in four 11.1, 8192 x 1536 8.4, 9.9.
template <int FMT, bool NORM, int MODE>
static int launch_rows(RowsArgs& a, cudaStream_t s) {
  const int chunks = a.K / 8;
  int nv = chunks <= 512 && a.rows * chunks <= 512L * sm_count() ? 1 : 4;
  const int tpr = (chunks + 32 * nv - 1) / (32 * nv) * 32;
  nv = (chunks + tpr - 1) / tpr;
  if (tpr > 1024) return RC_TOO_LARGE;
  const dim3 block(tpr, tpr >= 256 ? 1 : 256 / tpr);
  const unsigned grid = (unsigned)((a.rows + block.y - 1) / block.y);
  a.inv_k = 1.0f / (float)a.K;
  if (nv == 4 && tpr > 512) return launch_overlapped(lowbit_rows_kernel<FMT, NORM, MODE, 4, 1024>, grid, block, 0, s, a);
  switch (nv) {
    case 1: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, MODE, 1, 512>, grid, block, 0, s, a);
    case 2: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, MODE, 2, 512>, grid, block, 0, s, a);
    case 3: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, MODE, 3, 512>, grid, block, 0, s, a);
    default: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, MODE, 4, 512>, grid, block, 0, s, a);
  }
}

static int rows_any(RowsArgs& a, int fmt, cudaStream_t s) {
  if (a.rows <= 0 || a.K <= 0) return RC_OK;
  if (a.rows > 0x7fffffffL || a.K % (fmt == FMT_FP8 ? 128 : 32) || ((a.ldx | a.ldr | a.ldt | a.ldn) & 7)) return RC_BAD_ARG;
  if (!on16(a.x) || !on16(a.residual) || !on16(a.gain) || !on16(a.total) || !on16(a.normed) || !on16(a.codes) ||
      !on16(a.scales))
    return RC_BAD_ARG;
  if (fmt == FMT_NVFP4 && !a.row_scale) return RC_BAD_ARG;
  if (a.gain) {
    switch (fmt) {
      case FMT_MXFP4: return launch_rows<FMT_MXFP4, true, ROWS>(a, s);
      case FMT_NVFP4: return launch_rows<FMT_NVFP4, true, ROWS>(a, s);
      case FMT_FP8: return launch_rows<FMT_FP8, true, ROWS>(a, s);
      default: return RC_BAD_ARG;
    }
  }
  const int mode = a.place.row_of_pair ? GATHER : a.place.place_of_row ? PLACED : ROWS;
  switch (fmt * 3 + mode) {
    case FMT_MXFP4 * 3 + ROWS: return launch_rows<FMT_MXFP4, false, ROWS>(a, s);
    case FMT_MXFP4 * 3 + GATHER: return launch_rows<FMT_MXFP4, false, GATHER>(a, s);
    case FMT_MXFP4 * 3 + PLACED: return launch_rows<FMT_MXFP4, false, PLACED>(a, s);
    case FMT_NVFP4 * 3 + ROWS: return launch_rows<FMT_NVFP4, false, ROWS>(a, s);
    case FMT_NVFP4 * 3 + GATHER: return launch_rows<FMT_NVFP4, false, GATHER>(a, s);
    case FMT_NVFP4 * 3 + PLACED: return launch_rows<FMT_NVFP4, false, PLACED>(a, s);
    default: return RC_BAD_ARG;
  }
}

static int dequantize_any(const DequantArgs& a, int fmt, cudaStream_t s) {
  if (a.rows <= 0 || a.K <= 0) return RC_OK;
  if (a.K % (fmt == FMT_FP8 ? 128 : 32) || !on16(a.codes) || !on16(a.out) || (fmt == FMT_NVFP4 && !a.row_scale)) return RC_BAD_ARG;
  int x = 32;
  while (x < 256 && x < a.K / 8) x *= 2;
  const int y = 256 / x;
  const long gx = (a.K / 8 + x - 1) / x, want = (a.rows + 4 * y - 1) / (4 * y), most = (16L * sm_count() + gx - 1) / gx;
  const long gy = want < most ? want : most;
  const dim3 grid((unsigned)gx, (unsigned)(gy > 65535 ? 65535 : gy)), block(x, y);
  switch (fmt) {
    case FMT_MXFP4: return launch_overlapped(dequantize_kernel<FMT_MXFP4>, grid, block, 0, s, a);
    case FMT_NVFP4: return launch_overlapped(dequantize_kernel<FMT_NVFP4>, grid, block, 0, s, a);
    case FMT_FP8: return launch_overlapped(dequantize_kernel<FMT_FP8>, grid, block, 0, s, a);
    default: return RC_BAD_ARG;
  }
}

}  // namespace omni
