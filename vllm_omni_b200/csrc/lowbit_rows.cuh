// Rows to 4 and 8 bits and back (layouts: lowbit.cuh): kernels and their launchers.
//
// All are bound by memory traffic for many rows and by one round trip for few, so a row is read once and stays in registers: eight
// elements (16 bytes) per lane and access, lanes side by side, so that a block of 16, 32 or 128 is 2, 4 or 16 neighbouring lanes and its largest
// magnitude a few shuffles.
#pragma once
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "host_util.h"
#include "lowbit.cuh"

namespace omni {

// Where a launch's rows come from and go to.  `tiles` null: row r of x to row r, scales by groups of `group` rows (the experts of a weight), each from
// a new tile of 128 on.  Else expert rows: with `row_of_pair`, item p is pair p, whose source is row p / per; without, source and
// place are the item's own index.  Scales of row i of tile t stand at t * pitch + i; rows of no tile are left out.
struct RowPlace {
  long group;
  const int *row_of_pair, *tile_expert, *tile_row0, *tile_rows;
  int per, max_tiles, pitch;
};

struct RowsArgs {
  const bf16 *x, *residual, *gain;
  bf16 *total, *normed;
  long ldx, ldr, ldt, ldn, rows;
  uint8_t* codes;
  void* scales;
  float* row_scale;
  int K, tpr;                    // threads per row, a multiple of 32
  float eps;
  RowPlace place;
};

// largest magnitude of eight bf16, as a 15-bit pattern: ordered like the magnitudes, with infinity and NaN above all numbers
__device__ __forceinline__ uint32_t max_pattern(const uint4& u) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t a = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
  return max(a & 0xffffu, a >> 16);
}

template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ uint32_t e2m1x8(const float (&q)[8]) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(q[2 * i], q[2 * i + 1]), __NV_E2M1, cudaRoundNearest) << (8 * i);
  return out;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// One chunk of eight elements per lane; `row_inv` (nvfp4) the reciprocal of the row's factor.  Writes the codes and, from the first lane of a
// word, the scales.
template <int FMT>
__device__ __forceinline__ void quantize_chunk(const RowsArgs& a, const uint4& u, int chunk, long code_row, long scale_row, float row_inv, bool live) {
  const int lane = threadIdx.x & 31;
  const bool in = live && chunk * 8 < a.K;
  float v[8];
  unpack8(u, v);
  if (FMT == FMT_FP8) {
    // the arithmetic of the fp8 layers' own quantiser (gemm_fp8_sm100.cu)
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = fmaxf(amax, 1e-8f) * (1.0f / 448.0f), inv = 1.0f / scale;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
    if (in) {
      *reinterpret_cast<uint2*>(a.codes + code_row * a.K + chunk * 8) = make_uint2(w[0], w[1]);
      if ((lane & 15) == 0) reinterpret_cast<float*>(a.scales)[scale_row * (a.K / 128) + chunk / 16] = scale;
    }
    return;
  }
  const uint32_t top = group_max<FMT == FMT_MXFP4 ? 4 : 2>(max_pattern(u));
  uint32_t byte;
  float q[8];
  if (FMT == FMT_MXFP4) {
    // the power of two two below the largest magnitude's (6 = 1.5 * 2^2 is the largest code): dividing by it is exact
    const uint32_t e = top >> 7;
    byte = e == 255 ? 255 : e > 2 ? e - 2 : 0;
    const float inv = __uint_as_float(byte == 254 ? 1u << 22 : (254u - byte) << 23);       // 2^-(byte - 127); no scale is above 253
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] * inv;
  } else {
    // s = e4m3(max / 6).  The quotient is formed by one rounded reciprocal, then rounded to fp16: x / s of an 8-bit by a 4-bit mantissa is
    // either exactly halfway between two codes or off by 2^-9 of itself, so that the 11 bits of fp16 restore what the reciprocal's last
    // bit would make of a tie.
    const float s_want = __fdiv_rn(__uint_as_float(top << 16) * row_inv, 6.0f);
    byte = __nv_cvt_float_to_fp8(s_want, __NV_SATFINITE, __NV_E4M3);
    const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(__floats2half2_rn(v[2 * i] * row_inv * inv, v[2 * i + 1] * row_inv * inv));
      q[2 * i] = f.x;
      q[2 * i + 1] = f.y;
    }
    if (top >= 0x7f80u) byte = 0x7f;
  }
  if (in) *reinterpret_cast<uint32_t*>(a.codes + code_row * (a.K / 2) + chunk * 4) = e2m1x8(q);
  constexpr int PER = FMT == FMT_MXFP4 ? 4 : 2;                 // lanes of a block; a word is four blocks
  uint32_t word = (lane % PER) == 0 && chunk * 8 < a.K ? byte << (8 * ((lane / PER) & 3)) : 0u;
  word |= __shfl_xor_sync(0xffffffffu, word, PER);
  word |= __shfl_xor_sync(0xffffffffu, word, 2 * PER);
  const int words = scale_words(FMT, a.K), at = chunk / (4 * PER);
  if (live && lane % (4 * PER) == 0 && at < words)
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.scales) + scale_word_at(scale_row, at, words)) = word;
}

// NV chunks per thread, a.tpr threads per row, blockDim / tpr rows per block.
template <int FMT, bool NORM, int NV>
__global__ void __launch_bounds__(1024)
lowbit_rows_kernel(const RowsArgs a) {
  __shared__ uint32_t red[32];
  __shared__ int found[32];
  const int sub = threadIdx.x / a.tpr, tid = threadIdx.x - sub * a.tpr, lane = threadIdx.x & 31;
  const int warps = a.tpr >> 5, warp0 = sub * warps;
  const long item = (long)blockIdx.x * (blockDim.x / a.tpr) + sub;
  bool live = item < a.rows;
  pdl_begin();
  const RowPlace& pl = a.place;
  const bool tiled = pl.tile_expert != nullptr;
  long src = item, code_row = item, scale_row = 0;
  if (tiled) {
    if (pl.row_of_pair) {
      code_row = live ? pl.row_of_pair[item] : -1;
      src = item / pl.per;
    }
    live = live && code_row >= 0;
  } else {
    const long g = item / pl.group;
    scale_row = g * ((pl.group + 127) / 128 * 128) + (item - g * pl.group);
  }
  uint4 u[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = tid + i * a.tpr;
    u[i] = live && c * 8 < a.K ? *reinterpret_cast<const uint4*>(a.x + src * a.ldx + c * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
  if (tiled) {
    if (tid == 0) found[sub] = -1;
    __syncthreads();
    for (int t = tid; t < pl.max_tiles; t += a.tpr) {
      const int i = (int)code_row - pl.tile_row0[t];
      if (live && pl.tile_expert[t] >= 0 && i >= 0 && i < pl.tile_rows[t]) found[sub] = t * pl.pitch + i;
    }
    __syncthreads();
    scale_row = found[sub];
    live = live && scale_row >= 0;
  }
  if (NORM) {
    float ss = 0.f;
    if (a.residual) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = tid + i * a.tpr;
        if (live && c * 8 < a.K) {
          const uint4 r = *reinterpret_cast<const uint4*>(a.residual + src * a.ldr + c * 8);
          float v[8], w[8];
          unpack8(u[i], v);
          unpack8(r, w);
          u[i] = make_uint4(pack_bf16(v[0] + w[0], v[1] + w[1]), pack_bf16(v[2] + w[2], v[3] + w[3]), pack_bf16(v[4] + w[4], v[5] + w[5]),
                            pack_bf16(v[6] + w[6], v[7] + w[7]));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = tid + i * a.tpr;
      if (a.total && live && c * 8 < a.K) *reinterpret_cast<uint4*>(a.total + src * a.ldt + c * 8) = u[i];
      float v[8];
      unpack8(u[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (warps > 1) {
      if (lane == 0) red[threadIdx.x >> 5] = __float_as_uint(ss);
      __syncthreads();
      ss = 0.f;
      for (int w = 0; w < warps; ++w) ss += __uint_as_float(red[warp0 + w]);
      __syncthreads();
    }
    const float r = 1.0f / sqrtf(ss / (float)a.K + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = tid + i * a.tpr;
      if (live && c * 8 < a.K) {
        float v[8], g[8];
        unpack8(u[i], v);
        unpack8(*reinterpret_cast<const uint4*>(a.gain + c * 8), g);
        // rounded to bf16 before the blocks' scales are taken: the values a norm of its own would have stored
        u[i] = make_uint4(pack_bf16(v[0] * r * g[0], v[1] * r * g[1]), pack_bf16(v[2] * r * g[2], v[3] * r * g[3]),
                          pack_bf16(v[4] * r * g[4], v[5] * r * g[5]), pack_bf16(v[6] * r * g[6], v[7] * r * g[7]));
        if (a.normed) *reinterpret_cast<uint4*>(a.normed + src * a.ldn + c * 8) = u[i];
      }
    }
  }
  float row_inv = 1.f;
  if (FMT == FMT_NVFP4) {
    // the row's factor: the power of two that puts the row's largest magnitude into [2^10, 2^11), its block's scale into [170, 342)
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max(top, max_pattern(u[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (warps > 1) {
      if (lane == 0) red[threadIdx.x >> 5] = top;
      __syncthreads();
      for (int w = 0; w < warps; ++w) top = max(top, red[warp0 + w]);
    }
    const int e = (int)(top >> 7), field = top == 0 ? 127 : e > 11 ? e - 10 : 1;
    row_inv = __uint_as_float((uint32_t)(254 - field) << 23);
    if (live && tid == 0) a.row_scale[code_row] = e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)field << 23);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) quantize_chunk<FMT>(a, u[i], tid + i * a.tpr, code_row, scale_row, row_inv, live);
}

struct DequantArgs {
  const uint8_t* codes;
  const void* scales;
  const float* row_scale;
  void* out;
  long rows, group;
  int K, f32;
};

// Eight elements per thread.
template <int FMT>
__global__ void __launch_bounds__(256)
dequantize_kernel(const DequantArgs a) {
  pdl_begin();
  const int chunks = a.K / 8;
  const long total = a.rows * chunks;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long)gridDim.x * blockDim.x) {
    const long row = i / chunks;
    const int c = (int)(i - row * chunks);
    float v[8];
    if (FMT == FMT_FP8) {
      const uint2 u = *reinterpret_cast<const uint2*>(a.codes + row * a.K + c * 8);
      const float s = reinterpret_cast<const float*>(a.scales)[row * (a.K / 128) + c / 16];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)((e < 4 ? u.x : u.y) >> (8 * (e & 3))), __NV_E4M3))) * s;
    } else {
      constexpr int PER = FMT == FMT_MXFP4 ? 4 : 2;
      const uint32_t u = *reinterpret_cast<const uint32_t*>(a.codes + row * (a.K / 2) + c * 4);
      const long g = row / a.group, scale_row = g * ((a.group + 127) / 128 * 128) + (row - g * a.group);
      const int block = c / PER;
      const uint32_t byte = static_cast<const uint8_t*>(a.scales)[scale_word_at(scale_row, block >> 2, scale_words(FMT, a.K)) + (block & 3)];
      float s;
      if (FMT == FMT_MXFP4) s = __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 1u << 22 : byte << 23);
      else s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3))) * a.row_scale[row];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float2 f = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(u >> (8 * p)), __NV_E2M1)));
        v[2 * p] = f.x * s;
        v[2 * p + 1] = f.y * s;
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

// Threads per row and chunks per thread: up to two rows per SM a lane per chunk (one round trip); for more, four chunks per lane.
static void row_threads(int K, long rows, int& tpr, int& nv) {
  const int chunks = K / 8;
  nv = rows <= 2L * sm_count() ? 1 : 4;
  while (nv < 4 && chunks > 1024 * nv) nv *= 2;
  while (nv > 1 && chunks <= 32 * (nv / 2)) nv /= 2;
  tpr = (chunks + 32 * nv - 1) / (32 * nv) * 32;
}

template <int FMT, bool NORM>
static int launch_rows(RowsArgs& a, cudaStream_t s) {
  int nv;
  row_threads(a.K, a.rows, a.tpr, nv);
  if (a.tpr > 1024) return RC_TOO_LARGE;
  const int per = a.tpr >= 256 ? 1 : 256 / a.tpr, threads = per * a.tpr;
  const unsigned grid = (unsigned)((a.rows + per - 1) / per);
  switch (nv) {
    case 1: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, 1>, grid, threads, 0, s, a);
    case 2: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, 2>, grid, threads, 0, s, a);
    default: return launch_overlapped(lowbit_rows_kernel<FMT, NORM, 4>, grid, threads, 0, s, a);
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
      case FMT_MXFP4: return launch_rows<FMT_MXFP4, true>(a, s);
      case FMT_NVFP4: return launch_rows<FMT_NVFP4, true>(a, s);
      case FMT_FP8: return launch_rows<FMT_FP8, true>(a, s);
      default: return RC_BAD_ARG;
    }
  }
  switch (fmt) {
    case FMT_MXFP4: return launch_rows<FMT_MXFP4, false>(a, s);
    case FMT_NVFP4: return launch_rows<FMT_NVFP4, false>(a, s);
    default: return RC_BAD_ARG;
  }
}

static int dequantize_any(const DequantArgs& a, int fmt, cudaStream_t s) {
  if (a.rows <= 0 || a.K <= 0) return RC_OK;
  if (a.K % (fmt == FMT_FP8 ? 128 : 32) || !on16(a.codes) || !on16(a.out) || (fmt == FMT_NVFP4 && !a.row_scale)) return RC_BAD_ARG;
  const long blocks = (a.rows * (a.K / 8) + 255) / 256, most = (long)sm_count() * 16;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  switch (fmt) {
    case FMT_MXFP4: return launch_overlapped(dequantize_kernel<FMT_MXFP4>, grid, 256, 0, s, a);
    case FMT_NVFP4: return launch_overlapped(dequantize_kernel<FMT_NVFP4>, grid, 256, 0, s, a);
    case FMT_FP8: return launch_overlapped(dequantize_kernel<FMT_FP8>, grid, 256, 0, s, a);
    default: return RC_BAD_ARG;
  }
}

}  // namespace omni
