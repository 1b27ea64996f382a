// 4-bit operands of the block-scaled tensor instructions: where codes and scales lie, and the instructions.
//
// Rows [R, K] (K a multiple of 32): codes [R, K / 2], element 2 i in the low half of byte i, e2m1 (sign, 2 bits of exponent, 1 of
// mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6).  One scale byte per block of a row, in words of four neighbouring blocks:
//   mxfp4   blocks of 32, byte = exponent + 127 (e8m0); a word covers 128 elements, two steps of an MMA
//   nvfp4   blocks of 16, e4m3, and one fp32 factor per row;  a word covers 64 elements, one step
// Words stand in tiles of 128 rows x 4 bytes, [R / 128][words of a row][32][4] with row r at [r / 128][.][r % 32][r / 32 % 4]: a tile is
// the 32 lanes x 16 bytes that one tcgen05.cp brings into tensor memory for all four quadrants.  Bytes of blocks past K are zero
// (finite: codes past K arrive as zeros), those of rows past R are anything.
#pragma once
#include "ptx_sm100.cuh"

namespace omni {

typedef __nv_bfloat16 bf16;

inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

enum LowFmt : int { FMT_MXFP4 = 0, FMT_NVFP4 = 1, FMT_FP8 = 2 };

template <int FMT> struct LowCfg {
  static constexpr int BLOCK = FMT == FMT_MXFP4 ? 32 : FMT == FMT_NVFP4 ? 16 : 128;
  static constexpr int WORD = 4 * BLOCK;                      // elements of a word of scales (4-bit formats)
};
__host__ __device__ inline int scale_words(int fmt, int K) { return fmt == FMT_MXFP4 ? (K + 127) / 128 : (K + 63) / 64; }
// byte offset of the word of (row, word) where a row has `words` of them
__host__ __device__ inline long scale_word_at(long row, int word, int words) {
  return ((row >> 7) * words + word) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Instruction descriptor of the block-scaled kinds on e2m1 operands (both K-major), fp32 accumulation.
//   bits [4,6) which byte of B's scale words comes first    [7,10) A type (1 = e2m1)   [10,12) B type (1 = e2m1)
//   bits [17,23) N / 8    [23] scales: 0 = e4m3, 1 = e8m0    [27,29) M / 128    [29,31) which byte of A's scale words comes first
template <int FMT>
__host__ __device__ constexpr uint32_t fp4_idesc(uint32_t M, uint32_t N, uint32_t scale_id) {
  return (scale_id << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((FMT == FMT_MXFP4 ? 1u : 0u) << 23) | ((M >> 7) << 27) | (scale_id << 29);
}

// D[tmem] (+)= (A * scales) (B * scales)^T, K = 64 per instruction.  Scales in tensor memory: mxfp4 two bytes per row and step (of a word
// that serves two steps, ids 0 and 2), nvfp4 four.
template <int FMT, bool PAIR>
__device__ __forceinline__ void mma_fp4_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                           uint32_t b_scales, uint32_t accumulate) {
#define OMNI_FP4_MMA(GROUP, KIND)                                                                      \
  asm volatile(                                                                                        \
      "{\n\t.reg .pred p;\n\t"                                                                         \
      "setp.ne.b32 p, %4, 0;\n\t"                                                                      \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n"       \
      :                                                                                                \
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scales), "r"(b_scales) \
      : "memory")
  if (FMT == FMT_MXFP4) {
    if (PAIR) OMNI_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
    else OMNI_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
  } else {
    if (PAIR) OMNI_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else OMNI_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  }
#undef OMNI_FP4_MMA
}

// Descriptor of a tile of scale words in shared memory (512 bytes, 16-byte aligned): 32 rows of 16 bytes without swizzle, groups of 8 rows
// 128 bytes apart.
__device__ __forceinline__ uint64_t scale_tile_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}
// That tile into four columns of tensor memory, every quadrant of 32 lanes the same.  On pairs each CTA copies from its own shared memory.
// Issued by the thread that issues the MMAs, which run after it.
template <bool PAIR>
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint64_t desc) {
  if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

}  // namespace omni
