// A paged key/value cache of 8 bits and attention of single rows over it.
//
// Pages hold e4m3 codes [pages, page size, Hkv, D]; a value is its code times 2^e, e per (page, KV head), for keys and values apart.  Powers of two lose
// nothing next to other factors (a float's rounding is relative), make every value exact in bf16, and let a page be rounded again to a coarser scale at the
// cost of subnormal codes only.  Stored as fp32 [pages, Hkv].
//
//   omni_kv8_write      rows -> codes, scales of the pages they fall into
//   omni_kv8_read       rows of slots, or the rows of up to 16 block tables, -> bf16
//   omni_kv8_attn       rows of queries against the pages of their sequences
#include <cuda_fp16.h>

#include "host_util.h"
#include "ptx_sm100.cuh"

namespace omni {

constexpr int K8_GAP = 128;
constexpr int K8_LEAST = -120, K8_MOST = 120;      // exponents of scales: 448 * 2^120 is above every bf16, 2^-129 (the least code's value) still one

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }
// exponent of a stored scale; whatever else the word holds, one that scales can have
__device__ __forceinline__ int scale_exp(float s) { return min(max((int)((__float_as_uint(s) >> 23) & 0xff) - 127, K8_LEAST), K8_MOST); }
__device__ __forceinline__ uint32_t halves_of(uint32_t codes) {          // two e4m3 codes (low half) -> f16x2
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(codes));
  return h;
}
__device__ __forceinline__ uint32_t halves_of_hi(uint32_t codes) {       // the same of the high half
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(h) : "r"(codes));
  return h;
}
__device__ __forceinline__ float2 floats_of(uint32_t halves) { return __half22float2(*reinterpret_cast<__half2*>(&halves)); }
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {   // four codes, a in the lowest byte; beyond 448 saturates, NaN stays
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// ---------------------------------------------------------------------------------------------------------------------------------------- write
struct Kv8Write {
  const __nv_bfloat16 *k, *v;
  long k_rs, k_hs, v_rs, v_hs;           // pitches of rows and heads, in elements
  unsigned char *kc, *vc;
  float *ks, *vs;
  const int* slots;
  long n_slots;
  int T, Hkv, page, chunk;
  int* status;
};

// A run is the rows of one page, with fewer than 128 rows that are not written between two of them; the warp of its first row takes one head of it: largest magnitude, scale, rounding again of the rows before the
// first written one where the scale grows, codes.  A block looks for the runs that begin among `chunk` rows and deals out (run, keys or values).  Eight
// channels per lane: D / 8 lanes are a row, the warp takes 256 / D rows at a time.  The second pass over a run's rows finds them in L1.
template <int D>
__global__ void __launch_bounds__(256)
kv8_write_kernel(const __grid_constant__ Kv8Write p) {
  pdl_begin();
  constexpr int LANES = D / 8, ROWS = 32 / LANES;
  __shared__ int runs[64], n_runs;
  const int t0 = blockIdx.x * p.chunk, h = blockIdx.y;
  if (threadIdx.x < 32) {                // `chunk` is at most 64: two rows a lane
    int n = 0;
    for (int i0 = 0; i0 < p.chunk; i0 += 32) {
      const int t = t0 + i0 + threadIdx.x;
      bool first = false;
      if (i0 + threadIdx.x < p.chunk && t < p.T) {
        const int s = p.slots[t];
        if (s >= p.n_slots) atomicCAS(p.status, 0, ERR_BOUNDS);
        first = s >= 0 && s < p.n_slots;
        for (int b = t - 1; first && b >= 0 && b >= t - K8_GAP; --b) {
          const int before = p.slots[b];
          if (before < 0 || before >= p.n_slots) continue;
          first = before / p.page != s / p.page;
          break;
        }
      }
      const unsigned m = __ballot_sync(0xffffffffu, first);
      if (first) runs[n + __popc(m & ((1u << threadIdx.x) - 1))] = t;
      n += __popc(m);
    }
    if (threadIdx.x == 0) n_runs = n;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES, ch = lane % LANES * 8;
  for (int item = warp; item < 2 * n_runs; item += 8) {
    const int t1 = runs[item >> 1];
    const bool val = item & 1;
    const __nv_bfloat16* x = val ? p.v + h * p.v_hs : p.k + h * p.k_hs;
    const long rs = val ? p.v_rs : p.k_rs;
    unsigned char* cache = val ? p.vc : p.kc;
    float* scale = val ? p.vs : p.ks;
    const int at = p.slots[t1] / p.page;
    const long base = (long)at * p.page;
    // lowest row written, end of the run, largest magnitude (as bits: magnitudes of floats are ordered like integers)
    int low = p.page, t = t1;
    uint32_t most = 0;
    for (int skipped = 0, from = t1;;) {                                   // 32 rows from behind the last ones; t: behind the last one of the run
      const int s = from + lane < p.T ? p.slots[from + lane] : -1;
      const bool ok = s >= 0 && s < p.n_slots, mine = ok && s / p.page == at;
      const unsigned others = __ballot_sync(0xffffffffu, ok && !mine);
      const unsigned ours = __ballot_sync(0xffffffffu, mine) & (others ? (others & -others) - 1 : 0xffffffffu);
      if (!ours) {
        skipped += 32;
        from += 32;
        if (others || skipped >= K8_GAP || from >= p.T) break;
        continue;
      }
      const int rows = 32 - __clz(ours);
      low = min(low, (int)__reduce_min_sync(0xffffffffu, ours >> lane & 1 ? (unsigned)(s - base) : (unsigned)p.page));
#pragma unroll 4
      for (int r = sub; r < rows; r += ROWS) {
        if (!(ours >> r & 1)) continue;
        const uint4 u = *reinterpret_cast<const uint4*>(x + (from + r) * rs + ch);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a = (w[i] << 16) & 0x7fffffffu, b = w[i] & 0x7fff0000u;
          most = max(most, a < 0x7f800000u ? a : 0u);
          most = max(most, b < 0x7f800000u ? b : 0u);
        }
      }
      from += rows;
      t = from;
      skipped = 0;
      if (others) break;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    // least e with most <= 1.75 * 2^(8 + e)
    const int need = max((int)(most >> 23) - 127 - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0), K8_LEAST);
    float* my_scale = scale + (long)at * p.Hkv + h;
    int e = need;
    if (low > 0) {
      const int old = scale_exp(*my_scale);
      e = max(need, old);
      if (e > old) {
        const float f = pow2f(max(old - e, -126));                         // at 2^-126 every code becomes zero, as it would below
        for (int r = sub; r < low; r += ROWS) {
          unsigned char* c = cache + ((base + r) * p.Hkv + h) * D + ch;
          uint2 u = *reinterpret_cast<const uint2*>(c);
          uint32_t w[2] = {u.x, u.y};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 a = floats_of(halves_of(w[i])), b = floats_of(halves_of_hi(w[i]));
            w[i] = codes_of(a.x * f, a.y * f, b.x * f, b.y * f);
          }
          *reinterpret_cast<uint2*>(c) = make_uint2(w[0], w[1]);
        }
      }
    }
    __syncwarp();                                                          // the scale has been read
    if (lane == 0) *my_scale = pow2f(e);
    const float f = pow2f(-e);
    const int end = t;
    // the same slot twice in a run: later rows win, since a slot's writer is the lane group of its row and rows go in order within `r`
    for (t = t1; t < end; t += ROWS) {
      const int r = t + sub;
      const int s = r < end ? p.slots[r] : -1;
      if (s >= 0 && s < p.n_slots) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + r * rs + ch);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 a = unpack_bf16(w[2 * i]), b = unpack_bf16(w[2 * i + 1]);
          c[i] = codes_of(a.x * f, a.y * f, b.x * f, b.y * f);
        }
        bool last = true;                                                  // of the rows of this round with this slot
#pragma unroll
        for (int o = 1; o < ROWS; ++o) last &= !(sub + o < ROWS && r + o < end && p.slots[r + o] == s);
        if (last) *reinterpret_cast<uint2*>(cache + ((long)s * p.Hkv + h) * D + ch) = make_uint2(c[0], c[1]);
      }
      __syncwarp();
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------------------------------- read
constexpr int K8_TABLES = 16;
struct Kv8Read {
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int* index[K8_TABLES];           // slots of the rows, or block tables
  long row0[K8_TABLES], rows[K8_TABLES]; // first row written, rows
  __nv_bfloat16 *k, *v;                  // [.., Hkv, D]
  long n_slots;
  int Hkv, D, page, tables;              // tables: index is block tables
  int* status;
};

__global__ void __launch_bounds__(256)
kv8_read_kernel(const __grid_constant__ Kv8Read p) {
  pdl_begin();
  const int seg = blockIdx.y, vecs = p.Hkv * p.D / 16;
  const long n = p.rows[seg] * vecs;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long t = i / vecs;
    const int c = (int)(i - t * vecs) * 16;
    long slot;
    if (p.tables) {
      const long at = t / p.page;
      const long pg = p.index[seg][at];
      slot = pg < 0 ? p.n_slots : pg * p.page + (t - at * p.page);
    } else {
      slot = p.index[seg][t];
    }
    uint4 out[2][2] = {};
    if (slot >= 0 && slot < p.n_slots) {
      const long scale_at = slot / p.page * p.Hkv + c / p.D, from = slot * p.Hkv * p.D + c;
      const uint4 code[2] = {*reinterpret_cast<const uint4*>(p.kc + from), *reinterpret_cast<const uint4*>(p.vc + from)};
      const float f[2] = {pow2f(scale_exp(p.ks[scale_at])), pow2f(scale_exp(p.vs[scale_at]))};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t w[4] = {code[b].x, code[b].y, code[b].z, code[b].w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 lo = floats_of(halves_of(w[j])), hi = floats_of(halves_of_hi(w[j]));
          o[2 * j] = pack_bf16(lo.x * f[b], lo.y * f[b]);
          o[2 * j + 1] = pack_bf16(hi.x * f[b], hi.y * f[b]);
        }
        out[b][0] = make_uint4(o[0], o[1], o[2], o[3]);
        out[b][1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    } else if (slot >= p.n_slots) {
      atomicCAS(p.status, 0, ERR_BOUNDS);
    }
    const long to = (p.row0[seg] + t) * p.Hkv * p.D + c;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint4* dst = reinterpret_cast<uint4*>((b ? p.v : p.k) + to);
      dst[0] = out[b][0];
      dst[1] = out[b][1];
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------ attention
// One row of queries reads every key and value of its sequence once: a stream from HBM at half the bytes of bf16, so the arithmetic on the way has half the
// time.  Nothing is staged: codes go from their pages into the registers of the warp that uses them, become f16 there (exact: e4m3 has three bits of mantissa)
// and are operands of 16 x 8 x 16 products.
//   S[row, key]    = q K^T        the heads of a group are the rows (for several rows of queries of a sequence: their heads behind one another), keys the
//                                 columns; lane group j of a quad owns channels 16 j .. 16 j + 15 of every 64 for both operands
//   O^T[ch, row]  += V^T P^T      lane (g, j) loads channels g D / 8 .. of keys 2 j, 2 j + 1, 2 j + 8, 2 j + 9 and pairs neighbouring keys by byte permutes;
//                                 P^T needs no exchange, because the accumulator of S is laid out as this operand
// q is divided by a power of two per row, so that f16 holds it.  A page's key scale multiplies its scores.  Its value scale goes into the weights of the second
// product, w = 2^(s + e_v - m'), whose running maximum m' is apart from the softmax's m: w is at most 2^14 whatever the scales, and the mass that f16
// cannot hold is below 2^-38 of the largest for each key.  The sum of weights is that of the unrounded fp32 ones.
constexpr int K8_WARPS = 4, K8_KEYS = 32, K8_MAX_PARTS = 256;
constexpr float K8_LIFT = 14.f;

struct Kv8Attn {
  const __nv_bfloat16* q;
  long q_rs, q_hs;
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int *block_tables, *lens, *row_seq;        // row_seq null: row r is sequence r
  long bt_stride;
  int page, pages, max_keys, R, S, H, Hkv, chunks; // chunks of at most 16 heads of a group
  int pack, splits, subs;                          // rows per block; shares of the keys: blocks, and warps of a block
  float scale_log2;
  float *part_o, *part_lse;
  __nv_bfloat16* out;
  long o_rs, o_hs;
  int* status;
};

__device__ __forceinline__ uint4 ld_codes16(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_codes8(const unsigned char* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_f16_16x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// UP: more than 8 rows of the products are live.
template <int D, bool UP>
__global__ void __launch_bounds__(32 * K8_WARPS, UP ? 2 : 3)
kv8_attn_kernel(const __grid_constant__ Kv8Attn p) {
  pdl_begin();
  constexpr int NH = UP ? 2 : 1, CH = D / 64, MT = D / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int VH = p.Hkv * p.chunks, per_block = min(K8_WARPS, VH), sub = warp / per_block;
  const int vh = blockIdx.z * K8_WARPS + warp % per_block;
  if (sub >= p.subs || vh >= VH) return;
  const int G = p.H / p.Hkv, hk = vh / p.chunks, hc = (vh - hk * p.chunks) * 16, Gc = min(16, G - hc), h0 = hk * G + hc;
  const int parts = p.splits * p.subs, part = blockIdx.y * p.subs + sub;
  const long row = (long)p.Hkv * D;
  const int r0 = blockIdx.x * p.pack, r1 = min(p.R, r0 + p.pack);

  for (int r = r0, rn; r < r1; r = rn) {           // rows r .. rn - 1 are of one sequence
    int seq = r;
    rn = r + 1;
    if (p.row_seq) {
      seq = p.row_seq[r];
      while (rn < r1 && p.row_seq[rn] == seq) ++rn;
    }
    // head and row of this lane's rows g and g + 8 of the products
    int len[NH], head[NH], qrow[NH], most = 0;
    for (int i = r; i < rn; ++i) most = max(most, p.lens[i]);
    most = min(most, p.max_keys);
    if (seq < 0 || seq >= p.S) {
      if (most > 0) atomicCAS(p.status, 0, ERR_BOUNDS);
      most = 0;
    }
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      const int m = u * 8 + g, i = m / Gc;
      qrow[u] = r + i < rn ? r + i : -1;
      head[u] = h0 + m - i * Gc;
      len[u] = qrow[u] >= 0 && most > 0 ? min(max(p.lens[qrow[u]], 0), most) : 0;
    }
    const int tiles = (most + K8_KEYS - 1) / K8_KEYS, per = (tiles + p.splits - 1) / p.splits;
    const int t1 = min(tiles, (int)(blockIdx.y + 1) * per);
    int t = blockIdx.y * per + sub;
    const int* bt = p.block_tables + (long)seq * p.bt_stride;

    uint32_t q[NH][CH][4][2];
    float back[NH];                                // what q was divided by, times the scale
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      uint4 raw[CH][2];
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          raw[c][i] = make_uint4(0u, 0u, 0u, 0u);
          if (qrow[u] >= 0) raw[c][i] = *reinterpret_cast<const uint4*>(p.q + qrow[u] * p.q_rs + head[u] * p.q_hs + c * 64 + j * 16 + i * 8);
          const uint32_t w[4] = {raw[c][i].x, raw[c][i].y, raw[c][i].z, raw[c][i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max((w[k] << 16) & 0x7fffffffu, w[k] & 0x7fff0000u));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max((int)(top >> 23) - 127, -126), 126);
      const float f = pow2f(-e);
      back[u] = pow2f(e) * p.scale_log2;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w[4] = {raw[c][i].x, raw[c][i].y, raw[c][i].z, raw[c][i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = unpack_bf16(w[k]);
            q[u][c][i * 2 + (k >> 1)][k & 1] = pack_half(x.x * f, x.y * f);
          }
        }
    }
    float m[NH], mv[NH], l[NH], acc[NH][MT][4];
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      m[u] = mv[u] = -INFINITY;
      l[u] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][i][e] = 0.f;
    }

    // Lane n of a quad looks up the n-th eight keys of a tile: first row in the pool, exponents of the scales.  Eight keys past the end repeat the tile's first.
    auto look = [&](int t, int& at, float& fk, float& ev) {
      const int k0 = t * K8_KEYS + 8 * j < most ? t * K8_KEYS + 8 * j : t * K8_KEYS;
      const int col = k0 / p.page;
      int pg = bt[col];
      if (pg < 0 || pg >= p.pages) {
        atomicCAS(p.status, 0, ERR_BOUNDS);
        pg = 0;
      }
      at = pg * p.page + (k0 - col * p.page);
      fk = pow2f(scale_exp(p.ks[(long)pg * p.Hkv + hk]));
      ev = (float)scale_exp(p.vs[(long)pg * p.Hkv + hk]);
    };
    // rows past the end repeat the last key: valid memory, its weight is zero
    auto row_in = [&](int t, int n, int i) {
      const int k0 = t * K8_KEYS + (t * K8_KEYS + 8 * n < most ? 8 * n : 0);
      return min(i, most - 1 - k0);
    };
    uint4 kr[4][CH];
    uint4 vr[8];                                   // D = 64: x and y
    auto load_k = [&](int t, int at) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const unsigned char* k = p.k + (long)(__shfl_sync(0xffffffffu, at, n, 4) + row_in(t, n, g)) * row + hk * D + j * 16;
#pragma unroll
        for (int c = 0; c < CH; ++c) kr[n][c] = ld_codes16(k + c * 64);
      }
    };
    auto load_v = [&](int t, int at) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int a = __shfl_sync(0xffffffffu, at, n, 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned char* v = p.v + (long)(a + row_in(t, n, 2 * j + i)) * row + hk * D + g * (D / 8);
          if (D == 128) {
            vr[2 * n + i] = ld_codes16(v);
          } else {
            const uint2 x = ld_codes8(v);
            vr[2 * n + i].x = x.x;
            vr[2 * n + i].y = x.y;
          }
        }
      }
    };
    int at = 0, next_at = 0;
    float fk = 1.f, ev = 0.f, next_fk = 1.f, next_ev = 0.f;
    if (t < t1) {
      look(t, at, fk, ev);
      load_k(t, at);
      load_v(t, at);
      if (t + p.subs < t1) look(t + p.subs, next_at, next_fk, next_ev);
    }
#pragma unroll 1
    for (; t < t1; t += p.subs) {
      const int next = t + p.subs;
      float s[4][4] = {};
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t w[4] = {kr[n][c].x, kr[n][c].y, kr[n][c].z, kr[n][c].w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16_16x8(s[n], q[0][c][k][0], UP ? q[NH - 1][c][k][0] : 0u, q[0][c][k][1], UP ? q[NH - 1][c][k][1] : 0u, halves_of(w[k]), halves_of_hi(w[k]));
        }
      if (next < t1) load_k(next, next_at);
      uint32_t pw[NH][4];
#pragma unroll
      for (int u = 0; u < NH; ++u) {
        float mx = -INFINITY, mxv = -INFINITY, evn[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float f = __shfl_sync(0xffffffffu, fk, n, 4) * back[u];
          evn[n] = __shfl_sync(0xffffffffu, ev, n, 4);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float y = t * K8_KEYS + n * 8 + 2 * j + e < len[u] ? s[n][2 * u + e] * f : -INFINITY;
            s[n][2 * u + e] = y;
            mx = fmaxf(mx, y);
            mxv = fmaxf(mxv, y + evn[n]);
          }
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 2));
        const float was = m[u], was_v = mv[u];
        m[u] = fmaxf(was, mx);
        mv[u] = fmaxf(was_v, mxv);
        const float top = m[u] == -INFINITY ? 0.f : m[u], top_v = mv[u] == -INFINITY ? 0.f : mv[u];      // only scores of -inf so far: all weights are zero
        l[u] *= ex2_approx(was - top);
        const float beta = ex2_approx(was_v - top_v);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float y0 = s[n][2 * u], y1 = s[n][2 * u + 1], lift = evn[n] - top_v + K8_LIFT;
          l[u] += ex2_approx(y0 - top) + ex2_approx(y1 - top);
          pw[u][n] = pack_half(ex2_approx(y0 + lift), ex2_approx(y1 + lift));
        }
        const float b0 = __shfl_sync(0xffffffffu, beta, 8 * j), b1 = __shfl_sync(0xffffffffu, beta, 8 * j + 4);   // rows 2 j, 2 j + 1
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[u][i][0] *= b0; acc[u][i][1] *= b1;
          acc[u][i][2] *= b0; acc[u][i][3] *= b1;
        }
      }
      // channel pair (2 i, 2 i + 1) of a lane's D / 8: rows g and g + 8 of tile i
#pragma unroll
      for (int h = 0; h < 2; ++h)                  // keys 0 .. 15 and 16 .. 31
#pragma unroll
        for (int w = 0; w < MT / 2; ++w) {
          auto word = [&](const uint4& x) { return w == 0 ? x.x : (w == 1 ? x.y : (w == 2 ? x.z : x.w)); };
          const uint32_t a = word(vr[4 * h]), b = word(vr[4 * h + 1]), c = word(vr[4 * h + 2]), d = word(vr[4 * h + 3]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {            // channels 4 w + 2 i, + 1
            const uint32_t x = __byte_perm(a, b, i ? 0x7362 : 0x5140), y = __byte_perm(c, d, i ? 0x7362 : 0x5140);
            const uint32_t a0 = halves_of(x), a1 = halves_of_hi(x), a2 = halves_of(y), a3 = halves_of_hi(y);
#pragma unroll
            for (int u = 0; u < NH; ++u) mma_f16_16x8(acc[u][2 * w + i], a0, a1, a2, a3, pw[u][2 * h], pw[u][2 * h + 1]);
          }
        }
      if (next < t1) {
        load_v(next, next_at);
        fk = next_fk;
        ev = next_ev;
        if (next + p.subs < t1) look(next + p.subs, next_at, next_fk, next_ev);
      }
    }
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
      // O / l = acc 2^-14 / l 2^(m' - m), the two factors apart because their product may be too small for a float; a row without keys: zeros
      const bool none = l[u] == 0.f;
      const float inv = none ? 0.f : 0x1p-14f / l[u], level = none ? 0.f : ex2_approx(mv[u] - m[u]);
      if (parts > 1 && j == 0 && qrow[u] >= 0) p.part_lse[((long)qrow[u] * p.H + head[u]) * parts + part] = none ? -INFINITY : m[u] + log2f(l[u]);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {             // rows 2 j, 2 j + 1 of the products
        const int src = 8 * j + 4 * hh;
        const float f = __shfl_sync(0xffffffffu, inv, src), f2 = __shfl_sync(0xffffffffu, level, src);
        const int qr = __shfl_sync(0xffffffffu, qrow[u], src), hd = __shfl_sync(0xffffffffu, head[u], src);
        const bool no = __shfl_sync(0xffffffffu, none, src);
        if (qr < 0 || (parts > 1 && no)) continue;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[u][i][hh] *= f;
          acc[u][i][hh] *= f2;
          acc[u][i][2 + hh] *= f;
          acc[u][i][2 + hh] *= f2;
        }
        // a lane's channels are g D / 8 + 2 i + (0, 1), i < MT
        if (parts > 1) {
          float* o = p.part_o + (((long)qr * p.H + hd) * parts + part) * D + g * (D / 8);
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            *reinterpret_cast<float4*>(o + 2 * i) = make_float4(acc[u][i][hh], acc[u][i][2 + hh], acc[u][i + 1][hh], acc[u][i + 1][2 + hh]);
        } else {
          __nv_bfloat16* o = p.out + qr * p.o_rs + hd * p.o_hs + g * (D / 8);
#pragma unroll
          for (int i = 0; i < MT; i += 4) {
            uint4 w;
            w.x = pack_bf16(acc[u][i][hh], acc[u][i][2 + hh]);
            w.y = pack_bf16(acc[u][i + 1][hh], acc[u][i + 1][2 + hh]);
            w.z = pack_bf16(acc[u][i + 2][hh], acc[u][i + 2][2 + hh]);
            w.w = pack_bf16(acc[u][i + 3][hh], acc[u][i + 3][2 + hh]);
            *reinterpret_cast<uint4*>(o + 2 * i) = w;
          }
        }
      }
    }
  }
}

// out[row, head] = sum_s 2^(lse_s - top) o_s / sum_s 2^(lse_s - top) over the shares (at most 256): a block per (row, head), its warps take every fourth share.
template <int D>
__global__ void __launch_bounds__(128)
kv8_merge_kernel(const float* part_o, const float* part_lse, int parts, int H, __nv_bfloat16* out, long o_rs, long o_hs) {
  pdl_begin();
  constexpr int PER = D / 32;
  __shared__ float weight[K8_MAX_PARTS], sums[4][D], red[4];
  const long r = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* lse = part_lse + r * parts;
  const float a = threadIdx.x < parts ? lse[threadIdx.x] : -INFINITY, b = threadIdx.x + 128 < parts ? lse[threadIdx.x + 128] : -INFINITY;
  float top = fmaxf(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  const float wa = a == -INFINITY ? 0.f : ex2_approx(a - top), wb = b == -INFINITY ? 0.f : ex2_approx(b - top);
  weight[threadIdx.x] = wa;
  weight[threadIdx.x + 128] = wb;
  float den = wa + wb;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  if (lane == 0) red[warp] = den;
  __syncthreads();
  den = (red[0] + red[1]) + (red[2] + red[3]);
  const float* po = part_o + r * parts * D + lane * PER;
  float acc[PER] = {};
#pragma unroll 4
  for (int s = warp; s < parts; s += 4) {
    const float w = weight[s];
    if (w == 0.f) continue;                        // a share without keys has written no sum
    float x[PER];
    if (PER == 4) {
      const float4 y = *reinterpret_cast<const float4*>(po + (long)s * D);
      x[0] = y.x; x[1] = y.y; x[PER - 2] = y.z; x[PER - 1] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(po + (long)s * D);
      x[0] = y.x; x[1] = y.y;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = fmaf(x[i], w, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) sums[warp][lane * PER + i] = acc[i];
  __syncthreads();
  const float f = den != 0.f ? 1.0f / den : 0.f;   // not a number stays one
  const long row = r / H, head = r - row * H;
  for (int c = threadIdx.x * 2; c < D; c += 256) {
    const float x = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]), y = (sums[0][c + 1] + sums[1][c + 1]) + (sums[2][c + 1] + sums[3][c + 1]);
    *reinterpret_cast<uint32_t*>(out + row * o_rs + head * o_hs + c) = pack_bf16(x * f, y * f);
  }
}

// Shares of a row's keys: about 24 warps per SM in all, two rounds of the twelve that fit it, at least two tiles of 32 keys each.  The number depends on the
// rows, the heads and the tables' width, never on lengths: a row's result is the same whatever its neighbours hold.
static void kv8_shares(int blocks_of_rows, int VH, int max_keys, int& splits, int& subs) {
  subs = VH < K8_WARPS ? K8_WARPS / VH : 1;
  const long warps = (long)blocks_of_rows * VH, target = 24L * sm_count();
  const int tiles = (max_keys + K8_KEYS - 1) / K8_KEYS;
  long parts = (target + warps - 1) / warps;
  if (parts > tiles / 2) parts = tiles / 2;
  if (parts > K8_MAX_PARTS) parts = K8_MAX_PARTS;
  if (parts < 1) parts = 1;
  if (subs > parts) subs = (int)parts;
  splits = (int)(parts + subs - 1) / subs;
  if (splits * subs > K8_MAX_PARTS) splits = K8_MAX_PARTS / subs;
}
// Rows that share a block: as many as fill the products' sixteen rows, where rows share sequences at all.
static int kv8_pack(int R, int S, int G, bool mapped) { return mapped && R > S && G <= 8 ? 16 / G : 1; }

}  // namespace omni

using namespace omni;

static bool misaligned(const void* a, const void* b, const void* c, const void* d) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15;
}

// k, v bf16 [T, Hkv, D] at the given pitches (multiples of 8); pages uint8 [n_slots / page, page, Hkv, D], scales fp32 [n_slots / page, Hkv]; slots int32 [T],
// below zero: not written.  The rows of a page follow one another, with fewer than 128 others that are not written between two of them.
extern "C" int omni_kv8_write(const void* k, const void* v, long k_rs, long k_hs, long v_rs, long v_hs, void* kc, void* vc, float* ks, float* vs,
                              const int* slots, long n_slots, int T, int Hkv, int D, int page, int* status, void* stream) {
  if (T <= 0) return RC_OK;
  if (Hkv < 1 || Hkv > 65535 || (D != 64 && D != 128) || page < 1 || ((k_rs | k_hs | v_rs | v_hs) & 7) || misaligned(k, v, kc, vc) || n_slots > 0x7fffffffL) return RC_BAD_ARG;
  // rows per block: 64, or fewer where that leaves SMs without blocks
  int chunk = 64;
  while (chunk > 4 && (long)((T + chunk - 1) / chunk) * Hkv < 4L * sm_count()) chunk /= 2;
  const Kv8Write p = {(const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_rs, k_hs, v_rs, v_hs, (unsigned char*)kc, (unsigned char*)vc, ks, vs, slots, n_slots, T, Hkv, page,
                      chunk, status};
  const dim3 grid((unsigned)((T + chunk - 1) / chunk), (unsigned)Hkv);
  launch_overlapped(D == 64 ? kv8_write_kernel<64> : kv8_write_kernel<128>, grid, 256, 0, (cudaStream_t)stream, p);
  return (int)cudaGetLastError();
}

// n lists: index[i] int32 slots of rows[i] rows (tables = 0; below zero: zeros), or a block table of rows[i] tokens, to rows row0[i] .. of k, v bf16 [.., Hkv, D].
extern "C" int omni_kv8_read(const void* kc, const void* vc, const float* ks, const float* vs, int n, const void* const* index, const long* row0, const long* rows,
                             int tables, void* k, void* v, long n_slots, int Hkv, int D, int page, int* status, void* stream) {
  if (Hkv < 1 || (D != 64 && D != 128) || page < 1 || misaligned(kc, vc, k, v) || n_slots > 0x7fffffffL) return RC_BAD_ARG;
  for (int i0 = 0; i0 < n; i0 += K8_TABLES) {
    const int m = n - i0 < K8_TABLES ? n - i0 : K8_TABLES;
    Kv8Read p = {};
    p.kc = (const unsigned char*)kc; p.vc = (const unsigned char*)vc; p.ks = ks; p.vs = vs; p.k = (__nv_bfloat16*)k; p.v = (__nv_bfloat16*)v;
    p.n_slots = n_slots; p.Hkv = Hkv; p.D = D; p.page = page; p.tables = tables; p.status = status;
    long most = 0;
    for (int i = 0; i < m; ++i) {
      p.index[i] = (const int*)index[i0 + i];
      p.row0[i] = row0[i0 + i];
      p.rows[i] = rows[i0 + i];
      if (rows[i0 + i] > most) most = rows[i0 + i];
    }
    if (most <= 0) continue;
    long blocks = (most * (Hkv * D / 16) + 255) / 256;
    if (blocks > 16L * sm_count()) blocks = 16L * sm_count();
    launch_overlapped(kv8_read_kernel, dim3((unsigned)blocks, (unsigned)m), 256, 0, (cudaStream_t)stream, p);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
  }
  return RC_OK;
}

// Shares per (row, head) that omni_kv8_attn will write: sizes its scratch (fp32, shares x D and shares x 1).
extern "C" int omni_kv8_attn_shares(int R, int S, int H, int Hkv, int mapped, int max_keys) {
  if (R < 1 || Hkv < 1 || H < Hkv) return 1;
  const int G = H / Hkv, pack = kv8_pack(R, S, G, mapped != 0);
  int splits, subs;
  kv8_shares((R + pack - 1) / pack, Hkv * ((G + 15) / 16), max_keys, splits, subs);
  return splits * subs;
}

// q, out bf16 [R, H, D] at the given pitches (multiples of 8); pages as above, their size a multiple of 8; block_tables int32 [S, max_keys / page] at bt_stride;
// lens int32 [R]: keys that a row sees; row_seq int32 [R] or null (R = S).
extern "C" int omni_kv8_attn(const void* q, long q_rs, long q_hs, const void* kc, const void* vc, const float* ks, const float* vs, int pages, int page,
                             const int* block_tables, long bt_stride, const int* lens, const int* row_seq, int R, int S, int H, int Hkv, int D, int max_keys,
                             float scale, float* part_o, float* part_lse, void* out, long o_rs, long o_hs, int* status, void* stream) {
  if (R <= 0) return RC_OK;
  if (Hkv < 1 || H < 1 || H % Hkv || (D != 64 && D != 128) || page < 8 || (page & 7) || max_keys < 1 || pages < 1 || (long)pages * page > 0x7fffffffL ||
      (!row_seq && R != S) || ((q_rs | q_hs | o_rs | o_hs) & 7) || misaligned(q, kc, vc, out))
    return RC_BAD_ARG;
  Kv8Attn p = {};
  const int G = H / Hkv;
  p.chunks = (G + 15) / 16;
  const int VH = Hkv * p.chunks;
  if ((VH + K8_WARPS - 1) / K8_WARPS > 65535) return RC_BAD_ARG;
  p.pack = kv8_pack(R, S, G, row_seq != nullptr);
  const int blocks = (R + p.pack - 1) / p.pack;
  kv8_shares(blocks, VH, max_keys, p.splits, p.subs);
  const int parts = p.splits * p.subs;
  if (parts > 1 && (!part_o || !part_lse)) return RC_BAD_ARG;
  p.q = (const __nv_bfloat16*)q; p.q_rs = q_rs; p.q_hs = q_hs; p.k = (const unsigned char*)kc; p.v = (const unsigned char*)vc; p.ks = ks; p.vs = vs;
  p.block_tables = block_tables; p.lens = lens; p.row_seq = row_seq; p.bt_stride = bt_stride; p.page = page; p.pages = pages; p.max_keys = max_keys;
  p.R = R; p.S = S; p.H = H; p.Hkv = Hkv; p.scale_log2 = scale * 1.4426950408889634f; p.part_o = part_o; p.part_lse = part_lse;
  p.out = (__nv_bfloat16*)out; p.o_rs = o_rs; p.o_hs = o_hs; p.status = status;
  const dim3 grid((unsigned)blocks, (unsigned)p.splits, (unsigned)((VH + K8_WARPS - 1) / K8_WARPS));
  cudaStream_t st = (cudaStream_t)stream;
  const bool up = (p.chunks > 1 ? 16 : G) * p.pack > 8;
  launch_with(R <= 16, 1, D == 64 ? (up ? kv8_attn_kernel<64, true> : kv8_attn_kernel<64, false>) : (up ? kv8_attn_kernel<128, true> : kv8_attn_kernel<128, false>), grid,
              32 * K8_WARPS, 0, st, p);
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  if (parts == 1) return RC_OK;
  launch_overlapped(D == 64 ? kv8_merge_kernel<64> : kv8_merge_kernel<128>, (unsigned)((long)R * H), 128, 0, st, part_o, part_lse, parts, H, (__nv_bfloat16*)out, o_rs, o_hs);
  return (int)cudaGetLastError();
}
