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

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {       // of both halves
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
__device__ __forceinline__ uint32_t largest_of(uint4 u) {                // magnitudes of eight bf16, of those in even and in odd places
  return max2(max2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), max2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
  return ((w & 0x7fffu) < 0x7f80u ? w & 0x7fffu : 0u) | ((w & 0x7fff0000u) < 0x7f800000u ? w & 0x7fff0000u : 0u);
}
__device__ __forceinline__ uint32_t largest_finite(uint4 u) { return largest_of(make_uint4(finite_of(u.x), finite_of(u.y), finite_of(u.z), finite_of(u.w))); }

struct Kv8Run {
  int t, end, low, page;                 // first row and behind the last one, lowest row of the page that is written
  int slot;                              // of the first row, if every next row is in the next slot; -1 otherwise
};

// A run is the rows of one page, with fewer than 128 rows that are not written between two of them.  A block finds the runs that begin among `chunk` rows and deals out
// one head of each (keys or values) to its warps: one warp where there are many (decoded tokens, small pages), up to four where there are few.  Largest magnitude, scale,
// rounding again of the rows before the first written one where the scale grows, codes.  Eight channels per lane: D / 8 lanes are a row, a warp takes 2048 / D rows at
// a time, in registers from the first look to the codes unless the run is longer.  16435 rows of 8 heads of 128 in pages of 64 (101 MB, 15 us at the rate of memory)
// take 28.6 us: 109 instructions a warp for 512 bytes, the search for runs and both passes among them, and warps that wait while a block looks for its runs.  One
// warp per run with two looks at memory took 58; four heads a block, so that the runs are looked for less often, the same 28.6.  Seven rows take 3.5 us, a launch.
template <int D>
__global__ void __launch_bounds__(256, 3)
kv8_write_kernel(const __grid_constant__ Kv8Write p) {
  pdl_begin();
  constexpr int LANES = D / 8, ROWS = 32 / LANES, HELD = 8;
  __shared__ Kv8Run runs[64];
  __shared__ int begins[64], n_begin[2];
  __shared__ uint32_t largest[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t0 = blockIdx.x / p.Hkv * p.chunk, h = blockIdx.x % p.Hkv;
  if (threadIdx.x < 8) largest[threadIdx.x] = 0;
  if (threadIdx.x < 64) {                // `chunk` is at most 64
    const int t = t0 + threadIdx.x;
    bool first = false;
    if ((int)threadIdx.x < p.chunk && t < p.T) {
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
    if (first) begins[warp * 32 + __popc(m & ((1u << lane) - 1))] = t;
    if (lane == 0) n_begin[warp] = __popc(m);
  }
  __syncthreads();
  const int n_front = n_begin[0], n_runs = n_front + n_begin[1];
  for (int i = warp; i < n_runs; i += 8) {
    const int t1 = begins[i < n_front ? i : i - n_front + 32];
    const int first = p.slots[t1], at = first / p.page, base = at * p.page;
    int low = p.page, end = t1;
    bool next = true;
    for (int skipped = 0, from = t1;;) {                                   // 32 rows from behind the last ones
      const int s = from + lane < p.T ? p.slots[from + lane] : -1;
      const bool ok = s >= 0 && s < p.n_slots, mine = ok && s >= base && s - base < p.page;
      const unsigned others = __ballot_sync(0xffffffffu, ok && !mine);
      const unsigned ours = __ballot_sync(0xffffffffu, mine) & (others ? (others & -others) - 1 : 0xffffffffu);
      if (!ours) {
        skipped += 32;
        from += 32;
        if (others || skipped >= K8_GAP || from >= p.T) break;
        continue;
      }
      const int rows = 32 - __clz(ours);
      next = next && __all_sync(0xffffffffu, lane >= rows || s == first + (from + lane - t1));
      low = min(low, (int)__reduce_min_sync(0xffffffffu, ours >> lane & 1 ? (unsigned)(s - base) : (unsigned)p.page));
      from += rows;
      end = from;
      skipped = 0;
      if (others) break;
    }
    if (lane == 0) runs[i] = {t1, end, low, at, next ? first : -1};
  }
  __syncthreads();
  const int sub = lane / LANES, ch = lane % LANES * 8;
  const int team = n_runs <= 1 ? 4 : (n_runs == 2 ? 2 : 1), teams = 8 / team, mate = warp % team, step = team * ROWS;      // warps of an item, rows they take at once
  for (int round = 0; round < 2 * n_runs; round += teams) {
    const int item = round + warp / team;
    const bool live = item < 2 * n_runs, val = item & 1;
    Kv8Run run = {0, 0, 0, 0, 0};
    if (live) run = runs[item >> 1];
    const __nv_bfloat16* x = (val ? p.v + h * p.v_hs : p.k + h * p.k_hs) + ch;
    const long rs = val ? p.v_rs : p.k_rs;
    unsigned char* cache = (val ? p.vc : p.kc) + h * D + ch;
    float* my_scale = (val ? p.vs : p.ks) + (long)run.page * p.Hkv + h;
    const int old = run.low > 0 ? scale_exp(*my_scale) : K8_LEAST, pitch = p.Hkv * D;
    const int row = run.t + mate * ROWS, batch = HELD * step, rows = run.end - run.t;         // the warp's first rows, rows of a team's registers
    uint4 u[HELD];
    auto load = [&](int t) {             // rows t, t + step, .. of a run without gaps
      const __nv_bfloat16* from = x + (t + sub) * rs;
#pragma unroll
      for (int i = 0; i < HELD; ++i, t += step, from += step * rs) {
        if (t >= run.end) break;
        u[i] = make_uint4(0u, 0u, 0u, 0u);
        if (t + sub < run.end) u[i] = *reinterpret_cast<const uint4*>(from);
      }
    };
    // largest magnitudes: of floats, they are ordered like integers.  A run's first rows are looked at last, and stay.
    uint32_t pair = 0;
    if (run.slot >= 0) {
      for (int b = (rows - 1) / batch; b >= 0; --b) {
        load(row + b * batch);
        uint32_t here = 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
          if (row + b * batch + i * step >= run.end) break;
          here = max2(here, largest_of(u[i]));
        }
        if ((here & 0xffffu) >= 0x7f80u || here >= 0x7f800000u) {          // infinities and NaN set no scale
          here = 0;
#pragma unroll
          for (int i = 0; i < HELD; ++i) {
            if (row + b * batch + i * step >= run.end) break;
            here = max2(here, largest_finite(u[i]));
          }
        }
        pair = max2(pair, here);
      }
    } else {
      for (int t = row + sub; t < run.end; t += step)
        if (p.slots[t] >= 0 && p.slots[t] < p.n_slots) pair = max2(pair, largest_finite(*reinterpret_cast<const uint4*>(x + t * rs)));
    }
    uint32_t most = __reduce_max_sync(0xffffffffu, max(pair << 16, pair & 0xffff0000u));
    if (team > 1) {
      if (lane == 0) atomicMax(&largest[warp / team], most);
      __syncthreads();                                                     // the scale has been read, too
      most = largest[warp / team];
    }
    // least e with most <= 1.75 * 2^(8 + e)
    const int need = max((int)(most >> 23) - 127 - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0), K8_LEAST), e = max(need, old);
    if (run.low > 0 && e > old) {
      const float f = pow2f(max(old - e, -126));                           // at 2^-126 every code becomes zero, as it would below
      for (int r = mate * ROWS + sub; r < run.low; r += step) {
        unsigned char* c = cache + ((long)run.page * p.page + r) * pitch;
        uint2 o = *reinterpret_cast<const uint2*>(c);
        uint32_t w[2] = {o.x, o.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 a = floats_of(halves_of(w[i])), b = floats_of(halves_of_hi(w[i]));
          w[i] = codes_of(a.x * f, a.y * f, b.x * f, b.y * f);
        }
        *reinterpret_cast<uint2*>(c) = make_uint2(w[0], w[1]);
      }
    }
    __syncwarp();                                                          // all lanes have read the scale
    if (live && mate == 0 && lane == 0) *my_scale = pow2f(e);
    // A power of two of a bf16 is one: exact, but for what is below every code.
    const __nv_bfloat162 f = __bfloat162bfloat162(__float2bfloat16(pow2f(-e)));
    auto store = [&](uint4 r, int slot) {
      uint32_t w[4] = {r.x, r.y, r.z, r.w}, c[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 y = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w[j]), f);
        w[j] = *reinterpret_cast<const uint32_t*>(&y);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 lo = unpack_bf16(w[2 * j]), hi = unpack_bf16(w[2 * j + 1]);
        c[j] = codes_of(lo.x, lo.y, hi.x, hi.y);
      }
      *reinterpret_cast<uint2*>(cache + (long)slot * pitch) = make_uint2(c[0], c[1]);
    };
    if (run.slot >= 0) {
      for (int t0 = row; t0 < run.end; t0 += batch) {
        if (t0 != row) load(t0);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
          const int t = t0 + i * step;
          if (t >= run.end) break;
          if (t + sub < run.end) store(u[i], run.slot + (t + sub - run.t));
        }
      }
    } else {
      for (int t = row + sub; t < run.end; t += step) {
        int slot = p.slots[t];
        if (slot >= p.n_slots) slot = -1;
        if (slot >= 0)                   // the same slot twice: the last row is written
          for (int o = t + 1; o < run.end; ++o)
            if (p.slots[o] == slot) slot = -1;
        if (slot >= 0) store(*reinterpret_cast<const uint4*>(x + t * rs), slot);
      }
    }
    if (team > 1) break;                 // all items had a team
  }
}

// ----------------------------------------------------------------------------------------------------------------------------------------- read
constexpr int K8_TABLES = 16;
struct Kv8Read {
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int* index[K8_TABLES];           // slots of the rows, or block tables
  long row0[K8_TABLES];                  // first row written
  int rows[K8_TABLES];
  __nv_bfloat16 *k, *v;                  // [.., Hkv, D]
  long n_slots;
  int Hkv, D, page, shift, tables;       // tables: index is block tables; shift: log2 of the page's size, -1 if it has none
  int* status;
};

// Eight codes of a row per thread, keys and values, four rows at once: 16-byte stores side by side.  What a thread's place in a row says is worked out once.
// Bound by memory: 18185 rows of 8 heads of 128 (112 MB) take 18.7 us, 5985 GB/s; 128 x 350 rows 46.0 us, 5996 GB/s.
__global__ void __launch_bounds__(256)
kv8_read_kernel(const __grid_constant__ Kv8Read p) {
  pdl_begin();
  const int seg = blockIdx.y, vecs = p.Hkv * p.D / 8, rows = p.rows[seg], width = vecs < 256 ? vecs : 256, lines = 256 / width;
  const int* index = p.index[seg];
  if ((int)threadIdx.x >= lines * width) return;
  const int line = threadIdx.x / width;
  const long row_elems = (long)p.Hkv * p.D;
  for (int vec = threadIdx.x - line * width; vec < vecs; vec += width) {
    const int c = vec * 8, head = c / p.D;
    for (int t0 = (blockIdx.x * lines + line) * 4; t0 < rows; t0 += gridDim.x * lines * 4) {
      long slot[4];
      uint2 code[4][2];
      float f[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i;
        slot[i] = -1;
        if (t >= rows) continue;
        if (p.tables) {
          const int at = p.shift >= 0 ? t >> p.shift : t / p.page, pg = index[at];
          slot[i] = pg < 0 ? p.n_slots : (long)pg * p.page + (t - at * p.page);
        } else {
          slot[i] = index[t];
        }
        if (slot[i] >= p.n_slots) {
          atomicCAS(p.status, 0, ERR_BOUNDS);
          slot[i] = -1;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        code[i][0] = code[i][1] = make_uint2(0u, 0u);
        f[i][0] = f[i][1] = 0.f;
        if (slot[i] < 0) continue;
        const long scale_at = (long)(p.shift >= 0 ? (int)slot[i] >> p.shift : (int)slot[i] / p.page) * p.Hkv + head, from = slot[i] * row_elems + c;
        code[i][0] = *reinterpret_cast<const uint2*>(p.kc + from);
        code[i][1] = *reinterpret_cast<const uint2*>(p.vc + from);
        f[i][0] = pow2f(scale_exp(p.ks[scale_at]));
        f[i][1] = pow2f(scale_exp(p.vs[scale_at]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (t0 + i >= rows) break;
        const long to = (p.row0[seg] + t0 + i) * row_elems + c;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint32_t w[2] = {code[i][b].x, code[i][b].y};
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 lo = floats_of(halves_of(w[j])), hi = floats_of(halves_of_hi(w[j]));
            o[2 * j] = pack_bf16(lo.x * f[i][b], lo.y * f[i][b]);
            o[2 * j + 1] = pack_bf16(hi.x * f[i][b], hi.y * f[i][b]);
          }
          *reinterpret_cast<uint4*>((b ? p.v : p.k) + to) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------ attention
// One row of queries reads every key and value of its sequence once: a stream from HBM at half the bytes of bf16, so the arithmetic on the way has half the
// time, 23 bytes a clock and SM.  A warp that loads for itself spends it on addresses and on waiting (64 sequences of 2500 to 4096 keys, 8 KV heads of 128: 33 instructions a
// key and head, 152 us).  Here one warp of a block fetches pages by TMA, all heads of eight to 32 rows by one copy into [head][row][channel], swizzled so that nothing below
// meets a bank twice, through a ring of three or six stages; the others take 32 keys of one head a stage each.  Codes become f16 in registers (exact: e4m3 has three bits
// of mantissa) and are operands of 16 x 8 x 16 products.
//   S[row, key]    = q K^T        the heads of a group are the rows (for several rows of queries of a sequence: their heads behind one another), keys the
//                                 columns; lane group j of a quad owns channels D / 4 j .. of both operands
//   O^T[ch, row]  += V^T P^T      lane (g, j) holds channels g D / 8 .. of keys 2 j, 2 j + 1, 2 j + 8, 2 j + 9 and pairs neighbouring keys by byte permutes;
//                                 P^T needs no exchange, because the accumulator of S is laid out as this operand
// q is divided by a power of two per row, so that f16 holds it.  A page's key scale multiplies its scores.  Its value scale goes into the weights of the second
// product, w = 2^(s + e_v - m'), whose running maximum m' is apart from the softmax's m: w is at most 2^15 whatever the scales, and the mass that f16
// cannot hold is below 2^-38 of the largest for each key.  The sum of weights is that of the unrounded fp32 ones.
// Blocks are persistent, one an SM: a share (a run of keys of a row and of up to eight heads) follows another in the ring without a pause.
// 64 sequences of 2458 to 4096 keys, 32 heads on 8 of 128 (430 MB) 88 us with the joining of shares, 4.9 TB/s; one of 131071, 64 heads on 8, 51 us, 5.3 TB/s; one of 100 6 us.
// What is left: a share's beginning and end, some 4000 clocks in which the ring does not run full; shares that do not divide among the SMs; 650 instructions a warp
// for 32 keys, which keep a scheduler's two warps two thirds busy.
constexpr int K8_MAX_PARTS = 256, K8_MAX_GROUP = 128, K8_LISTED = 512;
constexpr float K8_LIFT = 14.f, K8_SLACK = 1.f;     // together below f16's 2^16
// Warps that compute, and the keys of a stage that each of them takes.  (Sixteen warps of 16 keys: 96 registers, which spill, and more instructions a key.)
// Sixteen rows of 128 channels leave registers for 16 keys at a time, and half as large stages.
constexpr int K8_WARPS = 8;
constexpr int k8_keys(int D, bool up) { return D == 128 && up ? 16 : 32; }

struct Kv8Attn {
  CUtensorMap mk, mv;                              // codes: {channels, slots, heads}, boxes {D, unit, heads_block}
  const __nv_bfloat16* q;
  long q_rs, q_hs;
  const float *ks, *vs;
  const int *block_tables, *lens, *row_seq;        // row_seq null: row r is sequence r
  long bt_stride;
  int page, shift, pages, max_keys, R, S, H, Hkv;  // shift: log2 of the page's size, -1 if it has none
  int chunks, heads, groups;                       // chunks of at most 16 heads of a group; KV heads of a block, blocks of them
  int pack, unit, subs;                            // rows per block; rows of a copy; warps that share a head's keys
  int share, splits, row_blocks;                   // keys of a share, shares of a row at most; blocks of rows
  bool listed;                                     // blocks take the shares there are; else a number stands for every share there may be
  float scale_log2;
  float *part_o, *part_lse;
  __nv_bfloat16* out;
  long o_rs, o_hs;
  int* status;
};

__device__ __forceinline__ void mma_f16_16x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Shared memory by its address, as loads that the compiler may move between barriers.
__device__ __forceinline__ uint4 shared4(uint32_t addr) { return *reinterpret_cast<const uint4*>(__cvta_shared_to_generic(addr)); }
__device__ __forceinline__ uint2 shared2(uint32_t addr) { return *reinterpret_cast<const uint2*>(__cvta_shared_to_generic(addr)); }

// What a share is, for the warp that fetches and for those that compute alike: rows r .. rn - 1 of one sequence, its keys from `from` to `to`.
struct Kv8Pass {
  int seq, rn, most, from, to;
};
__device__ __forceinline__ Kv8Pass kv8_pass(const Kv8Attn& p, int r, int r1, int split) {
  Kv8Pass a;
  a.seq = r;
  a.rn = r + 1;
  if (p.row_seq) {
    a.seq = p.row_seq[r];
    while (a.rn < r1 && p.row_seq[a.rn] == a.seq) ++a.rn;
  }
  a.most = 0;
  for (int i = r; i < a.rn; ++i) a.most = max(a.most, p.lens[i]);
  a.most = min(a.most, p.max_keys);
  if (a.seq < 0 || a.seq >= p.S) {
    if (a.most > 0) atomicCAS(p.status, 0, ERR_BOUNDS);
    a.most = 0;
  }
  a.from = min(a.most, split * p.share);
  a.to = min(a.most, a.from + p.share);
  return a;
}
// Shares that a block of rows has: one at least.
__device__ __forceinline__ int kv8_count(const int* lens, int rb, int pack, int R, int max_keys, int share) {
  int most = 0;
  for (int i = rb * pack; i < min(R, (rb + 1) * pack); ++i) most = max(most, lens[i]);
  return max(1, (min(most, max_keys) + share - 1) / share);
}
// The shares there are, one after another: `before` [row_blocks + 1] counts those of the blocks of rows before one.  Without it as many of every
// block, the first ones of all first; those behind a block's end are empty.
struct Kv8Item {
  int rb, group, split;
};
__device__ __forceinline__ Kv8Item kv8_item(const Kv8Attn& p, const int* before, int item) {
  const int k = item / p.groups, group = item - k * p.groups;
  if (!p.listed) {
    const int split = k / p.row_blocks;
    return {k - split * p.row_blocks, group, split};
  }
  int lo = 0, hi = p.row_blocks;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= k) lo = mid; else hi = mid;
  }
  return {lo, group, k - before[lo]};
}
__device__ __forceinline__ int kv8_column(const Kv8Attn& p, int key) { return p.shift >= 0 ? key >> p.shift : key / p.page; }
__device__ __forceinline__ int kv8_page(const Kv8Attn& p, int pg) {
  if (pg >= 0 && pg < p.pages) return pg;
  atomicCAS(p.status, 0, ERR_BOUNDS);
  return 0;
}

// UP: more than 8 rows of the products are live.  MANY: they may be of several rows of queries.
template <int D, bool UP, bool MANY>
__global__ void __launch_bounds__(32 * (K8_WARPS + 1), 1)
kv8_attn_kernel(const __grid_constant__ Kv8Attn p) {
  extern __shared__ __align__(1024) unsigned char ring[];
  __shared__ __align__(8) unsigned long long bars[12];
  __shared__ int s_abort, before[K8_LISTED + 1];
  __shared__ float sums[K8_WARPS][UP ? 16 : 8];
  constexpr int NH = UP ? 2 : 1, CH = D / 64, MT = D / 16, CW = K8_WARPS, KEYS = D == 128 && UP ? 16 : 32, NE = KEYS / 8, STAGES = 96 / KEYS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int VH = p.heads * p.chunks, keys = p.subs * KEYS, half = keys * p.heads * D;     // of a stage; bytes of its K
  const uint32_t base = smem_u32(ring), full = smem_u32(bars), empty = full + 8 * STAGES;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, VH * p.subs);
    }
    s_abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_begin();
  int items = p.row_blocks * p.splits;
  if (p.listed) {
    for (int rb = threadIdx.x; rb < p.row_blocks; rb += blockDim.x) before[rb + 1] = kv8_count(p.lens, rb, p.pack, p.R, p.max_keys, p.share);
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    if (warp == 0) {
      int run = 0;
      for (int i0 = 0; i0 < p.row_blocks; i0 += 32) {
        int n = i0 + lane < p.row_blocks ? before[i0 + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int up = __shfl_up_sync(0xffffffffu, n, o);
          if (lane >= o) n += up;
        }
        if (i0 + lane < p.row_blocks) before[i0 + lane + 1] = run + n;
        run += __shfl_sync(0xffffffffu, n, 31);
      }
    }
    __syncthreads();
    items = before[p.row_blocks];
  }
  items *= p.groups;
  int c = 0;                                       // stages so far

  if (warp == CW) {
    // the pages of a share, a unit a lane
    const int units = keys / p.unit, unit_bytes = p.unit * p.heads * D;
    const bool plain = p.pack == 1 && !p.row_seq;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const Kv8Item w = kv8_item(p, before, item);
      const int rb = w.rb, group = w.group, split = w.split, r1 = min(p.R, (rb + 1) * p.pack);
      for (int r = rb * p.pack; r < r1;) {
        // the first pages are asked for along with the length
        const int guess = plain && lane < units ? p.block_tables[(long)r * p.bt_stride + kv8_column(p, min(split * p.share + lane * p.unit, p.max_keys - 1))] : 0;
        const Kv8Pass a = kv8_pass(p, r, r1, split);
        r = a.rn;
        const int* bt = p.block_tables + (long)a.seq * p.bt_stride;
        auto slot_of = [&](int key) {
          const int col = kv8_column(p, key);
          return kv8_page(p, bt[col]) * p.page + (key - col * p.page);
        };
        int key = a.from + lane * p.unit, slot = 0;
        if (lane < units && key < a.to) slot = plain ? kv8_page(p, guess) * p.page + (key - kv8_column(p, key) * p.page) : slot_of(key);
        for (int k0 = a.from; k0 < a.to; k0 += keys, ++c) {
          const int s = c % STAGES;
          if (!mbar_wait(empty + 8 * s, ((c / STAGES) & 1) ^ 1, &s_abort, p.status, ERR_WAIT_EMPTY)) break;
          const int n = min(units, (a.to - k0 + p.unit - 1) / p.unit);
          if (lane == 0) mbar_expect_tx(full + 8 * s, 2 * n * unit_bytes);
          __syncwarp();
          if (lane < n) {
            const uint32_t at = base + s * 2 * half + lane * unit_bytes;
            tma_load_3d(at, &p.mk, full + 8 * s, 0, slot, group * p.heads);
            tma_load_3d(at + half, &p.mv, full + 8 * s, 0, slot, group * p.heads);
          }
          key += keys;
          if (lane < units && key < a.to) slot = slot_of(key);
        }
      }
    }
    if (*(volatile int*)&s_abort) {                // copies in flight end before the block does
      for (int i = 0; i < STAGES; ++i) {
        const unsigned long long t0 = globaltimer_ns();
        const int last = c - 1 - i;
        if (last < 0) break;
        while (!mbar_try_wait(full + 8 * (last % STAGES), (last / STAGES) & 1) && globaltimer_ns() - t0 < WAIT_LIMIT_NS) {}
      }
    }
    return;
  }

  const int vh = warp % VH, sub = warp / VH;
  if (sub >= p.subs) return;
  const int G = p.H / p.Hkv, head_in = vh / p.chunks, hc = (vh - head_in * p.chunks) * 16, Gc = min(16, G - hc);
  // where a lane's pieces of eight rows are, from the first of them: K rows g, V rows 2 j and 2 j + 1
  uint32_t k_at[CH], v_at[2];
#pragma unroll
  for (int x = 0; x < CH; ++x) k_at[x] = D == 128 ? g * 128 + (((2 * j + x) ^ g) << 4) : g * 64 + ((j ^ ((g >> 1) & 3)) << 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = 2 * j + i;
    v_at[i] = D == 128 ? row * 128 + ((g ^ row) << 4) : row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8;
  }
  uint32_t eight[NE];                              // this warp's eights of a stage
#pragma unroll
  for (int n = 0; n < NE; ++n) {
    const int k = sub * KEYS + n * 8, u = k / p.unit;
    eight[n] = (uint32_t)((u * p.heads + head_in) * p.unit + (k - u * p.unit)) * D;
  }

  // While the stages of a share go by, the next one's length and first pages, then its scales are fetched, and its queries before its sums are written, where a row is its
  // own sequence (`plain`): what follows from them does not stop the ring.
  const bool plain = p.pack == 1 && !p.row_seq;
  const uint32_t my_q = base + STAGES * 2 * CW * KEYS * D + warp * (NH * CH * 1024) + lane * 16;      // this warp's q: words of a lane in fours
  if ((int)blockIdx.x >= items) return;
  Kv8Item at = kv8_item(p, before, blockIdx.x), next = at;
  int next_len = 0, next_page = 0;
  float next_ks = 1.f, next_vs = 1.f;
  uint4 raw[NH][CH][2];
  auto first_key = [&](int split) { return split * p.share + lane / NE * keys + sub * KEYS + lane % NE * 8; };
  auto fetch_pages = [&] {
    next_len = p.lens[next.rb];
    next_page = p.block_tables[(long)next.rb * p.bt_stride + kv8_column(p, min(first_key(next.split), p.max_keys - 1))];
  };
  auto fetch_scales = [&] {
    const int key = first_key(next.split), hn = next.group * p.heads + head_in;
    const int pg = key < min(next_len, p.max_keys) && key < (next.split + 1) * p.share ? kv8_page(p, next_page) : 0;
    if (hn < p.Hkv) {
      next_ks = p.ks[(long)pg * p.Hkv + hn];
      next_vs = p.vs[(long)pg * p.Hkv + hn];
    }
  };
  // rows g and g + 8 of the products: their heads behind one another, row by row
  auto fetch_queries = [&](int r, int rn, int h0, bool real) {
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      const int m = u * 8 + g, i = m / Gc;
#pragma unroll
      for (int x = 0; x < CH; ++x)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          raw[u][x][k] = real && r + i < rn ? *reinterpret_cast<const uint4*>(p.q + (r + i) * p.q_rs + (h0 + m - i * Gc) * p.q_hs + j * (D / 4) + x * 16 + k * 8)
                                            : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  if (plain) {
    fetch_pages();
    if (!UP) fetch_queries(at.rb, at.rb + 1, (at.group * p.heads + head_in) * G + hc, at.group * p.heads + head_in < p.Hkv);
    fetch_scales();
  }
  for (int item = blockIdx.x; item < items; item += gridDim.x, at = next) {
    const int split = at.split, hk = at.group * p.heads + head_in, h0 = hk * G + hc, r1 = min(p.R, (at.rb + 1) * p.pack);
    const bool real = hk < p.Hkv;                  // the last block's heads may be fewer
    const bool more = item + (int)gridDim.x < items, fetch = plain && more;
    if (more) next = kv8_item(p, before, item + gridDim.x);
    for (int r = at.rb * p.pack; r < r1;) {
      Kv8Pass a;
      if (plain) {
        a = {r, r + 1, min(max(next_len, 0), p.max_keys), 0, 0};
        a.from = min(a.most, split * p.share);
        a.to = min(a.most, a.from + p.share);
      } else {
        a = kv8_pass(p, r, r1, split);
      }
      if (UP || !plain) fetch_queries(r, a.rn, h0, real);
      // head and row of this lane's rows g and g + 8 of the products
      int len[NH], head[NH], qrow[NH], least = a.most;
#pragma unroll
      for (int u = 0; u < NH; ++u) {
        const int m = u * 8 + g, i = m / Gc;
        qrow[u] = real && r + i < a.rn ? r + i : -1;
        head[u] = h0 + m - i * Gc;
        len[u] = qrow[u] < 0 ? 0 : (plain ? a.most : (a.most > 0 ? min(max(p.lens[qrow[u]], 0), a.most) : 0));
        if (qrow[u] >= 0) least = min(least, len[u]);
      }
      least = __reduce_min_sync(0xffffffffu, least);
      r = a.rn;
      // Scales of eight stages at a time: lane 4 i + n has those of the n-th eight of stage i (past the end: of the last one).
      const int* bt = p.block_tables + (long)a.seq * p.bt_stride;
      auto page_of = [&](int batch) {
        const int key = min(a.from + (batch * (32 / NE) + lane / NE) * keys + sub * KEYS + lane % NE * 8, (a.to - 1) & ~7);
        return bt[kv8_column(p, key)];
      };
      float ks = next_ks, vs = next_vs;
      int ahead = 0;
      if (a.from < a.to && real) {
        if (!plain) {
          const int pg = kv8_page(p, page_of(0));
          ks = p.ks[(long)pg * p.Hkv + hk];
          vs = p.vs[(long)pg * p.Hkv + hk];
        }
        if (a.to - a.from > 32 / NE * keys) ahead = page_of(1);
      }
      float back[NH];                              // what q was divided by, times the scale
#pragma unroll
      for (int u = 0; u < NH; ++u) {
        uint32_t top = 0;
#pragma unroll
        for (int x = 0; x < CH; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w[4] = {raw[u][x][i].x, raw[u][x][i].y, raw[u][x][i].z, raw[u][x][i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) top = max(top, max((w[k] << 16) & 0x7fffffffu, w[k] & 0x7fff0000u));
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(top >> 23) - 127, -126), 126);
        const float f = pow2f(-e);
        back[u] = pow2f(e) * p.scale_log2;
#pragma unroll
        for (int x = 0; x < CH; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w[4] = {raw[u][x][i].x, raw[u][x][i].y, raw[u][x][i].z, raw[u][x][i].w};
            uint32_t packed[4];                    // two steps of the product, their two words each
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 v = unpack_bf16(w[k]);
              packed[k] = pack_half(v.x * f, v.y * f);
            }
            st_shared_v4(my_q + ((u * CH + x) * 2 + i) * 512, make_uint4(packed[0], packed[1], packed[2], packed[3]));
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

      __syncwarp();
      float fks = 1.f, evs = 0.f, ks2 = 1.f, vs2 = 1.f;
      int i_stage = 0;
#pragma unroll 1
      for (int k0 = a.from; k0 < a.to; k0 += keys, ++c, ++i_stage) {
        if (i_stage % (32 / NE) == 0 && i_stage) {
          ks = ks2;
          vs = vs2;
        }
        if (i_stage % (32 / NE) == 2 && real && k0 + (32 / NE - 2) * keys < a.to) {
          const int pg = kv8_page(p, ahead);
          ks2 = p.ks[(long)pg * p.Hkv + hk];
          vs2 = p.vs[(long)pg * p.Hkv + hk];
          ahead = page_of(i_stage / (32 / NE) + 2);
        }
        if (fetch && i_stage == 1) fetch_pages();
        if (fetch && i_stage == 5) fetch_scales();
        if (i_stage % (32 / NE) == 0) {
          fks = pow2f(scale_exp(ks));
          evs = (float)scale_exp(vs);
        }
        const int s = c % STAGES, key = k0 + sub * KEYS;
        if (!mbar_wait(full + 8 * s, (c / STAGES) & 1, &s_abort, p.status, ERR_WAIT_FULL)) break;      // and on to the barriers below, which others wait at
        if (key < a.to && real) {
          const uint32_t at = base + s * 2 * half;
          float sc[NE][4] = {};
#pragma unroll
          for (int x = 0; x < CH; ++x) {
            uint4 kr[NE];
#pragma unroll
            for (int n = 0; n < NE; ++n) kr[n] = shared4(at + eight[n] + k_at[x]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 lo = shared4(my_q + (x * 2 + i) * 512), hi = UP ? shared4(my_q + (((NH - 1) * CH + x) * 2 + i) * 512) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
              for (int n = 0; n < NE; ++n) {
                mma_f16_16x8(sc[n], lo.x, hi.x, lo.y, hi.y, halves_of(i ? kr[n].z : kr[n].x), halves_of_hi(i ? kr[n].z : kr[n].x));
                mma_f16_16x8(sc[n], lo.z, hi.z, lo.w, hi.w, halves_of(i ? kr[n].w : kr[n].y), halves_of_hi(i ? kr[n].w : kr[n].y));
              }
            }
          }
          const bool ends = key + KEYS > least; // keys that some row does not see
          uint32_t pw[NH][NE];
          const int from_lane = i_stage % (32 / NE) * NE;
          float fk[NE], ev[NE];
#pragma unroll
          for (int n = 0; n < NE; ++n) {
            fk[n] = __shfl_sync(0xffffffffu, fks, from_lane + n);
            ev[n] = __shfl_sync(0xffffffffu, evs, from_lane + n);
          }
#pragma unroll
          for (int u = 0; u < NH; ++u) {
            float y[NE][2], mx = -INFINITY, mxv = -INFINITY;
#pragma unroll
            for (int n = 0; n < NE; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) y[n][e] = sc[n][2 * u + e] * (fk[n] * back[u]);
            if (ends)
#pragma unroll
              for (int n = 0; n < NE; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (key + n * 8 + 2 * j + e >= len[u]) y[n][e] = -INFINITY;
#pragma unroll
            for (int n = 0; n < NE; ++n) {
              const float m0 = fmaxf(y[n][0], y[n][1]);
              mx = fmaxf(mx, m0);
              mxv = fmaxf(mxv, m0 + ev[n]);
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 2));
            // The maxima are those of some tile before, as long as none since is more than 2^K8_SLACK larger: sums are seldom scaled.  A row moves by its own scores alone, so that
            // its weights are rounded the same whatever rows are beside it; the others' sums are multiplied by one.
            const bool moves = mx > m[u] + K8_SLACK || mxv > mv[u] + K8_SLACK;
            if (__any_sync(0xffffffffu, moves)) {
              const float was = m[u], was_v = mv[u];
              m[u] = moves ? fmaxf(was, mx) : was;
              mv[u] = moves ? fmaxf(was_v, mxv) : was_v;
              l[u] *= ex2_approx(was - (m[u] == -INFINITY ? 0.f : m[u]));          // only scores of -inf so far: all weights are zero
              const float beta = ex2_approx(was_v - (mv[u] == -INFINITY ? 0.f : mv[u]));
              const float b0 = __shfl_sync(0xffffffffu, beta, 8 * j), b1 = __shfl_sync(0xffffffffu, beta, 8 * j + 4);   // rows 2 j, 2 j + 1
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                acc[u][i][0] *= b0; acc[u][i][1] *= b1;
                acc[u][i][2] *= b0; acc[u][i][3] *= b1;
              }
            }
            const float top = m[u] == -INFINITY ? 0.f : m[u], lift = K8_LIFT - (mv[u] == -INFINITY ? 0.f : mv[u]);
#pragma unroll
            for (int n = 0; n < NE; ++n) {
              l[u] += ex2_approx(y[n][0] - top) + ex2_approx(y[n][1] - top);
              pw[u][n] = pack_half(ex2_approx(y[n][0] + (ev[n] + lift)), ex2_approx(y[n][1] + (ev[n] + lift)));
            }
          }
          // channel pair (2 i, 2 i + 1) of a lane's D / 8: rows g and g + 8 of tile i
#pragma unroll
          for (int h = 0; h < NE / 2; ++h) {       // sixteen keys at a time
            uint4 vr[4];                           // D = 64: x and y
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t from = at + half + eight[2 * h + (i >> 1)] + v_at[i & 1];
              if (D == 128) {
                vr[i] = shared4(from);
              } else {
                const uint2 x = shared2(from);
                vr[i].x = x.x;
                vr[i].y = x.y;
              }
            }
            if (ends)                              // values behind the end are nobody's: what they hold may not be a number
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key + h * 16 + (i >> 1) * 8 + 2 * j + (i & 1) >= a.to) vr[i] = make_uint4(0u, 0u, 0u, 0u);
            // Nor is what some rows do not see theirs: a product apart counts what is not a number for those that do.  (Code that others do not need would cost them
            // registers: 64 on 4 heads 85 -> 91 us.)
            if (MANY && ends && least < a.to) {
              auto odd_of = [](uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); };
              uint32_t odd = 0;
#pragma unroll
              for (int i = 0; i < 4; ++i) odd |= odd_of(vr[i].x) | odd_of(vr[i].y) | (D == 128 ? odd_of(vr[i].z) | odd_of(vr[i].w) : 0u);
              if (__any_sync(0xffffffffu, odd)) {
                uint4 one[4];                      // codes of 1
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  one[i] = make_uint4(odd_of(vr[i].x), odd_of(vr[i].y), D == 128 ? odd_of(vr[i].z) : 0u, D == 128 ? odd_of(vr[i].w) : 0u);
                  vr[i] = make_uint4(vr[i].x & ~one[i].x, vr[i].y & ~one[i].y, vr[i].z & ~one[i].z, vr[i].w & ~one[i].w);
                  one[i] = make_uint4(one[i].x & 0x38383838u, one[i].y & 0x38383838u, one[i].z & 0x38383838u, one[i].w & 0x38383838u);
                }
#pragma unroll
                for (int u = 0; u < NH; ++u) {
                  uint32_t sees[2];
#pragma unroll
                  for (int n = 0; n < 2; ++n) {
                    const int at = key + (2 * h + n) * 8 + 2 * j;
                    sees[n] = pack_half(at < len[u] ? 1.f : 0.f, at + 1 < len[u] ? 1.f : 0.f);
                  }
#pragma unroll
                  for (int w = 0; w < MT / 2; ++w) {
                    auto word = [&](const uint4& x) { return w == 0 ? x.x : (w == 1 ? x.y : (w == 2 ? x.z : x.w)); };
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                      const uint32_t x = __byte_perm(word(one[0]), word(one[1]), i ? 0x7362 : 0x5140), y = __byte_perm(word(one[2]), word(one[3]), i ? 0x7362 : 0x5140);
                      float n[4] = {};
                      mma_f16_16x8(n, halves_of(x), halves_of_hi(x), halves_of(y), halves_of_hi(y), sees[0], sees[1]);
#pragma unroll
                      for (int k = 0; k < 4; ++k)
                        if (n[k] != 0.f) acc[u][2 * w + i][k] = NAN;
                    }
                  }
                }
              }
            }
#pragma unroll
            for (int w = 0; w < MT / 2; ++w) {
              auto word = [&](const uint4& x) { return w == 0 ? x.x : (w == 1 ? x.y : (w == 2 ? x.z : x.w)); };
              const uint32_t v0 = word(vr[0]), v1 = word(vr[1]), v2 = word(vr[2]), v3 = word(vr[3]);
#pragma unroll
              for (int i = 0; i < 2; ++i) {        // channels 4 w + 2 i, + 1
                const uint32_t x = __byte_perm(v0, v1, i ? 0x7362 : 0x5140), y = __byte_perm(v2, v3, i ? 0x7362 : 0x5140);
                const uint32_t a0 = halves_of(x), a1 = halves_of_hi(x), a2 = halves_of(y), a3 = halves_of_hi(y);
#pragma unroll
                for (int u = 0; u < NH; ++u) mma_f16_16x8(acc[u][2 * w + i], a0, a1, a2, a3, pw[u][2 * h], pw[u][2 * h + 1]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * s);
      }

      if (fetch) {
        if (i_stage < 2) fetch_pages();
        const int hn = next.group * p.heads + head_in;
        if (!UP) fetch_queries(next.rb, next.rb + 1, hn * G + hc, hn < p.Hkv);        // sixteen rows have no registers for it
        if (i_stage < 6) fetch_scales();
      }
      float lse[NH];
      bool none[NH];
#pragma unroll
      for (int u = 0; u < NH; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        // O / l = acc 2^-14 / l 2^(m' - m), the two factors apart because their product may be too small for a float; a row without keys: zeros
        none[u] = l[u] == 0.f;
        lse[u] = none[u] ? -INFINITY : m[u] + log2f(l[u]);
        const float inv = none[u] ? 0.f : 0x1p-14f / l[u], level = none[u] ? 0.f : ex2_approx(mv[u] - m[u]);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {           // rows 2 j, 2 j + 1 of the products
          const int src = 8 * j + 4 * hh;
          const float f = __shfl_sync(0xffffffffu, inv, src), f2 = __shfl_sync(0xffffffffu, level, src);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            acc[u][i][hh] = acc[u][i][hh] * f * f2;
            acc[u][i][2 + hh] = acc[u][i][2 + hh] * f * f2;
          }
        }
      }
      // The sums of the warps of a head become one, two by two, through the memory of the giver's queries, which it needs no longer, in halves of its channels.  A lane
      // of either warp holds the same rows and channels.
      for (int step = 1; step < p.subs; step *= 2) {
        const int role = sub & (2 * step - 1);     // 0 takes, `step` gives
        float w0[NH][2], w1[NH][2];
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          if (role == step) {
#pragma unroll
            for (int u = 0; u < NH; ++u) {
              if (side == 0 && j == 0) sums[warp][u * 8 + g] = lse[u];
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int i = 0; i < MT / 2; i += 2) {
                  const int f = side * (MT / 2) + i;
                  st_shared_v4(my_q + ((u * 2 + hh) * (MT / 4) + i / 2) * 512,
                               make_uint4(__float_as_uint(acc[u][f][hh]), __float_as_uint(acc[u][f][2 + hh]), __float_as_uint(acc[u][f + 1][hh]), __float_as_uint(acc[u][f + 1][2 + hh])));
                }
            }
          }
          asm volatile("bar.sync %0, %1;" ::"r"(1 + vh), "r"(32 * p.subs) : "memory");
          if (role == 0) {
            const uint32_t from = my_q + step * VH * (NH * CH * 1024);
#pragma unroll
            for (int u = 0; u < NH; ++u) {
              if (side == 0) {
                const float other = sums[warp + step * VH][u * 8 + g], top = fmaxf(lse[u], other), at = top == -INFINITY ? 0.f : top;
                const float a0 = ex2_approx(lse[u] - at), a1 = ex2_approx(other - at), den = a0 + a1, inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                  w0[u][hh] = __shfl_sync(0xffffffffu, a0 * inv, 8 * j + 4 * hh);
                  w1[u][hh] = __shfl_sync(0xffffffffu, a1 * inv, 8 * j + 4 * hh);
                }
                none[u] = den == 0.f;
                lse[u] = none[u] ? -INFINITY : at + log2f(den);
              }
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int i = 0; i < MT / 2; i += 2) {
                  const int f = side * (MT / 2) + i;
                  const uint4 x = shared4(from + ((u * 2 + hh) * (MT / 4) + i / 2) * 512);
                  acc[u][f][hh] = acc[u][f][hh] * w0[u][hh] + __uint_as_float(x.x) * w1[u][hh];
                  acc[u][f][2 + hh] = acc[u][f][2 + hh] * w0[u][hh] + __uint_as_float(x.y) * w1[u][hh];
                  acc[u][f + 1][hh] = acc[u][f + 1][hh] * w0[u][hh] + __uint_as_float(x.z) * w1[u][hh];
                  acc[u][f + 1][2 + hh] = acc[u][f + 1][2 + hh] * w0[u][hh] + __uint_as_float(x.w) * w1[u][hh];
                }
            }
          }
          asm volatile("bar.sync %0, %1;" ::"r"(1 + vh), "r"(32 * p.subs) : "memory");
        }
      }
      if (sub) continue;
      const int parts = p.splits, part = split;
#pragma unroll
      for (int u = 0; u < NH; ++u) {
        if (parts > 1 && j == 0 && qrow[u] >= 0) p.part_lse[((long)qrow[u] * p.H + head[u]) * parts + part] = lse[u];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int src = 8 * j + 4 * hh;
          const int qr = __shfl_sync(0xffffffffu, qrow[u], src), hd = __shfl_sync(0xffffffffu, head[u], src);
          const bool no = __shfl_sync(0xffffffffu, none[u], src);
          if (qr < 0 || (parts > 1 && no)) continue;
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
}

// out[row, head] = sum_s 2^(lse_s - top) o_s / sum_s 2^(lse_s - top) over the shares (at most 256): a block per (row, head), its sixteen warps take every sixteenth share.
template <int D>
__global__ void __launch_bounds__(512)
kv8_merge_kernel(const float* part_o, const float* part_lse, const int* lens, int pack, int R, int max_keys, int share, int splits, int H, __nv_bfloat16* out, long o_rs, long o_hs) {
  pdl_begin();
  constexpr int PER = D / 32, WARPS = 16;
  __shared__ float sums[WARPS][D];
  const long r = blockIdx.x;
  const int parts = kv8_count(lens, (int)(r / H) / pack, pack, R, max_keys, share);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // every warp: the weights of all shares
  float w[K8_MAX_PARTS / 32], top = -INFINITY, den = 0.f;
#pragma unroll
  for (int i = 0; i < K8_MAX_PARTS / 32; ++i) {
    w[i] = lane + i * 32 < parts ? part_lse[r * splits + lane + i * 32] : -INFINITY;
    top = fmaxf(top, w[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
  for (int i = 0; i < K8_MAX_PARTS / 32; ++i) {
    w[i] = w[i] == -INFINITY ? -1.f : ex2_approx(w[i] - top);             // below zero: a share without keys, which has written no sum
    den += w[i] < 0.f ? 0.f : w[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  float acc[PER] = {};
  const float* po = part_o + r * splits * D + lane * PER;
#pragma unroll
  for (int i = 0; i < K8_MAX_PARTS / 32; ++i) {
    if (i * 32 >= parts) break;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int s = i * 32 + h * WARPS + warp;
      const float ws = __shfl_sync(0xffffffffu, w[i], h * WARPS + warp);
      if (!(ws < 0.f)) {
        float x[PER];
        if (PER == 4) {
          const float4 y = *reinterpret_cast<const float4*>(po + (long)s * D);
          x[0] = y.x; x[1] = y.y; x[PER - 2] = y.z; x[PER - 1] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(po + (long)s * D);
          x[0] = y.x; x[1] = y.y;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) acc[k] = fmaf(x[k], ws, acc[k]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) sums[warp][lane * PER + i] = acc[i];
  __syncthreads();
  const float f = den != 0.f ? 1.0f / den : 0.f;   // not a number stays one
  const long row = r / H, head = r - row * H;
  for (int c = threadIdx.x * 2; c < D; c += 1024) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      x += sums[i][c];
      y += sums[i][c + 1];
    }
    *reinterpret_cast<uint32_t*>(out + row * o_rs + head * o_hs + c) = pack_bf16(x * f, y * f);
  }
}

// The same for many rows of up to 32 shares, a warp per (row, head): 256 rows of 32 heads and three shares 102 us in all in place of 140; 256 heads of 22 shares 23 in place of 17.
template <int D>
__global__ void __launch_bounds__(128)
kv8_merge_few_kernel(const float* part_o, const float* part_lse, const int* lens, int pack, int R, int max_keys, int share, int splits, int H, __nv_bfloat16* out, long o_rs, long o_hs) {
  pdl_begin();
  constexpr int PER = D / 32;
  const long r = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= (long)R * H) return;
  const long row = r / H, head = r - row * H;
  const int parts = kv8_count(lens, (int)row / pack, pack, R, max_keys, share);
  float w = lane < parts ? part_lse[r * splits + lane] : -INFINITY, top = w;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  w = w == -INFINITY ? -1.f : ex2_approx(w - top);                         // below zero: a share without keys, which has written no sum
  float den = w < 0.f ? 0.f : w, acc[PER] = {};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  const float* po = part_o + r * splits * D + lane * PER;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float ws = __shfl_sync(0xffffffffu, w, s);
    if (!(ws < 0.f)) {
      float x[PER];
      if (PER == 4) {
        const float4 y = *reinterpret_cast<const float4*>(po + (long)s * D);
        x[0] = y.x; x[1] = y.y; x[PER - 2] = y.z; x[PER - 1] = y.w;
      } else {
        const float2 y = *reinterpret_cast<const float2*>(po + (long)s * D);
        x[0] = y.x; x[1] = y.y;
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) acc[k] = fmaf(x[k], ws, acc[k]);
    }
  }
  const float f = den != 0.f ? 1.0f / den : 0.f;   // not a number stays one
  uint32_t* o = reinterpret_cast<uint32_t*>(out + row * o_rs + head * o_hs + lane * PER);
#pragma unroll
  for (int k = 0; k < PER / 2; ++k) o[k] = pack_bf16(acc[2 * k] * f, acc[2 * k + 1] * f);
}

// How a call is dealt out.  Rows that share a block: as many as fill the products' sixteen rows, where rows share sequences at all.  A row's keys are cut into shares of the same
// number of keys, so that about as many shares as SMs, or a small multiple, follow from the rows, the heads and the tables' width, never from lengths: a row's result is the same
// whatever its neighbours hold.
struct Kv8Deal {
  int pack, chunks, heads, groups, subs, unit, share, splits, grid;
  bool up;
};
// `splits`: the number of shares as it was worked out before for the same sizes (0: it is now, which takes as long as a launch does).
static bool kv8_deal(int R, int S, int H, int Hkv, int D, bool mapped, int page, int max_keys, int splits, Kv8Deal& d) {
  const int G = H / Hkv;
  if (G > K8_MAX_GROUP) return false;
  d.pack = mapped && R > S && G <= 8 ? 16 / G : 1;
  d.chunks = (G + 15) / 16;
  d.up = (d.chunks > 1 ? 16 : G) * d.pack > 8;
  if (splits < 0 || splits > K8_MAX_PARTS) return false;
  const int warps = K8_WARPS, sms = sm_count(), fewest = (Hkv + warps / d.chunks - 1) / (warps / d.chunks);
  const long row_blocks = (R + d.pack - 1) / d.pack;
  // The heads of a block and the number of shares.  Few rows: rounds of blocks times the stages of a share and what it costs beside them (its queries and the way of its sums, some
  // two stages' time), and as much once more where shares are joined.  Many: blocks take the shares there are in turn; a row is taken to have four fifths of the table's keys.
  // Blocks of fewer heads, whose warps share the keys of one, are for calls that leave SMs without a block: a copy brings fewer bytes there.  32 heads on 8 of 128, 112 keys: 5.9 us
  // by a head a block, 7.9 by four shares of all heads; 640 keys 9.6 and, of 20 shares, 8.5, with a launch more; one of 131071 keys, 64 heads, 51 in 37 shares, 53 in 147.
  double best = 1e30;
  d.splits = 0;
  for (int heads = (Hkv + fewest - 1) / fewest;; heads = (heads + 1) / 2) {
    Kv8Deal t = d;
    t.heads = heads;
    t.groups = (Hkv + heads - 1) / heads;
    t.subs = 1;
    while (t.subs * 2 * t.heads * t.chunks <= warps) t.subs *= 2;
    const int keys = t.subs * k8_keys(D, t.up), stages = (max_keys + keys - 1) / keys;       // at most 256: 32 copies of eight rows
    t.unit = page % 32 == 0 && keys % 32 == 0 ? 32 : (page % 16 == 0 ? 16 : 8);
    const long blocks = row_blocks * t.groups;
    for (int n = splits ? splits : 1; n <= (splits ? splits : K8_MAX_PARTS) && n <= stages; ++n) {
      if (t.groups > fewest && blocks * n > sms) break;
      const int share = (stages + n - 1) / n * keys;
      if ((max_keys + share - 1) / share != n) continue;
      const double items = R > d.pack ? blocks * (0.8 * max_keys / share + 0.5) : (double)blocks * n, rounds = (double)((long)(items / sms) + 1);
      const double cost = (items == (rounds - 1.0) * sms ? rounds - 1.0 : rounds) * (share / keys + 2) + (n > 1 ? 2 + 0.008 * n : 0.0);
      if (cost < best) {
        best = cost;
        t.splits = n;
        t.share = share;
        d = t;
      }
    }
    if (heads == 1) break;
  }
  if (d.splits < 1) return false;
  const long blocks = row_blocks * d.groups;
  if (blocks * d.splits > 0x7fffffffL) return false;
  d.grid = blocks * d.splits < sms ? (int)(blocks * d.splits) : sms;
  return true;
}

// Codes as {channels, slots, heads}, boxes of `unit` slots and `heads` heads
static int kv8_tmap(CUtensorMap* out, const void* ptr, long slots, int Hkv, int D, int unit, int heads) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return RC_NO_DRIVER;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)slots, (cuuint64_t)Hkv}, strides[2] = {(cuuint64_t)Hkv * D, (cuuint64_t)D};
  const cuuint32_t box[3] = {(cuuint32_t)D, (cuuint32_t)unit, (cuuint32_t)heads}, each[3] = {1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(ptr), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? RC_OK : RC_TMAP;
}

}  // namespace omni

using namespace omni;

static int shift_of(int page) { return page & (page - 1) ? -1 : __builtin_ctz((unsigned)page); }       // log2, -1 if it has none
static bool misaligned(const void* a, const void* b, const void* c, const void* d) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15;
}

// A cache as the entry points take it: pages uint8 [pages, page, Hkv, D], scales fp32 [pages, Hkv]; set up once by who owns it.
struct Kv8Cache {
  void *kc, *vc;
  float *ks, *vs;
  int* status;
  int pages, page, Hkv, D;
};
static bool bad_cache(const Kv8Cache& c) {
  return c.Hkv < 1 || (c.D != 64 && c.D != 128) || c.page < 8 || (c.page & 7) || c.pages < 1 || (long)c.pages * c.page > 0x7fffffffL || misaligned(c.kc, c.vc, c.kc, c.vc);
}

// k, v bf16 [T, Hkv, D] at the given pitches (multiples of 8); slots int32 [T], below zero: not written.  The rows of a page follow one another, with fewer
// than 128 others that are not written between two of them.
extern "C" int omni_kv8_write(const Kv8Cache* cache, const void* k, const void* v, long k_rs, long k_hs, long v_rs, long v_hs, const int* slots, int T, void* stream) {
  if (T <= 0) return RC_OK;
  const Kv8Cache& c = *cache;
  if (bad_cache(c) || ((k_rs | k_hs | v_rs | v_hs) & 7) || misaligned(k, v, k, v)) return RC_BAD_ARG;
  // rows per block: 64, or fewer where that leaves SMs without blocks
  int chunk = 64;
  while (chunk > 4 && (long)((T + chunk - 1) / chunk) * c.Hkv < 4L * sm_count()) chunk /= 2;
  const Kv8Write p = {(const __nv_bfloat16*)k, (const __nv_bfloat16*)v, k_rs, k_hs, v_rs, v_hs, (unsigned char*)c.kc, (unsigned char*)c.vc, c.ks, c.vs, slots,
                      (long)c.pages * c.page, T, c.Hkv, c.page, chunk, c.status};
  const long grid = (long)((T + chunk - 1) / chunk) * c.Hkv;              // a chunk's heads side by side: their rows are
  if (grid > 0x7fffffffL) return RC_TOO_LARGE;
  launch_overlapped(c.D == 64 ? kv8_write_kernel<64> : kv8_write_kernel<128>, dim3((unsigned)grid), 256, 0, (cudaStream_t)stream, p);
  return (int)cudaGetLastError();
}

// n lists: index[i] int32 slots of rows[i] rows (tables = 0; below zero: zeros), or a block table of rows[i] tokens, to rows row0[i] .. of k, v bf16 [.., Hkv, D].
extern "C" int omni_kv8_read(const Kv8Cache* cache, int n, const void* const* index, const long* row0, const long* rows, int tables, void* k, void* v, void* stream) {
  const Kv8Cache& c = *cache;
  if (bad_cache(c) || misaligned(k, v, k, v)) return RC_BAD_ARG;
  for (int i0 = 0; i0 < n; i0 += K8_TABLES) {
    const int m = n - i0 < K8_TABLES ? n - i0 : K8_TABLES;
    Kv8Read p = {};
    p.kc = (const unsigned char*)c.kc; p.vc = (const unsigned char*)c.vc; p.ks = c.ks; p.vs = c.vs; p.k = (__nv_bfloat16*)k; p.v = (__nv_bfloat16*)v;
    p.n_slots = (long)c.pages * c.page; p.Hkv = c.Hkv; p.D = c.D; p.page = c.page; p.shift = shift_of(c.page); p.tables = tables; p.status = c.status;
    long most = 0;
    for (int i = 0; i < m; ++i) {
      p.index[i] = (const int*)index[i0 + i];
      p.row0[i] = row0[i0 + i];
      p.rows[i] = (int)rows[i0 + i];
      if (rows[i0 + i] > 0x7fffffffL - 65536) return RC_TOO_LARGE;
      if (rows[i0 + i] > most) most = rows[i0 + i];
    }
    if (most <= 0) continue;
    const int vecs = c.Hkv * c.D / 8, lines = 4 * (vecs < 256 ? 256 / vecs : 1);          // rows a block takes at once
    long blocks = (most + lines - 1) / lines;
    if (blocks > 16L * sm_count()) blocks = 16L * sm_count();
    launch_overlapped(kv8_read_kernel, dim3((unsigned)blocks, (unsigned)m), 256, 0, (cudaStream_t)stream, p);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
  }
  return RC_OK;
}

// Shares per (row, head) that omni_kv8_attn will write: sizes its scratch (fp32, shares x D and shares x 1); -1: sizes that it does not take.
extern "C" int omni_kv8_attn_shares(int R, int S, int H, int Hkv, int D, int mapped, int page, int max_keys) {
  Kv8Deal d;
  if (R < 1 || Hkv < 1 || H < Hkv || page < 8 || max_keys < 1 || !kv8_deal(R, S, H, Hkv, D, mapped != 0, page, max_keys, 0, d)) return -1;
  return d.splits;
}

template <int D, bool UP, bool MANY>
static int launch_kv8_attn(const Kv8Attn& p, int grid, cudaStream_t st) {
  static unsigned long long ready = 0;
  constexpr int warps = K8_WARPS, ring = 96 * 2 * warps * D, q = warps * (UP ? 2 : 1) * D * 16;       // a stage; queries
  if (int e = ensure_dynamic_smem((const void*)kv8_attn_kernel<D, UP, MANY>, ring + q, ready)) return e;
  launch_overlapped(kv8_attn_kernel<D, UP, MANY>, grid, 32 * (warps + 1), ring + q, st, p);
  return (int)cudaGetLastError();
}

// q, out bf16 [R, H, D] at the given pitches (multiples of 8); block_tables int32 [S, max_keys / page] at bt_stride; lens int32 [R]: keys that a row sees;
// row_seq int32 [R] or null (R = S).  `part`: fp32 [R, H, shares, D + 1] where there are several shares.
extern "C" int omni_kv8_attn(const Kv8Cache* cache, const void* q, long q_rs, long q_hs, const int* block_tables, long bt_stride, const int* lens, const int* row_seq,
                             int R, int S, int H, int max_keys, float scale, int shares, float* part, void* out, long o_rs, long o_hs, void* stream) {
  if (R <= 0) return RC_OK;
  const Kv8Cache& c = *cache;
  const int Hkv = c.Hkv, D = c.D, page = c.page;
  if (bad_cache(c) || H < 1 || H % Hkv || max_keys < 1 || (!row_seq && R != S) || ((q_rs | q_hs | o_rs | o_hs) & 7) || misaligned(q, out, q, out) || shares < 1 ||
      (shares > 1 && !part))
    return RC_BAD_ARG;
  Kv8Deal d;
  if (!kv8_deal(R, S, H, Hkv, D, row_seq != nullptr, page, max_keys, shares, d)) return RC_TOO_LARGE;
  float* part_lse = part + (long)R * H * shares * D;
  Kv8Attn p = {};
  if (int e = kv8_tmap(&p.mk, c.kc, (long)c.pages * page, Hkv, D, d.unit, d.heads)) return e;
  if (int e = kv8_tmap(&p.mv, c.vc, (long)c.pages * page, Hkv, D, d.unit, d.heads)) return e;
  p.q = (const __nv_bfloat16*)q; p.q_rs = q_rs; p.q_hs = q_hs; p.ks = c.ks; p.vs = c.vs; p.block_tables = block_tables; p.lens = lens; p.row_seq = row_seq;
  p.bt_stride = bt_stride; p.page = page; p.shift = shift_of(page); p.pages = c.pages; p.max_keys = max_keys; p.R = R; p.S = S; p.H = H;
  p.Hkv = Hkv; p.chunks = d.chunks; p.heads = d.heads; p.groups = d.groups; p.pack = d.pack; p.unit = d.unit; p.subs = d.subs; p.share = d.share; p.splits = d.splits;
  p.row_blocks = (R + d.pack - 1) / d.pack; p.listed = d.splits > 1 && p.row_blocks <= K8_LISTED && (long)p.row_blocks * d.groups * d.splits > d.grid;
  p.scale_log2 = scale * 1.4426950408889634f; p.part_o = part; p.part_lse = part_lse; p.out = (__nv_bfloat16*)out; p.o_rs = o_rs; p.o_hs = o_hs; p.status = c.status;
  cudaStream_t st = (cudaStream_t)stream;
  const auto launch = d.pack > 1 ? (D == 64 ? launch_kv8_attn<64, true, true> : launch_kv8_attn<128, true, true>)      // 16 / G rows of G heads: more than 8
                      : d.up     ? (D == 64 ? launch_kv8_attn<64, true, false> : launch_kv8_attn<128, true, false>)
                                 : (D == 64 ? launch_kv8_attn<64, false, false> : launch_kv8_attn<128, false, false>);
  if (int e = launch(p, d.grid, st))
    return e;
  if (shares == 1) return RC_OK;
  const bool few = d.splits <= 32 && (long)R * H >= 1024;
  launch_overlapped(few ? (D == 64 ? kv8_merge_few_kernel<64> : kv8_merge_few_kernel<128>) : (D == 64 ? kv8_merge_kernel<64> : kv8_merge_kernel<128>),
                    (unsigned)(few ? ((long)R * H + 3) / 4 : (long)R * H), few ? 128 : 512, 0, st, part, part_lse, lens, d.pack, R,
                    max_keys, d.share, d.splits, H, (__nv_bfloat16*)out, o_rs, o_hs);
  return (int)cudaGetLastError();
}
