// Tokens drawn from given random numbers: temperature, top-k, min-p and top-p over rows of logits.  All that decides the token is whole
// numbers; its log probability has the row's sum of weights in fp32, but for rows whose mass is summed in whole numbers for the token (no cut; top-p alone).
//
// For a row x with maximum m and temperature T, weights are whole numbers w_i = round(2^44 exp((x_i - m) / T)), so that sums of them have no order: blocks,
// threads and lists may add them as they come, and the plain definition in 64 bits gives the same token (a weight is within 2^-50 of itself before it is rounded).  The order of a row is (x down, index up).  A cut is the
// last element of that order that stays:
//   top-k   the k-th element;
//   min-p   elements whose weight is below min_p of the largest have no mass (they are the end of the order);
//   top-p   of what is left, with mass S, the last element before which less than top_p S lies.
// The token is the first kept index in the vocabulary's order at which the running mass passes u times the kept mass.
//
// A cluster of blocks owns a row, each a run of tiles of 4096 elements, a warp 256 neighbours of a tile; the row is read from HBM once and from L2 after that.
//   1  Largest element and fp32 sum of weights of every warp's piece.  They give the row's maximum and the sum for the log probability, and bounds that keep most
//      of the row out of what follows: at least k elements reach the k-th largest of the pieces' maxima; an element below (1 - top_p) / V of the whole mass lies behind
//      top-p's cut, since all such elements together are no more than what top-p drops.  Pieces whose maximum is below the bound are not read again.
//   2  top-k: what reaches the bound is a list.  top-p: a histogram of it, 2048 bins of (m - x) / T, 1/64 wide, with what a bin's mass needs beside its count (the sum of
//      positions in the bin: a chord through exp is off by at most 2^-15).
//   3  top-p: 64-bit weights of what is surely kept, as sums per piece, a list of the few bins that the cut can lie in, and 64-bit weights of what lies behind them: the border at
//      top_p S is compared with masses that differ by one element's, in flat rows a few millionths of S, and a sum in fp32 may be off by as much (2^-19 for
//      a sum of such depth).  Without a cut: 64-bit weights of every element once.
// The first block then sorts the list, finds the cut exactly, the tile that the random number falls into and the element in it.  Rows whose lists would be longer
// (thousands of equal logits) take histograms over keys, in the end over the indexes of ties, in the first block alone.
//
// Bound by instructions: of the 78 MB of 256 bf16 rows of 152064 a pass takes 12 us from memory; the largest alone takes 34 us, no cut 101 (13 fp64 instructions an element), k 50 58, p 0.9
// 206 (two more passes of some 35 instructions an element, 13 fp64 ones among those of the last; with S in fp32 it took 176).  One row: 5.6 us, 13, 12, 31: steps one after another
// in one cluster.
#include <cfloat>
#include <cuda_bf16.h>

#include "host_util.h"
#include "ptx_sm100.cuh"

namespace omni {

typedef unsigned long long u64;
constexpr int SG_THREADS = 512, SG_WARPS = SG_THREADS / 32, SG_TILE = SG_THREADS * 8, SG_PIECE = 256, SG_BINS = 2048, SG_LIST = 2048, SG_MAX_V = 262144;
constexpr int SG_MAX_CLUSTER = 8, SG_FEW = 128;         // lists up to SG_FEW are ranked by counting: k 100 16 us (19.5 sorted), k 200 25 (20.5 sorted)
constexpr int SG_TILES = SG_MAX_V / SG_TILE + 1;        // a row that does not begin on 16 bytes may reach into one tile more
constexpr int SG_PIECES = SG_TILES * SG_WARPS;
constexpr int SG_EACH = SG_LIST / SG_THREADS, SG_PER = SG_BINS / SG_THREADS, SG_PER_PIECE = (SG_PIECES + SG_THREADS - 1) / SG_THREADS;
constexpr float SG_RANGE = 32.f;                        // beyond exp(-32) = 2^-46.2 weights are zero
constexpr double SG_ONE = 17592186044416.0;             // 2^44

struct SampleGiven {
  const void* logits;
  long ld;
  int V;
  const float *temperature, *top_p, *min_p, *u;         // null: the value beside it, for every row
  const int* top_k;
  float temperature_v, top_p_v, min_p_v;
  int top_k_v;
  int* ids;
  float* logprob;
};

// keys in the order of x: larger x, larger key
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// place in the order: larger comes first
__device__ __forceinline__ u64 word_of(float x, int index) { return (u64)key_of(x) << 32 | (uint32_t)~index; }

enum SgMode : int { SG_ALL = 0, SG_TOP = 1, SG_WINDOW = 2, SG_SLOW = 3 };

struct SgShared {
  uint32_t count[SG_BINS];
  u64 list[SG_LIST];
  union {
    u64 mass[SG_BINS];                                  // of the list's elements, or of bins
    uint32_t frac[SG_BINS];
  };
  uint32_t key[SG_LIST];
  float top[SG_PIECES], sum[SG_PIECES];                 // of every piece of the row: maximum, weights relative to it
  u64 tile[SG_PIECES];                                  // kept mass
  float queue[SG_WARPS][SG_PIECE];
  double table[64];                                     // 2^(44 + j / 64)
  u64 whole[SG_MAX_CLUSTER];
  u64 scan[SG_WARPS];
  float scan_f[SG_WARPS];
  u64 found[4];
  uint32_t n_list, base;
  int mode, lo, hi;
  float first[2];                                       // least logits in front of the window, and in it
};

template <typename T>
__device__ __forceinline__ T* at_rank(T* p, uint32_t rank) {            // the same shared variable of another block of the cluster
  u64 out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<u64>(p)), "r"(rank));
  return reinterpret_cast<T*>(out);
}
// Barrier of the cluster, for warps whose threads may have left a loop at different times; its halves.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier() {
  cluster_arrive();
  cluster_wait();
}

// Sum over the warp of values below 2^59: three additions of 22 bits each.
__device__ __forceinline__ u64 warp_sum(u64 v) {
  const u64 lo = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3fffffu), mid = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 22) & 0x3fffffu);
  return lo + (mid << 22) + ((u64)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 44)) << 44);
}
// Exclusive prefix of v over the block's threads, and the total.
template <typename N>
__device__ __noinline__ N block_prefix(N v, N& total, N* sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  N run = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const N up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();                                      // the previous use of `sh` is over
  if (lane == 31) sh[warp] = run;
  __syncthreads();
  const N mine = lane < SG_WARPS ? sh[lane] : N(0);                      // every warp adds up the others' sums by its lanes
  N all = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const N up = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += up;
  }
  total = __shfl_sync(0xffffffffu, all, 31);
  return __shfl_sync(0xffffffffu, all - mine, warp) + (run - v);
}
// Sorts a list down, n <= SG_LIST; what lies behind n up to the next power of two becomes zero.  Pairs that are at most 32 apart lie in the 64 elements of one warp, whatever the
// distance: steps between them need no barrier of the block.
__device__ __noinline__ void sort_down(u64* list, int n) {
  int m = 64;
  while (m < n) m *= 2;
  for (int i = n + threadIdx.x; i < m; i += SG_THREADS) list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= m; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      if (j > 32) __syncthreads();
      for (int t = threadIdx.x; t < m / 2; t += SG_THREADS) {
        const int a = (t & ~(j - 1)) * 2 | (t & (j - 1)), b = a | j;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & k) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      if (j > 32) __syncthreads();
      else __syncwarp();
    }
  __syncthreads();
}
// The same for n <= SG_THREADS words, one a thread: steps within a warp are shuffles.
__device__ __noinline__ void sort_down_few(u64* list, int n) {
  const int t = threadIdx.x;
  int m = 32;
  while (m < n) m *= 2;
  u64 x = t < n ? list[t] : 0;
  for (int k = 2; k <= m; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      u64 y;
      if (j >= 32) {
        __syncthreads();
        list[t] = x;
        __syncthreads();
        y = list[t ^ j];
      } else {
        y = __shfl_xor_sync(0xffffffffu, x, j);
      }
      const bool front = (t & j) == 0, down = (t & k) == 0;
      x = (front == down) == (x > y) ? x : y;
    }
  __syncthreads();
  list[t] = x;
  __syncthreads();
}
// Appends the marked ones of a thread's eight elements to the block's list.  All 32 lanes call it; one addition to the counter for them all.
__device__ __forceinline__ void append(SgShared& sh, unsigned marks, const float (&x)[8], int index0) {
  if (!__any_sync(0xffffffffu, marks)) return;
  const int lane = threadIdx.x & 31, mine = __popc(marks);
  int run = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  uint32_t to = 0;
  if (lane == 31) to = atomicAdd(&sh.n_list, (uint32_t)run);
  to = __shfl_sync(0xffffffffu, to, 31) + run - mine;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (marks >> j & 1) {
      if (to < SG_LIST) sh.list[to] = word_of(x[j] + 0.f, index0 + j);
      ++to;
    }
}
// The lists of the cluster's blocks behind the first one's.
__device__ __forceinline__ void join_lists(SgShared& sh, uint32_t rank) {
  __syncthreads();
  const uint32_t n = sh.n_list;
  if (rank == 0 || n == 0) return;
  if (threadIdx.x == 0) sh.base = atomicAdd(at_rank(&sh.n_list, 0), n);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < min(n, (uint32_t)SG_LIST); i += SG_THREADS)
    if (sh.base + i < SG_LIST) *at_rank(&sh.list[sh.base + i], 0) = sh.list[i];
}

// For n <= SG_FEW words of the list and masses beside them, by counting (no barrier, and a group of threads reads its words at once): the element of this
// thread, its rank and the mass before it.  A group of 1 to 32 neighbours works on an element; all of them get the answer.  BY_INDEX: in the order of the
// indexes, by the words' lower halves (larger first there, too).
struct SgPlace {
  int e, rank;                                          // e < 0: none
  bool first;                                           // of its group
  u64 before;
};
template <bool BY_INDEX>
__device__ __forceinline__ SgPlace place_of(const u64* list, const u64* mass, int n) {
  int group = 32;
  while (n * group > SG_THREADS) group /= 2;
  const int e = threadIdx.x / group, g = threadIdx.x & (group - 1);
  SgPlace at = {e < n ? e : -1, 0, g == 0, 0};
  const u64 me = e < n ? list[e] : 0;
  if (e < n)
#pragma unroll 4
    for (int j = g; j < n; j += group) {
      const u64 word = list[j];
      const bool ahead = BY_INDEX ? (uint32_t)word > (uint32_t)me : word > me;
      at.rank += ahead;
      at.before += ahead ? mass[j] : 0ull;
    }
  __syncwarp();
  for (int o = group / 2; o > 0; o /= 2) {
    at.rank += __shfl_xor_sync(0xffffffffu, at.rank, o);
    at.before += __shfl_xor_sync(0xffffffffu, at.before, o);
  }
  return at;
}

// What a thread needs to turn elements into bins and weights.
struct SgRow {
  float mx, to_bin, log2_t;                             // bins and powers of two per two units of x: halves of any two numbers have a difference
  double mx_d, to_64, inv_t, least;                     // 64ths of powers of two per unit; min_p 2^44
  const double* table;
  __device__ __forceinline__ float place(float x) const { return __fmul_rn(__fmaf_rn(x, -0.5f, 0.5f * mx), to_bin); }       // in bins behind the largest, which is finite; monotone
  // 2^44 exp((x - m) / T) before it is rounded, within some 2^-50 of itself; 0 beyond the range.  2^(y / 64) = 2^(n / 64) e^(r ln 2 / 64), n the whole number next to y, |r| <= 1/2:
  // 2^(j / 64) from a table, e^.. by its series to the fifth power (the sixth is below 2^-54), the exponent added to the table's.
  // Every copy of this has to give the same bits: no products and sums that a compiler may fuse in one place and not in another.
  __device__ __forceinline__ double weight(float x) const {
    const double y = x == mx ? 0.0 : __dmul_rn(__dsub_rn((double)x, mx_d), to_64);
    const double shifted = __dadd_rn(y, 6755399441055744.0);             // 1.5 * 2^52: the low word is n
    const int n = __double2loint(shifted);
    const double r = __dsub_rn(y, __dsub_rn(shifted, 6755399441055744.0));
    constexpr double c = 0.010830424696249145;                           // ln 2 / 64
    double p = c * c * c * c * c / 120;
    p = __fma_rn(p, r, c * c * c * c / 24);
    p = __fma_rn(p, r, c * c * c / 6);
    p = __fma_rn(p, r, c * c / 2);
    p = __fma_rn(p, r, c);
    p = __dmul_rn(p, r);
    const double t = table[n & 63];
    const double scaled = __hiloint2double(__double2hiint(t) + ((n >> 6) << 20), __double2loint(t));
    return y > -64.0 * 46.5 ? __fma_rn(scaled, p, scaled) : 0.0;
  }
  __device__ __forceinline__ static u64 rounded(double w) {             // whole numbers up to 2^51 by the same shift
    const double s = __dadd_rn(w, 6755399441055744.0);
    return (u64)__double_as_longlong(s) & 0x7ffffffffffffull;
  }
  // weight with min-p's test on the unrounded one
  __device__ __forceinline__ u64 kept(float x) const {
    const double w = weight(x);
    return w >= least ? rounded(w) : 0ull;
  }
  __device__ __noinline__ u64 kept_one(float x) const { return kept(x); }   // one copy: what runs once is bound by fetching its instructions
  __device__ __forceinline__ double scaled(float x) const { return x == mx ? 0.0 : ((double)x - mx_d) * inv_t; }
};

// Elements 8 v .. 8 v + 7 of a row whose first one lies `off` behind a 16-byte boundary, counted from the boundary.  What is not of the row and what is not a number
// becomes -inf: an element that is never drawn.
template <typename T>
struct SgVec {
  uint4 a, b;                                           // bf16: a
};
template <typename T>
__device__ __forceinline__ SgVec<T> load8(const T* row, int off, int V, int v) {
  const int i0 = v * 8 - off;
  SgVec<T> r;
  if (i0 >= 0 && i0 + 8 <= V) {
    r.a = *reinterpret_cast<const uint4*>(row + i0);
    if (sizeof(T) == 4) r.b = *reinterpret_cast<const uint4*>(row + i0 + 4);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j;
      w[j] = i >= 0 && i < V ? __float_as_uint((float)row[i]) : 0xff800000u;
    }
    if (sizeof(T) == 2) {
      r.a = make_uint4(w[0] >> 16 | w[1], w[2] >> 16 | w[3], w[4] >> 16 | w[5], w[6] >> 16 | w[7]);
    } else {
      r.a = make_uint4(w[0], w[1], w[2], w[3]);
      r.b = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  return r;
}
// as they are, not a number among them
template <typename T>
__device__ __forceinline__ void raw8(const SgVec<T>& r, float (&x)[8]) {
  const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
  if (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(a[j] << 16);
      x[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
    }
  } else {
    const uint32_t b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = __uint_as_float(a[j]);
      x[4 + j] = __uint_as_float(b[j]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void fetch8(const T* row, int off, int V, int v, float (&x)[8]) {
  raw8(load8(row, off, V, v), x);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = x[j] == x[j] ? x[j] + 0.f : -INFINITY;           // one zero: -0 + 0 = 0
}

template <typename T>
__device__ __noinline__ u64 slow_cut(const T* row, int off, int V, const SgRow& r, SgShared& sh, bool by_mass, double limit, u64 floor_word, u64& upto);

template <typename T>
__global__ void __launch_bounds__(SG_THREADS, 2)
sample_given_kernel(const __grid_constant__ SampleGiven p) {
  extern __shared__ __align__(16) unsigned char raw[];
  SgShared& sh = *reinterpret_cast<SgShared*>(raw);
  const uint32_t rank = cluster_ctarank();
  uint32_t nc;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nc));
  const int row = blockIdx.x / nc, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = p.V;
  for (int b = tid; b < SG_BINS; b += SG_THREADS) {
    sh.count[b] = 0;
    sh.frac[b] = 0;
  }
  if (tid < 64) sh.table[tid] = exp2((double)tid * (1.0 / 64)) * SG_ONE;
  if (tid == 0) sh.n_list = 0;
  cluster_arrive();                                     // this block has started: its shared memory may be written
  const T* x0 = reinterpret_cast<const T*>(p.logits) + (long)row * p.ld;
  const int off = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
  const int vecs = (V + off + 7) / 8, tiles = (vecs + SG_THREADS - 1) / SG_THREADS, per = (tiles + nc - 1) / nc, pieces = tiles * SG_WARPS;
  const int tile0 = min(tiles, (int)rank * per), tile1 = min(tiles, tile0 + per);
  pdl_begin();
  SgVec<T> ahead = load8(x0, off, V, tile0 * SG_THREADS + tid), ahead2 = load8(x0, off, V, (tile0 + 1) * SG_THREADS + tid);
  const float T_in = p.temperature ? p.temperature[row] : p.temperature_v;
  const bool greedy = !(T_in > 0.f);
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_v;
  const float min_in = p.min_p ? p.min_p[row] : p.min_p_v, min_p = min_in > 0.f ? fminf(min_in, 1.f) : 0.f;         // not a number: no cut
  const int k_in = p.top_k ? p.top_k[row] : p.top_k_v;
  const bool by_k = !greedy && k_in > 0 && k_in < V, by_p = !greedy && top_p < 1.f;
  SgRow r;
  r.inv_t = greedy ? 1.0 : 1.0 / (double)T_in;
  r.to_bin = 2.f * (float)fmin(SG_BINS / SG_RANGE * r.inv_t, 1e38);      // finite: times zero is zero
  r.log2_t = 2.f * (float)fmin(1.4426950408889634 * r.inv_t, 1e38);
  r.to_64 = 92.332482616893656 * r.inv_t;                                // 64 / ln 2
  r.least = (double)min_p * SG_ONE;
  r.table = sh.table;

  // 1.  The next tile's elements are on their way while this one's are worked on.
  const bool need_sum = greedy || by_k || by_p;
  cluster_wait();                                       // and so have the others, while the first tiles were on their way
#pragma unroll 1
  for (int t = tile0; t < tile1; ++t) {
    float x[8];
    raw8(ahead, x);
    ahead = ahead2;
    if (t + 2 < tile1) ahead2 = load8(x0, off, V, (t + 2) * SG_THREADS + tid);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);                  // passes over what is not a number
    top = of_key(__reduce_max_sync(0xffffffffu, key_of(top + 0.f)));
    float sum = 0.f;
    if (need_sum) {
      if (top < INFINITY) {
        const float base = top == -INFINITY ? 0.f : 0.5f * top;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += ex2_approx(__fmaf_rn(x[j], 0.5f, -base) * r.log2_t);
        if (sum != sum) {                                                // not a number: nothing
          sum = 0.f;
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {
            float y = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) y = i == j ? x[i] : y;
            sum += ex2_approx(fmaxf(__fmaf_rn(y, 0.5f, -base) * r.log2_t, -200.f));
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += x[j] == INFINITY ? 1.f : 0.f;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane < nc) {
      *at_rank(&sh.top[t * SG_WARPS + warp], lane) = top;
      *at_rank(&sh.sum[t * SG_WARPS + warp], lane) = sum;
    }
  }
  cluster_barrier();
  // every block: the maximum, the sum in the order of the pieces
  r.mx = -INFINITY;
  for (int i = tid; i < pieces; i += SG_THREADS) r.mx = fmaxf(r.mx, sh.top[i]);
  r.mx = of_key(__reduce_max_sync(0xffffffffu, key_of(r.mx)));
  if (lane == 0) sh.scan_f[warp] = r.mx;
  __syncthreads();
  for (int w = 0; w < SG_WARPS; ++w) r.mx = fmaxf(r.mx, sh.scan_f[w]);
  if (r.mx == -INFINITY) {
    if (rank == 0 && tid == 0) {
      p.ids[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
    }
    return;
  }
  r.mx_d = r.mx;
  double approx = 0.0;                                                   // the sum of weights over the largest
  if (need_sum) {
#pragma unroll
    for (int i = 0; i < SG_PER_PIECE; ++i) {
      const int at = tid + i * SG_THREADS;
      if (at < pieces) {
        const float d = sh.top[at] == r.mx ? 0.f : fmaxf(__fmaf_rn(sh.top[at], 0.5f, -0.5f * r.mx) * r.log2_t, -200.f);
        approx += (double)(sh.sum[at] * ex2_approx(d));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) approx += __shfl_xor_sync(0xffffffffu, approx, o);
    if (lane == 0) sh.scan[warp] = (u64)__double_as_longlong(approx);
    __syncthreads();
    approx = 0.0;
    for (int w = 0; w < SG_WARPS; ++w) approx += __longlong_as_double((long long)sh.scan[w]);
  }
  if (greedy) {
    if (rank) return;
    // the first piece with the largest element
    if (tid == 0) sh.hi = SG_PIECES;
    __syncthreads();
    for (int i = tid; i < pieces; i += SG_THREADS)
      if (sh.top[i] == r.mx) atomicMin(&sh.hi, i);
    __syncthreads();
    if (warp == 0) {
      float x[8];
      const int v = sh.hi * 32 + lane;
      fetch8(x0, off, V, v, x);
      int at = V;
#pragma unroll
      for (int j = 7; j >= 0; --j)
        if (x[j] == r.mx) at = v * 8 - off + j;
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0) {
        p.ids[row] = at;
        if (p.logprob) p.logprob[row] = (float)-log(approx);
      }
    }
    return;
  }

  // The bound: what is below it is not kept (and -inf never).  SG_ALL: no bound and no list.
  float bound = -FLT_MAX;
  int mode = SG_ALL;
  if (by_k && V > SG_LIST) {
    // the k-th largest of the pieces' maxima, rounded down to its upper 16 bits: two histograms of 256 bins
    uint32_t got = 0;
    int left = k_in;
    uint32_t* h = reinterpret_cast<uint32_t*>(sh.queue);
#pragma unroll 1
    for (int shift = 24; shift >= 16 && left > 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) h[tid] = 0;
      __syncthreads();
      for (int i = tid; i < pieces; i += SG_THREADS) {
        const uint32_t key = key_of(sh.top[i]);
        if (shift == 24 || key >> 24 == got >> 24) atomicAdd(&h[key >> shift & 255], 1u);
      }
      __syncthreads();
      // every warp: eight bins a lane, from the highest on
      int n[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] = (int)h[255 - lane * 8 - i];
        mine += n[i];
      }
      int run = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const unsigned reached = __ballot_sync(0xffffffffu, run >= left);
      if (!reached) {                                                     // fewer pieces than k
        got = 0;
        break;
      }
      const int who = __ffs(reached) - 1;
      int before = run - mine, bin = -1, ahead_of = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (bin < 0 && before + n[i] >= left) {
          bin = 255 - lane * 8 - i;
          ahead_of = before;
        }
        before += n[i];
      }
      got |= (uint32_t)__shfl_sync(0xffffffffu, bin, who) << shift;
      left -= __shfl_sync(0xffffffffu, ahead_of, who);
    }
    bound = fmaxf(bound, got ? of_key(got) : -INFINITY);
  }
  if (by_p && !by_k) {
    // in units of the largest: (1 - p) Z / V, with room for what is rounded; with min-p its own bound, which S respects
    const float share = min_p > 0.f ? min_p * (1.f - 1e-5f) : (1.f - fmaxf(top_p, 0.f)) * (float)approx / (float)V * (1.f - 1e-4f);
    const float below = log2f(share) / (0.5f * r.log2_t);
    bound = fmaxf(bound, share > 0.f ? r.mx + below - 1e-5f * (fabsf(r.mx) + fabsf(below)) : bound);
  }
  auto piece_top = [&](int t) { return sh.top[t * SG_WARPS + warp]; };
  if (by_k) {
    // 2, top-k
#pragma unroll 1
    for (int t = tile0; t < tile1; ++t) {
      if (piece_top(t) < bound) continue;
      const int v = t * SG_THREADS + tid;
      float x[8];
      raw8(load8(x0, off, V, v), x);
      unsigned marks = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) marks |= (unsigned)(x[j] >= bound) << j;                // not a number: no
      append(sh, marks, x, v * 8 - off);
    }
    join_lists(sh, rank);
    cluster_barrier();
    mode = *at_rank(&sh.n_list, 0) > SG_LIST ? SG_WINDOW : SG_TOP;        // pieces of very different sizes, or k beyond their number: the histogram
    cluster_barrier();                                                   // all have read it
    if (mode == SG_WINDOW && tid == 0) sh.n_list = 0;
  } else if (by_p) {
    mode = SG_WINDOW;
  }
  if (mode == SG_WINDOW && r.mx == INFINITY) mode = SG_SLOW;
  if (mode == SG_WINDOW) {
    // 2, histogram of what reaches the bound
#pragma unroll 1
    for (int t = tile0; t < tile1; ++t) {
      if (piece_top(t) < bound) continue;
      float x[8];
      raw8(load8(x0, off, V, t * SG_THREADS + tid), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // 2^23 and what is below it, rounded down: whole numbers in the low bits.  What is far beyond the range counts into the last bin.
        const float y = fminf(r.place(x[j]), (float)SG_BINS - 0.001f), whole = __fadd_rd(y, 8388608.f);
        const uint32_t b = __float_as_uint(whole) & (SG_BINS - 1);
        const float part = __fsub_rn(y, __fsub_rn(whole, 8388608.f));
        if (x[j] >= bound) {
          atomicAdd(&sh.count[b], 1u);
          if (by_p) atomicAdd(&sh.frac[b], __float_as_uint(__fmaf_rn(part, 8192.f, 8388608.f)) & 0x3fffu);
        }
      }
    }
    __syncthreads();
    if (rank)
      for (int b = tid; b < SG_BINS; b += SG_THREADS)
        if (const uint32_t n = sh.count[b]) {
          atomicAdd(at_rank(&sh.count[b], 0), n);
          if (by_p) atomicAdd(at_rank(&sh.frac[b], 0), sh.frac[b]);
        }
    cluster_barrier();
    if (rank == 0) {
      u64 n[SG_PER], mine = 0, all;
#pragma unroll
      for (int i = 0; i < SG_PER; ++i) {
        n[i] = sh.count[tid * SG_PER + i];
        mine += n[i];
      }
      const u64 before = block_prefix(mine, all, sh.scan);
      if (tid == 0) {
        sh.mode = SG_WINDOW;
        sh.lo = SG_BINS;
        sh.hi = 0;
      }
      __syncthreads();
      if (by_k) {
        // the bin of the k-th
        u64 b = before;
#pragma unroll
        for (int i = 0; i < SG_PER; ++i) {
          if (b < (u64)k_in && b + n[i] >= (u64)k_in) {
            sh.hi = sh.lo = tid * SG_PER + i;
            if (by_p) sh.lo = 0;                                          // the list is what top-p chooses from: all of it
            if ((by_p ? b : 0) + n[i] > SG_LIST) sh.mode = SG_SLOW;
            sh.found[0] = b;                                              // elements before the window
          }
          b += n[i];
        }
        if (tid == 0 && all < (u64)k_in) sh.mode = SG_SLOW;
      } else if (all <= SG_LIST) {
        if (tid == 0) {
          sh.lo = 0;
          sh.hi = SG_BINS;
        }
      } else {
        // mass of a bin to 2^-15 of it: count less the chord's share of the positions, half of what the chord is above exp at most
        constexpr float drop = 0.015503562f, above = 1.52587890625e-5f;   // 1 - exp(-1/64), (1/64)^2 / 16
        float m[SG_PER], sum_m = 0.f, total;
#pragma unroll
        for (int i = 0; i < SG_PER; ++i) {
          const int b = tid * SG_PER + i;
          m[i] = __expf((float)b * (-SG_RANGE / SG_BINS)) * ((float)n[i] * (1.f - above) - (float)sh.frac[b] * (drop / 8192.f));
          sum_m += m[i];
        }
        float b = block_prefix(sum_m, total, sh.scan_f);
        if (!(min_p > 0.f)) total = (float)approx;
        const float want = top_p * total, margin = total * 1.2e-4f;       // the error on either side, with room
        int first = SG_BINS, last = 0;
#pragma unroll
        for (int i = 0; i < SG_PER; ++i) {
          if (n[i]) {
            if (b + m[i] >= want - margin) first = min(first, tid * SG_PER + i);
            if (b <= want + margin) last = tid * SG_PER + i;
          }
          b += m[i];
        }
        first = __reduce_min_sync(0xffffffffu, first);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) {
          atomicMin(&sh.lo, first);
          atomicMax(&sh.hi, last);
        }
        __syncthreads();
        u64 inside = 0, listed;
#pragma unroll
        for (int i = 0; i < SG_PER; ++i)
          if (tid * SG_PER + i >= sh.lo && tid * SG_PER + i <= sh.hi) inside += n[i];
        block_prefix(inside, listed, sh.scan);
        if (tid == 0 && (listed > SG_LIST || sh.hi < sh.lo)) sh.mode = SG_SLOW;
      }
      __syncthreads();
      // The least logits whose place is in front of the window, and in front of its end: five bits of their keys at a time, a lane for each of 32 values.
      if (warp < 2) {
        const float end = warp == 0 ? (float)sh.lo : (sh.hi >= SG_BINS - 1 ? INFINITY : (float)sh.hi + 1.f);
        const uint32_t most = key_of(r.mx);
        uint32_t key = 0;
#pragma unroll 1
        for (int shift = 27; shift > -5; shift -= 5) {
          const int by = max(shift, 0);
          const uint32_t last = min(key + ((uint32_t)lane << by) + ((1u << by) - 1), most);
          const unsigned m = __ballot_sync(0xffffffffu, r.place(of_key(last)) < end);
          key += m ? (uint32_t)(__ffs(m) - 1) << by : 0;
        }
        if (lane == 0) sh.first[warp] = end > 0.f ? of_key(key) : INFINITY;
      }
      __syncthreads();
      if (tid > 0 && tid < nc) {
        *at_rank(&sh.mode, tid) = sh.mode;
        *at_rank(&sh.first[0], tid) = sh.first[0];
        *at_rank(&sh.first[1], tid) = sh.first[1];
      }
    }
    cluster_barrier();
    mode = sh.mode;
  }

  // 3
  const bool whole_row = by_p && !by_k && !(min_p > 0.f);                 // S is the mass of the row
  if (mode == SG_ALL) {
    u64 whole = 0;
#pragma unroll 1
    for (int t = tile0; t < tile1; ++t) {
      float x[8];
      raw8(load8(x0, off, V, t * SG_THREADS + tid), x);
      u64 sure = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double w = r.weight(x[j]);                                  // not a number: 0
        const u64 n = SgRow::rounded(w);
        whole += n;
        sure += w >= r.least ? n : 0ull;
      }
      sure = warp_sum(sure);
      if (lane == 0) *at_rank(&sh.tile[t * SG_WARPS + warp], 0) = sure;
    }
    u64 a;
    block_prefix(whole, a, sh.scan);
    if (tid == 0) *at_rank(&sh.whole[rank], 0) = a;
    cluster_barrier();
  } else if (mode == SG_WINDOW) {
    // 64-bit weights of what is in front of the window and, for top-p's mass S, of what lies behind it: down to min-p's bound, or of the whole row.  The list's are the first block's.
    // Where few of a piece's elements count they are pushed together before their weights are computed.
    const bool by_both = by_p && !by_k && !whole_row;                     // S is what min-p leaves
    const float front = fmaxf(sh.first[0], bound), inside = fmaxf(sh.first[1], bound), need = by_both ? bound : inside;
    u64 rest = 0;
    float* q = sh.queue[warp];
#pragma unroll 1
    for (int t = tile0; t < tile1; ++t) {
      const float top = piece_top(t);
      u64 sure = 0;
      if (whole_row ? !(r.place(top) >= (float)SG_BINS) : top >= need) {  // beyond the range there is no mass
        float x[8];
        raw8(load8(x0, off, V, t * SG_THREADS + tid), x);
        unsigned listed = 0, mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          mine |= (unsigned)(x[j] >= front) << j;
          listed |= (unsigned)(x[j] >= inside) << j;
        }
        listed &= ~mine;
        append(sh, listed, x, (t * SG_THREADS + tid) * 8 - off);
        if (whole_row) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const u64 w = SgRow::rounded(r.weight(x[j]));                 // not a number: 0
            if (x[j] >= front) sure += w;
            else if (!(listed >> j & 1)) rest += w;
          }
          sure = warp_sum(sure);
        } else {
          if (by_both) {
#pragma unroll
            for (int j = 0; j < 8; ++j) mine |= (unsigned)(x[j] >= bound && x[j] < inside) << j;
          }
          if (__any_sync(0xffffffffu, mine)) {
            const int has = __popc(mine);
            int run = has;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
              const int up = __shfl_up_sync(0xffffffffu, run, o);
              if (lane >= o) run += up;
            }
            const int n = __shfl_sync(0xffffffffu, run, 31);
            float* to = q + run - has;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (mine >> j & 1) *to++ = x[j];
            __syncwarp();
#pragma unroll 1
            for (int i = lane; i < n; i += 32) {
              const u64 w = r.kept(q[i]);
              if (q[i] >= front) sure += w;
              else rest += w;
            }
            __syncwarp();
            sure = warp_sum(sure);
          }
        }
      }
      if (lane == 0) *at_rank(&sh.tile[t * SG_WARPS + warp], 0) = sure;
    }
    u64 a;
    block_prefix(rest, a, sh.scan);
    if (tid == 0) *at_rank(&sh.whole[rank], 0) = a;
    join_lists(sh, rank);
    cluster_barrier();
    if (by_k && by_p) mode = SG_TOP;
  }
  if (rank) return;

  float u = p.u[row];
  u = u > 0.f ? u : 0.f;
  // The running mass has to pass it; u = 1 takes the last element with mass.
  auto pass = [&](u64 total) { return fmin((double)u * (double)total, __longlong_as_double(__double_as_longlong((double)total) - 1)); };
  const int n_list = min(sh.n_list, (uint32_t)SG_LIST);
  if (mode == SG_TOP && n_list <= SG_FEW) {
    if (tid < n_list) sh.mass[tid] = r.kept_one(of_key((uint32_t)(sh.list[tid] >> 32)));
    __syncthreads();
    SgPlace at = place_of<false>(sh.list, sh.mass, n_list);
    u64 m = at.e >= 0 && at.rank < k_in ? sh.mass[at.e] : 0ull, total;
    block_prefix(at.first ? m : 0ull, total, sh.scan);
    if (by_p) {
      if (at.rank && !((double)at.before < (double)top_p * (double)total)) m = 0;
      block_prefix(at.first ? m : 0ull, total, sh.scan);
    }
    if (at.e >= 0 && at.first) sh.mass[at.e] = m;                         // every thread has read the masses before
    __syncthreads();
    at = place_of<true>(sh.list, sh.mass, n_list);
    const double want = pass(total);
    if (at.e >= 0 && at.first && (double)at.before <= want && (double)(at.before + m) > want) {
      const u64 word = sh.list[at.e];
      p.ids[row] = (int)~(uint32_t)word;
      if (p.logprob) p.logprob[row] = (float)(r.scaled(of_key((uint32_t)(word >> 32))) - log(approx));
    }
    return;
  }
  if (mode == SG_TOP) {
    const int each = n_list <= SG_THREADS ? 1 : SG_EACH, n = min(k_in, n_list);      // neighbours of the order per thread
    if (each == 1) sort_down_few(sh.list, n_list);
    else sort_down(sh.list, n_list);
    u64 mine = 0, total;
#pragma unroll 1
    for (int i = 0; i < each; ++i) {
      const int at = tid * each + i;
      const u64 w = at < n ? r.kept_one(of_key((uint32_t)(sh.list[at] >> 32))) : 0ull;
      sh.mass[at] = w;
      mine += w;
    }
    u64 before = block_prefix(mine, total, sh.scan);
    const double limit = by_p ? (double)top_p * (double)total : DBL_MAX;
    mine = 0;
    // what stays, in the order of the indexes: the complement of the index, larger first, and the place in the order before
    u64 word[SG_EACH];
#pragma unroll
    for (int i = 0; i < SG_EACH; ++i) {
      const int at = tid * each + i;
      if (i >= each || at >= n) {
        word[i] = 0;
        continue;
      }
      const bool stays = at == 0 || (double)before < limit;
      before += sh.mass[at];
      word[i] = stays ? sh.list[at] << 32 | (uint32_t)at : 0;
      if (stays) mine += sh.mass[at];
      sh.key[at] = (uint32_t)(sh.list[at] >> 32);
    }
    block_prefix(mine, total, sh.scan);
#pragma unroll
    for (int i = 0; i < SG_EACH; ++i)
      if (i < each) sh.list[tid * each + i] = word[i];
    __syncthreads();
    if (each == 1) sort_down_few(sh.list, n);
    else sort_down(sh.list, n);
    mine = 0;
#pragma unroll 1
    for (int i = 0; i < each; ++i)
      if (const u64 w = sh.list[tid * each + i]) mine += sh.mass[(uint32_t)w];
    u64 at_mass = block_prefix(mine, total, sh.scan);
    const double want = pass(total);
    if ((double)at_mass <= want && (double)(at_mass + mine) > want) {
#pragma unroll 1
      for (int i = 0; i < each; ++i) {
        const u64 w = sh.list[tid * each + i], m = w ? sh.mass[(uint32_t)w] : 0ull;
        if ((double)at_mass <= want && (double)(at_mass + m) > want) {
          p.ids[row] = (int)~(uint32_t)(w >> 32);
          if (p.logprob) p.logprob[row] = (float)(r.scaled(of_key(sh.key[(uint32_t)w])) - log(approx));
        }
        at_mass += m;
      }
    }
    return;
  }
  u64 whole = 0, cut = 0;
  if (mode == SG_ALL || mode == SG_WINDOW)
    for (uint32_t c = 0; c < nc; ++c) whole += sh.whole[c];
  if (mode == SG_WINDOW) {
    u64 mine = 0, sure, listed;
#pragma unroll
    for (int i = 0; i < SG_PER_PIECE; ++i)
      if (tid + i * SG_THREADS < pieces) mine += sh.tile[tid + i * SG_THREADS];
    block_prefix(mine, sure, sh.scan);
    const int each = n_list <= SG_THREADS ? 1 : SG_EACH;                        // neighbours of the order per thread
    if (each == 1) sort_down_few(sh.list, n_list);
    else sort_down(sh.list, n_list);
    mine = 0;
#pragma unroll 1
    for (int i = 0; i < each; ++i) {
      const int at = tid * each + i;
      const u64 w = at < n_list ? r.kept_one(of_key((uint32_t)(sh.list[at] >> 32))) : 0ull;
      sh.mass[at] = w;
      mine += w;
    }
    u64 before = block_prefix(mine, listed, sh.scan);
    const u64 behind = whole;
    whole = sure + listed + behind;
    const double limit = (double)top_p * (double)whole;
    const u64 front = by_k ? sh.found[0] : 0;
    // The last one that stays.
    u64 last = ~0ull;
#pragma unroll 1
    for (int i = 0; i < each; ++i) {
      const int at = tid * each + i;
      if (at < n_list && (by_k ? front + at < (u64)k_in : (double)(sure + before) < limit || (at == 0 && sure == 0))) last = min(last, sh.list[at]);
      before += sh.mass[at];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) last = min(last, __shfl_xor_sync(0xffffffffu, last, o));
    __syncthreads();
    if (lane == 0) sh.scan[warp] = last;
    __syncthreads();
    for (int w = 0; w < SG_WARPS; ++w) last = min(last, sh.scan[w]);
    // The window holds the cut if its first element or something before it stays, and what lies behind does not.
    if (sh.n_list <= SG_LIST && ~last && (by_k || !(behind && (double)(sure + listed) < limit))) {
      cut = last;
      // pieces get what is kept of the list
      for (int i = tid; i < n_list; i += SG_THREADS) {
        const u64 word = sh.list[i];
        if (word >= cut && sh.mass[i]) atomicAdd(&sh.tile[((int)~(uint32_t)word + off) / SG_PIECE], sh.mass[i]);
      }
      __syncthreads();
    } else {
      mode = SG_SLOW;
    }
  }
  if (mode == SG_SLOW) {
    // weights of the whole row, cuts by histograms, sums per piece: all by this block
    u64 upto = 0, mine = 0, mine_kept = 0, kept;
#pragma unroll 1
    for (int v = tid; v < vecs; v += SG_THREADS) {
      float x[8];
      fetch8(x0, off, V, v, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double w = r.weight(x[j]);
        const u64 n = SgRow::rounded(w);
        mine += n;
        if (w >= r.least) mine_kept += n;
      }
    }
    block_prefix(mine, whole, sh.scan);
    block_prefix(mine_kept, kept, sh.scan);
    cut = 0;
    if (by_k) {
      cut = slow_cut(x0, off, V, r, sh, false, (double)k_in, 0, upto);
      kept = upto;
    }
    if (by_p) cut = slow_cut(x0, off, V, r, sh, true, (double)top_p * (double)kept, cut, upto);
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      const int v = t * SG_THREADS + tid;
      u64 sure = 0;
      float x[8];
      fetch8(x0, off, V, v, x);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (word_of(x[j], v * 8 - off + j) >= cut) sure += r.kept_one(x[j]);
      sure = warp_sum(sure);
      if (lane == 0) sh.tile[t * SG_WARPS + warp] = sure;
    }
    __syncthreads();
  }
  // the piece that the random number falls into, three neighbours per thread
  u64 n3[SG_PER_PIECE], mine = 0, total;
#pragma unroll
  for (int i = 0; i < SG_PER_PIECE; ++i) {
    const int at = tid * SG_PER_PIECE + i;
    n3[i] = at < pieces ? sh.tile[at] : 0ull;
    mine += n3[i];
  }
  u64 before = block_prefix(mine, total, sh.scan);
  const double want = pass(total);
  if ((double)before <= want && (double)(before + mine) > want) {
#pragma unroll
    for (int i = 0; i < SG_PER_PIECE; ++i) {
      if ((double)before <= want && (double)(before + n3[i]) > want) {
        sh.found[0] = (u64)(tid * SG_PER_PIECE + i);
        sh.found[1] = before;
      }
      before += n3[i];
    }
  }
  __syncthreads();
  if (warp) return;
  // eight rounds of 32 neighbours
  const int index = ((int)sh.found[0] * SG_PIECE) - off + lane;
  before = sh.found[1];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = index + j * 32;
    sh.queue[0][j * 32 + lane] = i >= 0 && i < V ? (float)x0[i] : -INFINITY;
  }
#pragma unroll 1
  for (int j = 0; j < 8; ++j) {
    const int i = index + j * 32;
    float x = sh.queue[0][j * 32 + lane];
    x = x == x ? x + 0.f : -INFINITY;
    const u64 m = word_of(x, i) >= cut ? r.kept_one(x) : 0ull;
    u64 run = m;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const u64 up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    run += before;
    const unsigned passed = __ballot_sync(0xffffffffu, (double)run > want);
    if (passed) {
      if (lane == __ffs(passed) - 1) {
        p.ids[row] = i;
        if (p.logprob) p.logprob[row] = (float)(r.scaled(x) - log(mode == SG_WINDOW && !whole_row ? approx : (double)whole * (1.0 / SG_ONE)));
      }
      break;
    }
    before = __shfl_sync(0xffffffffu, run, 31);
  }
}

// The last element of the order, among those with words from floor_word on, before which less than `limit` of mass lies or fewer than `limit` elements (as doubles); the first one
// at least.  `upto`: the mass up to and with it.  Histograms of the words in [lo, hi], narrower from level to level, until a bin's elements fit the list.
template <typename T>
__device__ __noinline__ u64 slow_cut(const T* row, int off, int V, const SgRow& r, SgShared& sh, bool by_mass, double limit, u64 floor_word, u64& upto) {
  const int tid = threadIdx.x, lane = tid & 31, vecs = (V + off + 7) / 8;
  u64 lo = floor_word, hi = word_of(r.mx, 0), mass_before = 0, count_before = 0;
  int shift = 53;                                       // 64 - 11
  for (;;) {
    const u64 span = hi - lo;
    shift = span < SG_BINS ? 0 : 53 - __clzll((long long)span);          // span >> shift is below 2048
    __syncthreads();
    for (int b = tid; b < SG_BINS; b += SG_THREADS) {
      sh.count[b] = 0;
      sh.mass[b] = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int v0 = 0; v0 < vecs; v0 += SG_THREADS) {
      const int v = v0 + tid;
      int at = -1;
      uint32_t run = 0;
      u64 m = 0;
      if (v < vecs) {
        float x[8];
        fetch8(row, off, V, v, x);
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
          const u64 word = word_of(x[j], v * 8 - off + j);
          if (x[j] == -INFINITY || word < lo || word > hi) continue;
          const int b = (int)((hi - word) >> shift);
          if (b != at) {
            if (run) { atomicAdd(&sh.count[at], run); atomicAdd(&sh.mass[at], m); }
            at = b;
            run = 0;
            m = 0;
          }
          ++run;
          m += r.kept_one(x[j]);
        }
      }
      int same;
      __match_all_sync(0xffffffffu, at, &same);
      if (same) {
        run = __reduce_add_sync(0xffffffffu, run);
        m = warp_sum(m);
        if (lane) run = 0;
      }
      if (run) { atomicAdd(&sh.count[at], run); atomicAdd(&sh.mass[at], m); }
    }
    __syncthreads();
    u64 m[SG_PER], n[SG_PER], m_sum = 0, n_sum = 0, all_m, all_n;
#pragma unroll
    for (int i = 0; i < SG_PER; ++i) {
      m[i] = sh.mass[tid * SG_PER + i];
      n[i] = sh.count[tid * SG_PER + i];
      m_sum += m[i];
      n_sum += n[i];
    }
    u64 mb = block_prefix(m_sum, all_m, sh.scan) + mass_before, nb = block_prefix(n_sum, all_n, sh.scan) + count_before;
    // the last bin with elements that begins below the limit, the first one with elements at least
    int last = -1;
    u64 last_m = 0, last_n = 0, inside = 0;
#pragma unroll
    for (int i = 0; i < SG_PER; ++i) {
      if (n[i] > 0 && (nb == count_before || (by_mass ? (double)mb : (double)nb) < limit)) {
        last = tid * SG_PER + i;
        last_m = mb;
        last_n = nb;
        inside = n[i];
      }
      mb += m[i];
      nb += n[i];
    }
    const int most = __reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (lane == 0) sh.scan[tid >> 5] = (u64)(long long)most;
    __syncthreads();
    int bin = -1;
    for (int w = 0; w < SG_WARPS; ++w) bin = max(bin, (int)(long long)sh.scan[w]);
    if (bin >= 0 && last == bin) {
      sh.found[0] = last_m;
      sh.found[1] = last_n;
      sh.found[2] = inside;
    }
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    if (bin < 0) {                                      // no elements: the cut stays where it was
      upto = mass_before;
      return floor_word;
    }
    mass_before = sh.found[0];
    count_before = sh.found[1];
    inside = sh.found[2];
    const u64 front = hi - ((u64)bin << shift), width = (1ull << shift) - 1;
    lo = max(lo, front > width ? front - width : 0ull);
    hi = front;
    if (inside > SG_LIST) continue;
#pragma unroll 1
    for (int v = tid; v < vecs; v += SG_THREADS) {
      float x[8];
      fetch8(row, off, V, v, x);
#pragma unroll 1
      for (int j = 0; j < 8; ++j) {
        const u64 word = word_of(x[j], v * 8 - off + j);
        if (x[j] == -INFINITY || word < lo || word > hi) continue;
        const uint32_t to = atomicAdd(&sh.n_list, 1u);
        sh.list[to] = word;
      }
    }
    __syncthreads();
    const int count = (int)inside;
    sort_down(sh.list, count);
    u64 mine = 0, all;
    for (int i = 0; i < SG_EACH; ++i) {
      const int at = tid * SG_EACH + i;
      if (at < count) mine += sh.mass[at] = r.kept_one(of_key((uint32_t)(sh.list[at] >> 32)));
    }
    u64 before = block_prefix(mine, all, sh.scan) + mass_before;
    last = -1;
    for (int i = 0; i < SG_EACH; ++i) {
      const int at = tid * SG_EACH + i;
      if (at >= count) break;
      const u64 me = sh.mass[at];
      if (at == 0 || (by_mass ? (double)before : (double)(count_before + at)) < limit) {
        last = at;
        last_m = before + me;
      }
      before += me;
    }
    const int end = __reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (lane == 0) sh.scan[tid >> 5] = (u64)(long long)end;
    __syncthreads();
    int at = -1;
    for (int w = 0; w < SG_WARPS; ++w) at = max(at, (int)(long long)sh.scan[w]);
    if (last == at) sh.found[0] = last_m;
    __syncthreads();
    upto = sh.found[0];
    const u64 got = sh.list[at];
    __syncthreads();
    return got;
  }
}

}  // namespace omni

using namespace omni;

// logits [B, V] of pitch ld, bf16 or fp32; parameters per row or (null) one value for all; u fp32 [B]; ids int32 [B], logprob fp32 [B] or null.
extern "C" int omni_sample_given(const void* logits, int is_bf16, long ld, int V, int B, const float* u, const float* temperature, float temperature_v, const int* top_k,
                                 int top_k_v, const float* top_p, float top_p_v, const float* min_p, float min_p_v, int* ids, float* logprob, void* stream) {
  if (B <= 0) return RC_OK;
  if (V < 1 || V > SG_MAX_V) return RC_BAD_ARG;
  const SampleGiven p = {logits, ld, V, temperature, top_p, min_p, u, top_k, temperature_v, top_p_v, min_p_v, top_k_v, ids, logprob};
  // Two blocks fit an SM: as many a row as make two rounds of them at most, since rows differ in what they cost (two draws of 256 rows of 152064, all kinds: 149 and 132 us with
  // two blocks a row, 192 and 193 with one, 162 and 135 with four; of 100 rows 81 and 76 with four, 108 and 105 with two, 87 and 80 with eight), a tile each at least.
  int nc = 1;
  while (nc < SG_MAX_CLUSTER && (long)B * nc * 2 <= 4L * sm_count() && nc * 2 * SG_TILE <= V) nc *= 2;
  if ((long)B * nc > 0x7fffffffL) return RC_TOO_LARGE;
  static unsigned long long ready[2] = {0, 0};
  const void* fn = is_bf16 ? (const void*)sample_given_kernel<__nv_bfloat16> : (const void*)sample_given_kernel<float>;
  if (int e = ensure_dynamic_smem(fn, (int)sizeof(SgShared), ready[is_bf16 ? 0 : 1])) return e;
  launch_with(true, nc, is_bf16 ? sample_given_kernel<__nv_bfloat16> : sample_given_kernel<float>, dim3((unsigned)(B * nc)), SG_THREADS, sizeof(SgShared),
              (cudaStream_t)stream, p);
  return (int)cudaGetLastError();
}
