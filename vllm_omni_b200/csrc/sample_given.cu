// Tokens drawn from given random numbers: temperature, top-k, min-p and top-p over rows of logits, exactly.
//
// For a row x with maximum m and temperature T, weights are whole numbers w_i = round(2^44 exp((x_i - m) / T)), so that sums of them have no order: blocks,
// threads and atomics may add them as they come, and the plain definition in 64 bits gives the same token.  The order of a row is (x down, index up).  A cut is
// the last element of that order that stays:
//   top-k   the k-th element;
//   min-p   elements whose weight is below min_p of the largest have no mass (they are the end of the order);
//   top-p   of what is left, with mass S, the last element before which less than top_p S lies.
// The token is the first kept index in the vocabulary's order at which the running mass passes u times the kept mass.
//
// A row is read once and stays in the shared memory of a cluster, one slice of the vocabulary per block, in fp32.  A cut is found by a histogram of 2048 bins
// (count and mass) over x, then of the bin that it falls into: over its keys, in the end over the indexes of ties; once at most 1024 elements are left in a
// bin every block gets a list of them and ranks it.  Threads own an odd number of neighbouring elements, so that walking them has no bank conflicts and
// their sums are prefixes in the vocabulary's order.
#include <cuda_bf16.h>

#include "host_util.h"
#include "ptx_sm100.cuh"

namespace omni {

constexpr int SG_THREADS = 512, SG_BINS = 2048, SG_LIST = 1024, SG_MAX_V = 262144, SG_MAX_CLUSTER = 8;
constexpr int SG_PER = SG_BINS / SG_THREADS;
constexpr double SG_ONE = 17592186044416.0;             // 2^44
typedef unsigned long long u64;

struct SampleGiven {
  const void* logits;
  long ld;
  int V, per;                                           // elements per thread (odd); a block owns SG_THREADS * per
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

struct SgShared {
  u64 mass[SG_BINS];
  uint32_t count[SG_BINS];
  u64 list[SG_LIST];                                    // key << 32 | ~index: larger comes first in the order
  u64 list_w[SG_LIST];
  u64 from[SG_MAX_CLUSTER], from2[SG_MAX_CLUSTER];      // a word of every block of the cluster
  u64 scan[SG_THREADS / 32];
  u64 found[4];
  uint32_t n_list;
};

template <typename T>
__device__ __forceinline__ T* at_rank(T* p, uint32_t rank) {            // the same shared variable of another block of the cluster
  u64 out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<u64>(p)), "r"(rank));
  return reinterpret_cast<T*>(out);
}

// Barrier of the cluster, for warps whose threads may have left a loop at different times.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Exclusive prefix of v over the block's threads, and the total.
__device__ __forceinline__ u64 block_prefix(u64 v, u64& total, u64* sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  u64 run = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const u64 up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();                                      // the previous use of `sh` is over
  if (lane == 31) sh[warp] = run;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SG_THREADS / 32; ++w) {
    const u64 x = sh[w];
    before += w < warp ? x : 0;
    all += x;
  }
  total = all;
  return before + run - v;
}

template <typename T>
__global__ void __launch_bounds__(SG_THREADS)
sample_given_kernel(const __grid_constant__ SampleGiven p) {
  extern __shared__ __align__(16) unsigned char raw[];
  SgShared& sh = *reinterpret_cast<SgShared*>(raw);
  float* xs = reinterpret_cast<float*>(raw + sizeof(SgShared));
  const uint32_t rank = cluster_ctarank();
  uint32_t nc;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nc));
  const int row = blockIdx.x / nc, tid = threadIdx.x;
  const int first = rank * SG_THREADS * p.per, n = max(0, min(p.V - first, SG_THREADS * p.per));
  const int mine = tid * p.per, mine_end = min(n, mine + p.per);
  pdl_begin();
  const float T_in = p.temperature ? p.temperature[row] : p.temperature_v;
  const bool greedy = !(T_in > 0.f);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)T_in;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_v, min_p = fminf(p.min_p ? p.min_p[row] : p.min_p_v, 1.f);
  const int k_in = p.top_k ? p.top_k[row] : p.top_k_v;

  // the row into shared memory, its largest element (and of equal ones the first)
  const T* lg = reinterpret_cast<const T*>(p.logits) + (long)row * p.ld + first;
  u64 best = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += SG_THREADS) {
    float x = (float)lg[i];
    if (!(x == x)) x = -INFINITY;                       // not a number: never drawn
    if (x == 0.f) x = 0.f;                              // one zero
    xs[i] = x;
    best = max(best, (u64)key_of(x) << 32 | (uint32_t)~(first + i));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) sh.scan[tid >> 5] = best;
  __syncthreads();
  if (tid < nc) {
    best = sh.scan[0];
    for (int w = 1; w < SG_THREADS / 32; ++w) best = max(best, sh.scan[w]);
    *at_rank(&sh.from[rank], tid) = best;
  }
  cluster_barrier();
  best = 0;
  for (uint32_t c = 0; c < nc; ++c) best = max(best, sh.from[c]);
  const int best_id = (int)~(uint32_t)best;
  const uint32_t top_key = (uint32_t)(best >> 32);
  const float mx = __uint_as_float(top_key & 0x80000000u ? top_key & 0x7fffffffu : ~top_key);
  const bool nothing = mx == -INFINITY;

  auto scaled = [&](float x) { return x == mx ? 0.0 : ((double)x - (double)mx) * inv_t; };
  auto weight = [&](float x) {
    const double z = scaled(x);
    return z > -32.0 ? (u64)__double2ll_rn(exp(z) * SG_ONE) : 0ull;
  };
  // min-p compares the unrounded weight; below it an element has no mass
  auto kept_weight = [&](float x, u64& w) {
    const double z = scaled(x);
    const double e = z > -745.0 ? exp(z) : 0.0;
    w = z > -32.0 ? (u64)__double2ll_rn(e * SG_ONE) : 0ull;
    return e >= (double)min_p;
  };

  // all weights, the mass of those that min-p keeps
  u64 all = 0, kept = 0;
  const bool by_k = !greedy && k_in > 0 && k_in < p.V, by_p = !greedy && top_p < 1.f;
  if (by_k || by_p)
    for (int b = tid; b < SG_BINS; b += SG_THREADS) { sh.mass[b] = 0; sh.count[b] = 0; }
  __syncthreads();
  const float to_bin = SG_BINS / (32.f * (greedy ? 1.f : T_in));
  auto bin_of = [&](float x) { return (int)fminf((mx - x) * to_bin, (float)(SG_BINS - 1)); };        // monotone; -inf - -inf does not come here
  if (!nothing) {
#pragma unroll 1
    for (int i = mine; i < mine_end; ++i) {
      const float x = xs[i];
      u64 w;
      const bool in = kept_weight(x, w);
      all += w;
      if (in) kept += w;
      if (by_k || by_p) {
        const int b = x == mx ? 0 : bin_of(x);
        atomicAdd(&sh.count[b], 1u);
        if (in && w) atomicAdd(&sh.mass[b], w);
      }
    }
  }
  u64 all_block, kept_block;
  block_prefix(all, all_block, sh.scan);
  const u64 my_prefix = block_prefix(kept, kept_block, sh.scan);
  if (tid < nc) *at_rank(&sh.from2[rank], tid) = all_block;
  cluster_barrier();                                   // histograms and sums of every block are there
  u64 whole = 0;
  for (uint32_t c = 0; c < nc; ++c) whole += sh.from2[c];

  // The cut, as key << 32 | ~index of the last kept element: an element stays if its word is not less.
  u64 cut = 0;
  // Finds the last element of the order before which less than `limit` (as a double, of mass) or fewer than `limit` (of count) lies; elements below `floor_word`
  // are not there.  `upto`: the mass up to and with it.
  // A level looks at the elements with word in [lo, hi] by sub-bins; `inside` counts mass and elements before lo's first.
  auto select = [&](bool by_mass, double limit, u64 floor_word, bool have_histogram, u64& upto) {
    u64 hi = ~0ull, lo = floor_word, mass_before = 0, count_before = 0;
    int level = 0, shift = 0;
    for (;;) {
      // sub-bin of an element at this level: 0 is the front of the order
      auto sub = [&](float x, u64 word) {
        if (level == 0) return x == mx ? 0 : bin_of(x);
        return (int)((hi - word) >> shift);
      };
      if (!(level == 0 && have_histogram)) {
        for (int b = tid; b < SG_BINS; b += SG_THREADS) { sh.mass[b] = 0; sh.count[b] = 0; }
        __syncthreads();
#pragma unroll 1
        for (int i = mine; i < mine_end; ++i) {
          const float x = xs[i];
          const u64 word = (u64)key_of(x) << 32 | (uint32_t)~(first + i);
          if (word < lo || word > hi) continue;
          u64 w;
          const bool in = kept_weight(x, w);
          const int b = sub(x, word);
          atomicAdd(&sh.count[b], 1u);
          if (in && w) atomicAdd(&sh.mass[b], w);
        }
        cluster_barrier();
      }
      // the cluster's histogram: every block adds it up for itself
      u64 m[SG_PER], cn[SG_PER], m_sum = 0, c_sum = 0;
#pragma unroll
      for (int i = 0; i < SG_PER; ++i) {
        m[i] = cn[i] = 0;
        for (uint32_t c = 0; c < nc; ++c) {
          m[i] += *at_rank(&sh.mass[tid * SG_PER + i], c);
          cn[i] += *at_rank(&sh.count[tid * SG_PER + i], c);
        }
        m_sum += m[i];
        c_sum += cn[i];
      }
      u64 tm, tc;
      u64 mb = block_prefix(m_sum, tm, sh.scan) + mass_before, cb = block_prefix(c_sum, tc, sh.scan) + count_before;
      if (tid == 0) sh.found[0] = ~0ull;
      __syncthreads();
      // the last bin with elements before which less than the limit lies (the first one that has elements if there is none)
      int last = -1;
      u64 last_m = 0, last_c = 0;
#pragma unroll
      for (int i = 0; i < SG_PER; ++i) {
        const bool ok = cn[i] > 0 && (cb == count_before || (by_mass ? (double)mb : (double)cb) < limit);
        if (ok) { last = tid * SG_PER + i; last_m = mb; last_c = cb; }
        mb += m[i];
        cb += cn[i];
      }
      // the largest such bin over the block
      int most = __reduce_max_sync(0xffffffffu, last);
      if ((tid & 31) == 0) sh.scan[tid >> 5] = (u64)(long long)most;
      __syncthreads();
      int bin = -1;
      for (int w = 0; w < SG_THREADS / 32; ++w) bin = max(bin, (int)(long long)sh.scan[w]);
      __syncthreads();
      if (bin < 0) {                                    // no elements at all: the cut stays open
        upto = mass_before;
        cluster_barrier();
        return floor_word;
      }
      if (last == bin) {
        sh.found[0] = last_m;
        sh.found[1] = last_c;
        sh.found[2] = cn[bin - tid * SG_PER];
      }
      __syncthreads();
      mass_before = sh.found[0];
      count_before = sh.found[1];
      const u64 inside = sh.found[2];
      if (tid == 0) sh.n_list = 0;
      cluster_barrier();                               // all have read the histograms; every list is empty
      if (inside <= SG_LIST) {
#pragma unroll 1
        for (int i = mine; i < mine_end; ++i) {
          const float x = xs[i];
          const u64 word = (u64)key_of(x) << 32 | (uint32_t)~(first + i);
          if (word < lo || word > hi || sub(x, word) != bin) continue;
          u64 w;
          if (!kept_weight(x, w)) w = 0;
          const uint32_t to = atomicAdd(at_rank(&sh.n_list, 0), 1u);    // one counter for the cluster, so that every list has the same order
          for (uint32_t c = 0; c < nc; ++c) {
            *at_rank(&sh.list[to], c) = word;
            *at_rank(&sh.list_w[to], c) = w;
          }
        }
        cluster_barrier();
        // rank of every element of the list: what lies before it
        if (tid == 0) { sh.found[0] = ~0ull; sh.found[1] = 0; }
        __syncthreads();
        u64 lowest = ~0ull, total_at = 0;
        for (int e = tid; e < (int)inside; e += SG_THREADS) {
          const u64 word = sh.list[e];
          u64 bm = mass_before, bc = count_before;
          for (int j = 0; j < (int)inside; ++j)
            if (sh.list[j] > word) { bm += sh.list_w[j]; ++bc; }
          if ((bc == count_before || (by_mass ? (double)bm : (double)bc) < limit) && word < lowest) { lowest = word; total_at = bm + sh.list_w[e]; }
        }
        atomicMin(&sh.found[0], lowest);
        __syncthreads();
        const u64 got = sh.found[0];
        if (lowest == got) sh.found[1] = total_at;
        __syncthreads();
        upto = sh.found[1];
        cluster_barrier();
        return got;
      }
      // narrower: the words of this bin
      if (level == 0) {
        // bounds of the bin's keys: those of its elements
        u64 a = 0, z = ~0ull;
#pragma unroll 1
        for (int i = mine; i < mine_end; ++i) {
          const float x = xs[i];
          const u64 word = (u64)key_of(x) << 32 | (uint32_t)~(first + i);
          if (word < lo || word > hi || sub(x, word) != bin) continue;
          a = max(a, word);
          z = min(z, word);
        }
        if (tid == 0) { sh.found[0] = 0; sh.found[1] = ~0ull; }
        __syncthreads();
        atomicMax(&sh.found[0], a);
        atomicMin(&sh.found[1], z);
        __syncthreads();
        if (tid < nc) {
          *at_rank(&sh.from[rank], tid) = sh.found[0];
          *at_rank(&sh.from2[rank], tid) = sh.found[1];
        }
        cluster_barrier();
        for (uint32_t c = 0; c < nc; ++c) {
          a = max(a, sh.from[c]);
          z = min(z, sh.from2[c]);
        }
        hi = a;
        lo = z;
      } else {
        const u64 top = hi - ((u64)bin << shift), width = (1ull << shift) - 1;
        lo = max(lo, top > width ? top - width : 0);
        hi = top;
      }
      ++level;
      const u64 span = hi - lo;
      shift = span < SG_BINS ? 0 : 64 - __clzll((long long)span) - 11;   // span >> shift is below 2048
    }
  };

  u64 upto = 0, cut_mass = 0;
  bool truncated = false;
  if (!nothing && by_k) {
    cut = select(false, (double)k_in, 0, true, upto);
    cut_mass = upto;
    truncated = true;
  }
  if (!nothing && by_p) {
    u64 mass = cut_mass;
    if (!by_k) {
      if (tid < nc) *at_rank(&sh.from[rank], tid) = kept_block;
      cluster_barrier();
      mass = 0;
      for (uint32_t c = 0; c < nc; ++c) mass += sh.from[c];
    }
    cut = select(true, (double)top_p * (double)mass, cut, !by_k, upto);
    truncated = true;
  }

  // kept mass in the vocabulary's order
  u64 before = my_prefix, block_total = kept_block, own = kept;
  if (truncated) {
    own = 0;
#pragma unroll 1
    for (int i = mine; i < mine_end; ++i) {
      const float x = xs[i];
      if (((u64)key_of(x) << 32 | (uint32_t)~(first + i)) < cut) continue;
      u64 w;
      if (kept_weight(x, w)) own += w;
    }
    before = block_prefix(own, block_total, sh.scan);
  }
  if (tid < nc) *at_rank(&sh.from[rank], tid) = block_total;
  cluster_barrier();
  u64 total = 0;
  for (uint32_t c = 0; c < nc; ++c) {
    if (c < rank) before += sh.from[c];
    total += sh.from[c];
  }
  const double log_all = log((double)whole * (1.0 / SG_ONE));
  if (nothing || greedy) {
    if (rank == 0 && tid == 0) {
      p.ids[row] = nothing ? -1 : best_id;
      if (p.logprob) p.logprob[row] = nothing ? -INFINITY : (float)-log_all;
    }
  } else {
    float u = p.u[row];
    u = u > 0.f ? u : 0.f;
    const double want = fmin((double)u * (double)total, __longlong_as_double(__double_as_longlong((double)total) - 1));   // u = 1: the last one
    if ((double)before <= want && (double)(before + own) > want) {
      u64 at = before;
      for (int i = mine; i < mine_end; ++i) {
        const float x = xs[i];
        if (((u64)key_of(x) << 32 | (uint32_t)~(first + i)) < cut) continue;
        u64 w;
        if (kept_weight(x, w)) at += w;
        if ((double)at > want) {
          p.ids[row] = first + i;
          if (p.logprob) p.logprob[row] = (float)(scaled(x) - log_all);
          break;
        }
      }
    }
  }
  cluster_barrier();                                   // no block leaves while another may read its shared memory
}

}  // namespace omni

using namespace omni;

// logits [B, V] of pitch ld, bf16 or fp32; parameters per row or (null) one value for all; u fp32 [B]; ids int32 [B], logprob fp32 [B] or null.
extern "C" int omni_sample_given(const void* logits, int is_bf16, long ld, int V, int B, const float* u, const float* temperature, float temperature_v, const int* top_k,
                                 int top_k_v, const float* top_p, float top_p_v, const float* min_p, float min_p_v, int* ids, float* logprob, void* stream) {
  if (B <= 0) return RC_OK;
  if (V < 1 || V > SG_MAX_V) return RC_BAD_ARG;
  SampleGiven p = {logits, ld, V, 0, temperature, top_p, min_p, u, top_k, temperature_v, top_p_v, min_p_v, top_k_v, ids, logprob};
  int nc = 1;
  while (nc < SG_MAX_CLUSTER && V > nc * SG_THREADS * 9) nc *= 2;
  p.per = ((V + nc * SG_THREADS - 1) / (nc * SG_THREADS)) | 1;
  if ((long)B * nc > 0x7fffffffL) return RC_TOO_LARGE;
  const int smem = (int)sizeof(SgShared) + SG_THREADS * p.per * 4;
  static unsigned long long ready[2] = {0, 0};
  const void* fn = is_bf16 ? (const void*)sample_given_kernel<__nv_bfloat16> : (const void*)sample_given_kernel<float>;
  if (int e = ensure_dynamic_smem(fn, (int)sizeof(SgShared) + SG_THREADS * (SG_MAX_V / (SG_MAX_CLUSTER * SG_THREADS) + 1) * 4, ready[is_bf16 ? 0 : 1])) return e;
  launch_with(true, nc, is_bf16 ? sample_given_kernel<__nv_bfloat16> : sample_given_kernel<float>, dim3((unsigned)(B * nc)), SG_THREADS, smem, (cudaStream_t)stream, p);
  return (int)cudaGetLastError();
}
